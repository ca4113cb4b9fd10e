// Error text and version of include/s4d_decoder.h (its own library, so that a program of the DFA
// path alone loads nothing of it).
#include <stdarg.h>
#include <stdio.h>

#include "common.cuh"
#include "s4d_decoder.h"

namespace s4d {

static thread_local char g_last_error[512] = "";

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

}  // namespace s4d

extern "C" {

const char* s4d_decoder_last_error(void) { return s4d::g_last_error; }

int s4d_decoder_abi_version(void) { return 1; }

}  // extern "C"
