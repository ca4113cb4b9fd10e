// Error text and version of include/s4d_decoder.h (its own library, so that a program of the DFA
// path alone loads nothing of it).
#include <stdarg.h>
#include <stdio.h>

#include "common.cuh"
#include "s4d_decoder.h"

namespace s4d {

static thread_local char g_last_error[512] = "";
static thread_local unsigned long long g_wait_limit_ns = 2000000000ull;

unsigned long long decoder_wait_limit_ns() { return g_wait_limit_ns; }

void set_error(const char* fmt, ...) {
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(g_last_error, sizeof(g_last_error), fmt, ap);
  va_end(ap);
}

}  // namespace s4d

extern "C" {

const char* s4d_decoder_last_error(void) { return s4d::g_last_error; }

int s4d_decoder_abi_version(void) { return 2; }

uint64_t s4d_decoder_set_wait_limit_ns(uint64_t limit_ns) {
  const uint64_t prev = s4d::g_wait_limit_ns;
  s4d::g_wait_limit_ns = limit_ns;
  return prev;
}

}  // extern "C"
