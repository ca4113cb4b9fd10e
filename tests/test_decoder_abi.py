"""The decoder library's C ABI: it loads, exports what include/s4d_decoder.h declares, and rejects bad
arguments on the host with a status code (no GPU needed: none of these calls reaches a launch)."""
import os
import re
import subprocess

import pytest
import torch

import sparse4d_tt_b200 as s4d
from sparse4d_tt_b200 import _lib as L
from sparse4d_tt_b200 import _lib_decoder as D

REPO = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
HEADER = os.path.join(REPO, "include", "s4d_decoder.h")
OK, INVALID, UNSUPPORTED = L.S4D_OK, L.S4D_ERR_INVALID_ARG, L.S4D_ERR_UNSUPPORTED_SHAPE
P = 0x1000  # an aligned address that no call here gets to read


@pytest.fixture(scope="module")
def lib():
    if not os.path.exists(D.LIB_PATH):
        import importlib.util

        spec = importlib.util.spec_from_file_location("s4d_build", os.path.join(REPO, "sparse4d-tt_b200", "build.py"))
        b = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(b)
        b.build_decoder()
    return D.lib()


def test_exports_are_the_header(lib):
    text = re.sub(r"/\*.*?\*/", "", open(HEADER).read(), flags=re.S)
    declared = set(re.findall(r"\b(s4d_[a-z_0-9]+)\s*\(", text))
    out = subprocess.run(["nm", "-D", "--defined-only", D.LIB_PATH], capture_output=True, text=True).stdout
    exported = {ln.split()[-1] for ln in out.splitlines() if " T " in ln}
    assert {n for n in exported if n.startswith("s4d_")} == declared == set(D.SIGNATURES)
    assert lib.s4d_decoder_abi_version() == D.ABI_VERSION


def test_attention_args_format_is_the_struct(tmp_path):
    """The packed arguments have the C struct's size and field offsets."""
    import shutil
    import struct

    cc = shutil.which("gcc") or shutil.which("cc")
    if cc is None:
        pytest.skip("no C compiler")
    fields = ("batch q q_stride k_stride out lse slope_stride q_pos k_len workspace workspace_bytes error_flag scale dtype "
              "dslopes_per_row dout dout_stride dq dslopes").split()
    src = tmp_path / "o.c"
    src.write_text('#include "s4d_decoder.h"\n#include <stdio.h>\n#include <stddef.h>\nint main(void){'
                   + "".join(f'printf("%zu ", offsetof(s4d_attention_args, {f}));' for f in fields)
                   + 'printf("%zu", sizeof(s4d_attention_args));return 0;}')
    subprocess.run([cc, "-I", os.path.join(REPO, "include"), str(src), "-o", str(tmp_path / "o")], check=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "o")], capture_output=True, text=True).stdout.split()]
    before = ("", "7q", "7q3P", "7q3P3q", "7q3P9q", "7q3P9qP", "7q3P9q3P", "7q3P9q3P3q", "7q3P9q3P3q4P", "7q3P9q3P3q5P",
              "7q3P9q3P3q6P", "7q3P9q3P3q6PN", "7q3P9q3P3q6PNP", "7q3P9q3P3q6PNP2f", "7q3P9q3P3q6PNP2fi",
              "7q3P9q3P3q6PNP2f2i", "7q3P9q3P3q6PNP2f2iP", "7q3P9q3P3q6PNP2f2iP3q", "7q3P9q3P3q6PNP2f2iP3q3P")
    assert got == [struct.calcsize("@" + f) for f in before] + [D.ATTENTION_ARGS.size]


def norm_fwd(lib, **kw):
    a = dict(x=P, ld=256, dtype=0, w=P, b=P, pt=0, y=P, yld=256, mean=P, rstd=P, rows=4, width=256, eps=1e-5)
    a.update(kw)
    st = lib.s4d_norm_forward(a["x"], a["ld"], a["dtype"], a["w"], a["b"], a["pt"], a["y"], a["yld"], a["mean"],
                              a["rstd"], a["rows"], a["width"], a["eps"], None)
    return st, lib.s4d_decoder_last_error().decode()


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=9), INVALID, "dtype"), (dict(pt=1), INVALID, "weight and bias"), (dict(rows=-1), INVALID, "rows"),
    (dict(width=0), INVALID, "width"), (dict(width=16385, ld=16385, yld=16385), UNSUPPORTED, "16384"),
    (dict(yld=255), INVALID, "strides"), (dict(ld=-1), INVALID, "strides"), (dict(x=None), INVALID, "null"),
    (dict(y=None), INVALID, "null"), (dict(mean=None), INVALID, "together"), (dict(x=P + 2), INVALID, "misaligned"),
    (dict(eps=-1.0), INVALID, "eps"), (dict(eps=float("nan")), INVALID, "eps"),
    (dict(rows=1 << 40), UNSUPPORTED, "too many"), (dict(rows=0, x=None, y=None), OK, ""),
])
def test_norm_forward_rejects_on_host(lib, kw, status, text):
    st, msg = norm_fwd(lib, **kw)
    assert st == status and text in msg, (st, msg)


def norm_bwd(lib, **kw):
    a = dict(dy=P, dld=256, x=P, ld=256, dtype=1, w=P, pt=1, mean=P, rstd=P, dx=P, dxld=256, dw=P, db=P, rows=5000,
             width=256, ws=P, wsb=1 << 20)
    a.update(kw)
    st = lib.s4d_norm_backward(a["dy"], a["dld"], a["x"], a["ld"], a["dtype"], a["w"], a["pt"], a["mean"], a["rstd"],
                               a["dx"], a["dxld"], a["dw"], a["db"], a["rows"], a["width"], a["ws"], a["wsb"], None)
    return st, lib.s4d_decoder_last_error().decode()


@pytest.mark.parametrize("kw,status,text", [
    (dict(pt=2), INVALID, "weight and bias"), (dict(dy=None), INVALID, "null"), (dict(mean=None), INVALID, "null"),
    (dict(ws=None), INVALID, "workspace"), (dict(wsb=16), INVALID, "workspace"), (dict(ws=P + 8), INVALID, "workspace"),
    (dict(dld=-4), INVALID, "strides"), (dict(dxld=8), INVALID, "strides"), (dict(dw=P + 1), INVALID, "misaligned"),
    (dict(width=20000), UNSUPPORTED, "16384"),
])
def test_norm_backward_rejects_on_host(lib, kw, status, text):
    st, msg = norm_bwd(lib, **kw)
    assert st == status and text in msg, (st, msg)


def test_norm_workspace(lib):
    assert lib.s4d_norm_backward_workspace_bytes(0, 256) == 0
    assert lib.s4d_norm_backward_workspace_bytes(5, 0) == 0
    assert lib.s4d_norm_backward_workspace_bytes(8, 256) == 0  # summed by the one launch
    assert lib.s4d_norm_backward_workspace_bytes(3000, 256) % (2 * 256 * 4) == 0
    assert lib.s4d_norm_backward_workspace_bytes(3000, 256) > 0
    assert lib.s4d_norm_backward_workspace_bytes(1 << 40, 256) == 0
    assert lib.s4d_norm_backward_workspace_bytes(100000, 16384) >= 2 * 16384 * 4


def test_norm_rejects_cpu_tensors_and_bad_arguments():
    x = torch.zeros(4, 8)
    with pytest.raises(ValueError, match="CUDA"):
        s4d.decoder_norm_forward(x)
    with pytest.raises(ValueError, match="CUDA"):
        s4d.decoder_norm(x, torch.ones(8), torch.zeros(8))
    with pytest.raises(ValueError, match="CUDA"):
        s4d.decoder_norm_backward(x, x, None, torch.zeros(4), torch.zeros(4))
