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


# ---- attention ------------------------------------------------------------------------------------------


def attention_args(**kw):
    a = dict(batch=2, queries=10, keys=20, heads=4, kv_heads=2, dim=64, pos_dim=0, q=P, k=P, v=P,
             q_stride=(2560, 256, 64), k_stride=(2560, 128, 64), v_stride=(2560, 128, 64), out=P, lse=P, slopes=0,
             slope_stride=(0, 0, 1), q_pos=0, k_pos=0, q_segment=0, k_segment=0, k_len=0, ws=0, wsb=0, flag=0,
             scale=0.125, softcap=0.0, dtype=1, per_row=0, dout=P, dout_stride=(2560, 256, 64), dq=P, dk=P, dv=P,
             dslopes=0)
    a.update(kw)
    return D.ATTENTION_ARGS.pack(
        a["batch"], a["queries"], a["keys"], a["heads"], a["kv_heads"], a["dim"], a["pos_dim"], a["q"], a["k"], a["v"],
        *a["q_stride"], *a["k_stride"], *a["v_stride"], a["out"], a["lse"], a["slopes"], *a["slope_stride"], a["q_pos"],
        a["k_pos"], a["q_segment"], a["k_segment"], a["k_len"], a["ws"], a["wsb"], a["flag"], a["scale"], a["softcap"],
        a["dtype"], a["per_row"], a["dout"], *a["dout_stride"], a["dq"], a["dk"], a["dv"], a["dslopes"])


SHARED = [
    (dict(dtype=0), INVALID, "bf16 or f16"), (dict(batch=-1), INVALID, "sizes"), (dict(heads=3), INVALID, "multiple"),
    (dict(kv_heads=0), INVALID, "sizes"), (dict(dim=60), UNSUPPORTED, "dim"), (dict(dim=136), UNSUPPORTED, "dim"),
    (dict(dim=0), UNSUPPORTED, "dim"), (dict(pos_dim=3), UNSUPPORTED, "pos_dim"),
    (dict(scale=float("inf")), INVALID, "scale"), (dict(scale=float("nan")), INVALID, "scale"),
    (dict(softcap=-1.0), INVALID, "softcap"), (dict(softcap=float("nan")), INVALID, "softcap"),
    (dict(queries=1 << 31), UNSUPPORTED, "too many"), (dict(keys=1 << 31), UNSUPPORTED, "too many"),
    (dict(batch=1 << 20, queries=1 << 20), UNSUPPORTED, "too many"), (dict(q_segment=P), INVALID, "together"),
    (dict(q=P + 8), INVALID, "misaligned"), (dict(k_len=P + 2), INVALID, "misaligned"), (dict(q=0), INVALID, "null q"),
    (dict(v=0), INVALID, "null k or v"), (dict(out=0), INVALID, "null q or out"),
    (dict(pos_dim=1), INVALID, "null slopes"), (dict(pos_dim=1, slopes=P, q_pos=P), INVALID, "null slopes"),
    (dict(q_stride=(2560, 256, 60)), INVALID, "strides"), (dict(k_stride=(2560, 0, 64)), INVALID, "strides"),
    (dict(v_stride=(-8, 128, 64)), INVALID, "strides"), (dict(v_stride=(1 << 40, 128, 64)), INVALID, "strides"),
]


@pytest.mark.parametrize("kw,status,text", SHARED)
def test_attention_rejects_on_host(lib, kw, status, text):
    for fn in (lib.s4d_attention_forward, lib.s4d_attention_backward):
        st = fn(attention_args(ws=P, wsb=1 << 30, **kw), None)
        msg = lib.s4d_decoder_last_error().decode()
        assert st == status and text in msg, (st, msg)


@pytest.mark.parametrize("kw,text", [
    (dict(softcap=1025.0), "1024"), (dict(softcap=float("inf")), "1024"), (dict(softcap=1e-38, scale=100.0), "too large"),
    (dict(scale=3e38), "too large"), (dict(scale=-3e38), "too large"),
])
def test_attention_rejects_scales_without_an_fp32_score(lib, kw, text):
    for fn in (lib.s4d_attention_forward, lib.s4d_attention_backward):
        st = fn(attention_args(ws=P, wsb=1 << 30, **kw), None)
        msg = lib.s4d_decoder_last_error().decode()
        assert st == INVALID and text in msg, (st, msg)


@pytest.mark.parametrize("kw,status,text", [
    (dict(dtype=2), UNSUPPORTED, "bf16"), (dict(keys=(1 << 19) + 1), UNSUPPORTED, "524288"), (dict(dk=0), INVALID, "together"),
    (dict(dout=0), INVALID, "null dout"), (dict(dq=0), INVALID, "null dout"), (dict(lse=0), INVALID, "null dout"),
    (dict(dslopes=P), INVALID, "without a distance bias"), (dict(dout_stride=(2560, 256, 4)), INVALID, "strides of dout"),
    (dict(dq=P + 8), INVALID, "misaligned"), (dict(wsb=64), INVALID, "workspace"), (dict(ws=0), INVALID, "workspace"),
    (dict(batch=0, q=0, k=0, v=0, out=0, dout=0, dq=0, dk=0, dv=0), OK, ""),
])
def test_attention_backward_rejects_on_host(lib, kw, status, text):
    st = lib.s4d_attention_backward(attention_args(**dict(dict(ws=P, wsb=1 << 30), **kw)), None)
    assert st == status and text in lib.s4d_decoder_last_error().decode()


def test_attention_forward_empty_and_workspace(lib):
    assert lib.s4d_attention_forward(attention_args(batch=0, q=0, k=0, v=0, out=0), None) == OK
    assert lib.s4d_attention_forward(attention_args(queries=0, q=0, out=0), None) == OK
    need = lib.s4d_attention_forward_workspace_bytes
    assert need(attention_args()) == 0                                       # short keys: one part
    assert need(attention_args(batch=64, queries=900, keys=900)) == 0        # rows enough
    long = dict(batch=1, queries=1, keys=1 << 20, heads=1, kv_heads=1, k_stride=(64, 64, 64), v_stride=(64, 64, 64))
    assert need(attention_args(**long)) % (65 * 4) == 0 and need(attention_args(**long)) > 0
    st = lib.s4d_attention_forward(attention_args(**long), None)
    assert st == INVALID and "workspace" in lib.s4d_decoder_last_error().decode()
    assert need(attention_args(heads=3)) == 0 and need(attention_args(batch=-2)) == 0
    assert lib.s4d_attention_forward(None, None) == INVALID
    assert need(None) == 0 and lib.s4d_attention_backward_workspace_bytes(None) == 0


def test_attention_rejects_cpu_tensors():
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    for call in (lambda: s4d.decoder_attention_forward(q, q, q), lambda: s4d.decoder_attention(q, q, q),
                 lambda: s4d.decoder_attention_backward(q, q, q, q, q, torch.zeros(1, 2, 4))):
        with pytest.raises(ValueError, match="CUDA"):
            call()


def test_launches_go_to_the_tensors_device(monkeypatch):
    """A guard is entered only when the tensors' device is not the current one."""
    entered = []

    class Guard:
        def __init__(self, index):
            self.index = index

        def __enter__(self):
            entered.append(self.index)

        def __exit__(self, *exc):
            entered.append("out")

    monkeypatch.setattr(torch._C, "_cuda_getDevice", lambda: 0, raising=False)
    monkeypatch.setattr(torch.cuda, "device", Guard)
    with D.on_device(0):
        pass
    assert not entered
    with D.on_device(3):
        entered.append("in")
    assert entered == [3, "in", "out"]


def test_overlap():
    x = torch.zeros(100, 64)
    a, b = x[:, :32], x[:, 32:]
    assert D.overlap(x, a) and D.overlap(a, b)          # a and b interleave: their ranges meet
    assert not D.overlap(x[:50], x[50:]) and D.overlap(x[:51], x[50:])
    assert not D.overlap(x[:0], x) and not D.overlap(x, torch.zeros(3))
    assert D.overlap(x[0].expand(5, 64), x[0]) and not D.overlap(x[0].expand(5, 64), x[1])


def test_calls_module_leaves_what_is_not_its_to_take():
    """Tensors off the current CUDA device, wrong counts and wrong kinds of arguments answer None."""
    c = D.calls()
    x, s = torch.zeros(4, 8), torch.zeros(4)
    assert c.norm_forward(x, None, None, 1e-5) is None
    assert c.norm_forward(x, None, None) is None and c.norm_forward(None, None, None, 1e-5) is None
    assert c.norm_forward(3, None, None, 1e-5) is None
    assert c.norm_backward(x, x, None, s, s, True, True, True) is None
    q = torch.zeros(1, 4, 2, 64, dtype=torch.bfloat16)
    assert c.attention_forward(q, q, q, None, 0.0, *[None] * 6) is None
    assert c.attention_forward(None, None, None, None, 0.0, *[None] * 6) is None


def test_wait_limit_is_per_thread_and_restorable(lib):
    import threading

    prev = lib.s4d_decoder_set_wait_limit_ns(12345)
    assert prev == 2_000_000_000
    seen = []
    t = threading.Thread(target=lambda: seen.append(lib.s4d_decoder_set_wait_limit_ns(7)))
    t.start()
    t.join()
    assert seen == [2_000_000_000]  # another thread keeps its own default
    assert lib.s4d_decoder_set_wait_limit_ns(prev) == 12345


def test_calls_module_of_another_torch_is_not_taken(monkeypatch, tmp_path):
    """The module is compiled against torch's and Python's internals: one that was built for other versions is neither
    kept by the build nor loaded."""
    from sparse4d_tt_b200 import build as b

    built = []

    def run(cmd, what, verbose):
        built.append(cmd[cmd.index("-o") + 1])
        open(built[-1], "w").close()

    monkeypatch.setattr(b, "_run", run)
    monkeypatch.setattr(b, "LIB_DIR", str(tmp_path))
    first = b.build_calls()
    assert b.build_calls() == first and len(built) == 1
    monkeypatch.setattr(torch, "__version__", "9.9.9")
    monkeypatch.setattr(D, "_calls", None)
    with pytest.raises(RuntimeError, match="not built"):
        D.calls()
    second = b.build_calls()
    assert second != first and len(built) == 2
    os.utime(second, (0, 0))  # older than its sources and its flags
    assert b.build_calls() == second and len(built) == 3
