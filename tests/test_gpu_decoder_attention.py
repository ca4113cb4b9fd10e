"""decoder_attention against its definition in 64 bits (attention_ref.py).

Bound of the forward pass, h half a step of the type: P is rounded once (h of P |V| a key), a score is
off by e (score_error) and so is the log-sum-exp, which moves a weight by 2 e relative; sums over the
keys in fp32 add at most (tiles + 160) u; the result is rounded once (h of |out|).  So
|error| <= h |out| + (1 + h) (h + 2 e + 200 u) sum P |V|; fp16 weights below its normal range are off
by 2^-25 each instead."""
import math

import pytest
import torch

from attention_ref import U, half_step, reference, score_error
from sparse4d_tt_b200 import _lib_decoder as lib_decoder
from sparse4d_tt_b200 import decoder_attention, decoder_attention_backward, decoder_attention_forward
from sparse4d_tt_b200._lib import S4D_FLAG_WAIT_TIMEOUT
from sparse4d_tt_b200.graph import capture

pytestmark = pytest.mark.gpu


def make(B, Nq, Nk, H, G, D, dtype=torch.bfloat16, pos=0, slopes="head", segments=None, k_len=None, cap=0.0, seed=0):
    g = torch.Generator().manual_seed(seed * 7919 + Nq * 31 + Nk)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    q, k, v = (t.to(dtype).cuda() for t in (r(B, Nq, H, D), r(B, Nk, G, D), r(B, Nk, G, D)))
    how = {"softcap": cap}
    if pos:
        how["q_pos"], how["k_pos"] = (torch.rand(B, Nq, pos, generator=g) * 60).cuda(), (
            torch.rand(B, Nk, pos, generator=g) * 60).cuda()
        how["slopes"] = (0.2 * torch.rand(*((H,) if slopes == "head" else (B, Nq, H)), generator=g)).cuda()
    if segments is not None:
        how["q_segment"], how["k_segment"] = (torch.as_tensor(s, dtype=torch.int32).expand(B, -1).contiguous().cuda()
                                              for s in segments)
    if k_len is not None:
        how["k_len"] = torch.tensor(k_len, dtype=torch.int32).cuda()
    return q, k, v, how


def check_forward(q, k, v, how, out, lse):
    ref = reference(q, k, v, **how)
    h = half_step(q.dtype)
    e = score_error(q, k, how.get("scale"), how.get("softcap", 0.0), how.get("slopes"), how.get("q_pos"),
                    how.get("k_pos"))
    tol = h * ref["out"].abs() + (1 + h) * (h + 2 * e + 200 * U) * ref["out_abs"]
    if q.dtype == torch.float16:  # subnormal weights and results
        tol = tol + 2.0 ** -24 + 2.0 ** -25 * v.nan_to_num(0, 0, 0).abs().double().sum(1).max()
    err = (out.double() - ref["out"]).abs()
    assert out.shape == q.shape and out.dtype == q.dtype
    assert (err <= tol).all(), (err - tol).max()
    empty = ref["lse"] == -math.inf
    assert torch.equal(lse == -math.inf, empty)
    gap = torch.where(empty, torch.zeros_like(ref["lse"]), lse.double() - ref["lse"]).abs()
    assert gap.max() <= e + 300 * U * (1 + ref["lse"].masked_fill(empty, 0).abs().max()), gap.max()
    return ref


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Nq,Nk,H,G,D", [
    (1, 1, 1, 1, 1, 64), (2, 5, 3, 2, 2, 64), (1, 128, 128, 2, 1, 64), (1, 129, 257, 3, 3, 64), (2, 900, 900, 8, 8, 64),
    (1, 200, 300, 6, 2, 32), (2, 77, 130, 4, 4, 8), (1, 150, 401, 4, 2, 128), (1, 300, 140, 3, 1, 96),
    (2, 65, 128, 5, 5, 72), (1, 1, 5000, 8, 2, 128), (3, 4, 1000, 8, 8, 64), (1, 16, 2050, 14, 2, 40),
])
def test_plain(cuda_device, dtype, B, Nq, Nk, H, G, D):
    q, k, v, how = make(B, Nq, Nk, H, G, D, dtype)
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pos,slopes", [(1, "head"), (2, "head"), (2, "row"), (0, None)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_bias_and_cap(cuda_device, D, pos, slopes, cap):
    for dtype, shape in ((torch.bfloat16, (2, 190, 333, 4, 2)), (torch.float16, (1, 3, 700, 4, 4))):
        q, k, v, how = make(*shape, D, dtype, pos=pos, slopes=slopes, cap=cap)
        check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))


def ids(*sizes):
    """Segment ids: sizes of documents in order, a negative size is padding."""
    out, d = [], 0
    for n in sizes:
        out += [-1] * -n if n < 0 else [d] * n
        d += n > 0
    return out


@pytest.mark.parametrize("q_ids,k_ids", [
    (ids(300, 80, 20), ids(300, 80, 20)), (ids(128, 128, 128), ids(128, 128, 128)), (ids(10, -5, 200, 1), ids(3, 90, -7, 1)),
    ([i % 3 for i in range(150)], [i % 4 for i in range(290)]), ([-1] * 40, [0] * 60), ([5] * 40, [7] * 500),
    ([7], [i // 100 for i in range(1500)]),
])
@pytest.mark.parametrize("k_len", [None, [260, 0]])
def test_documents(cuda_device, q_ids, k_ids, k_len):
    """Contiguous, interleaved, padded and unmatched documents, alone and with valid lengths."""
    q, k, v, how = make(2, len(q_ids), len(k_ids), 4, 2, 64, segments=(q_ids, k_ids), k_len=k_len, pos=1)
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))


@pytest.mark.parametrize("Nq", [1, 200])
@pytest.mark.parametrize("Nk", [600, 1300])
def test_valid_lengths(cuda_device, Nq, Nk):
    """No key, one, ends inside and at tiles, all, and values outside the range."""
    lens = [0, 1, 127, 128, 129, Nk, Nk + 50, -3]
    q, k, v, how = make(len(lens), Nq, Nk, 2, 1, 64, torch.float16, k_len=lens, cap=10.0)
    out, lse = decoder_attention_forward(q, k, v, **how)
    check_forward(q, k, v, how, out, lse)
    assert not out[0].any() and not out[7].any() and (lse[0] == -math.inf).all()


def test_no_keys_no_queries_no_batch(cuda_device):
    q, k, v, _ = make(2, 5, 3, 2, 1, 64)
    out, lse = decoder_attention_forward(q, k[:, :0], v[:, :0])
    assert not out.any() and (lse == -math.inf).all()
    assert decoder_attention_forward(q[:, :0], k, v)[0].shape == (2, 0, 2, 64)
    assert decoder_attention_forward(q[:0], k[:0], v[:0])[0].shape == (0, 5, 2, 64)


@pytest.mark.parametrize("bad", [math.nan, math.inf, -math.inf])
@pytest.mark.parametrize("Nq", [2, 300])
@pytest.mark.parametrize("D", [64, 128])
def test_values_behind_masks_do_not_reach_out(cuda_device, D, Nq, bad):
    """Keys past the valid length, padding and another document hold infinities and NaNs: the rows that do
    not see them are bit-equal to the ones without; the rows that do are not numbers."""
    sizes = ids(150, 60, 90, -20)
    qid = [sizes[i * len(sizes) // Nq] for i in range(Nq)]
    q, k, v, how = make(2, Nq, len(sizes), 4, 2, D, segments=(qid, sizes), k_len=[320, 280], pos=2, cap=20.0)
    clean, clean_lse = decoder_attention_forward(q, k, v, **how)
    k2, v2 = k.clone(), v.clone()
    how2 = dict(how, k_pos=how["k_pos"].clone())
    k2[0, 300:], v2[0, 300:] = bad, bad      # padding ids
    k2[1, 280:], v2[1, 280:] = bad, bad      # past the valid length
    how2["k_pos"][0, 300:] = bad
    v2[:, 160] = bad                         # document 1
    out, lse = decoder_attention_forward(q, k2, v2, **how2)
    seg = torch.tensor(qid, device="cuda")
    other = seg != 1
    assert torch.isfinite(clean).all()
    tol = 2 * half_step(torch.bfloat16)  # a bad tile's products are added in another order
    err = (out[:, other].float() - clean[:, other].float()).abs()
    assert (err <= tol * (clean[:, other].float().abs() + 1.0)).all(), err.max()
    assert torch.equal(lse, clean_lse)
    sees = out[:, ~other]
    assert not torch.isfinite(sees).any()
    for _ in range(60):  # the masked tiles' slow way runs beside the other stream of tiles: never another result
        again, _ = decoder_attention_forward(q, k2, v2, **how2)
        assert torch.equal(again[:, other], out[:, other]) and not torch.isfinite(again[:, ~other]).any()


def test_rows_that_are_no_numbers_stay_alone(cuda_device):
    q, k, v, how = make(1, 140, 200, 2, 2, 64)
    clean, _ = decoder_attention_forward(q, k, v, **how)
    q[0, 7] = math.nan
    out, lse = decoder_attention_forward(q, k, v, **how)
    keep = [i for i in range(140) if i != 7]
    assert torch.equal(out[:, keep], clean[:, keep]) and torch.isnan(out[0, 7]).all() and torch.isnan(lse[0, :, 7]).all()


def test_large_scores(cuda_device):
    """Scores of thousands, growing along the keys, so that the running maximum moves at every tile."""
    q, k, v, how = make(1, 130, 900, 2, 2, 64)
    ramp = torch.linspace(0.1, 60, 900, device="cuda").to(k.dtype)
    k = k.abs() * ramp[None, :, None, None]
    q = q.abs()
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))
    how["scale"] = -0.125  # and a negative scale
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))


def test_strides_and_views(cuda_device):
    """The slices of one [B, N, 3, H, D] projection, [B, H, N, D] storage, expanded heads, odd offsets."""
    g = torch.Generator().manual_seed(5)
    qkv = torch.randn(2, 170, 3, 4, 64, generator=g).bfloat16().cuda()
    q, k, v = qkv.unbind(2)
    want, wl = decoder_attention_forward(q.contiguous(), k.contiguous(), v.contiguous())
    got, gl = decoder_attention_forward(q, k, v)
    assert torch.equal(want, got) and torch.equal(wl, gl)
    t = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v)]
    assert torch.equal(want, decoder_attention_forward(*t)[0])
    e = k[:, :, :1].expand(-1, -1, 4, -1)
    assert torch.equal(decoder_attention_forward(q, e, e)[0], decoder_attention_forward(q, k[:, :, :1], k[:, :, :1])[0])
    flat = torch.zeros(q.numel() + 3, dtype=q.dtype, device="cuda")
    odd = flat[3:].view(q.shape)
    odd.copy_(q)
    assert torch.equal(want, decoder_attention_forward(odd, k, v)[0])
    tr = k.transpose(1, 3).contiguous().transpose(1, 3)
    assert torch.equal(want, decoder_attention_forward(q, tr, v)[0])
    out = torch.empty_like(want)
    assert decoder_attention_forward(q, k, v, out=out)[0] is out and torch.equal(out, want)


def test_long_cache_offsets(cuda_device):
    """A cache whose element offsets pass 2^31: the last batch entry equals its own copy."""
    keys, G, D = 9000, 8, 128
    rows = (1 << 31) // (keys * G * D) + 2
    k = torch.zeros(rows, keys, G, D, dtype=torch.bfloat16, device="cuda")
    k[-1].normal_()
    q = torch.randn(rows, 1, G, D, device="cuda").bfloat16()
    out, _ = decoder_attention_forward(q, k, k)
    assert k.numel() > 1 << 31
    alone, _ = decoder_attention_forward(q[-1:], k[-1:].clone(), k[-1:].clone())
    assert not out[:-1].any()
    ref = reference(q[-1:], k[-1:], k[-1:])["out"]
    for t in (out[-1:], alone):
        assert (t.double() - ref).abs().max() <= 3 * half_step(torch.bfloat16) * ref.abs().max()


def test_equal_bits_streams_and_graphs(cuda_device):
    """Equal calls give equal bits, split along the keys or not; captured twice and replayed in turn with
    the eager call between them (their workspaces do not meet)."""
    for shape in ((1, 300, 900, 4, 4, 64), (1, 2, 4000, 4, 2, 128)):
        q, k, v, how = make(*shape, pos=2)
        call = lambda: decoder_attention_forward(q, k, v, **how)  # noqa: E731
        first = [t.clone() for t in call()]
        a, b = capture(call), capture(call)
        side = torch.cuda.Stream()
        side.wait_stream(torch.cuda.current_stream())
        with torch.cuda.stream(side):
            other = call()
        torch.cuda.current_stream().wait_stream(side)
        for run in (a.replay, call, b.replay, a.replay):
            assert all(torch.equal(x, y) for x, y in zip(first, run()))
        assert all(torch.equal(x, y) for x, y in zip(first, other))
        q.neg_()
        assert torch.equal(a.replay()[0], call()[0]) and not torch.equal(call()[0], first[0])


# ---- gradients --------------------------------------------------------------------------------------


def check_backward(q, k, v, how, dout, grads, out=None):
    ref = reference(q, k, v, **how, dout=dout)
    h = half_step(q.dtype)
    names = ("dq", "dk", "dv") + (("dslopes",) if "slopes" in how else ())
    assert (grads[3] is None) == ("slopes" not in how)
    for n, got in zip(names, grads):
        want, tol = ref[n], ref[n + "_tol"]
        if n == "dslopes":
            if how["slopes"].dim() == 1:
                tol = tol.sum((0, 1)) + want.shape[0] * want.shape[1] * U * want.abs().sum((0, 1))
                want = want.sum((0, 1))
            tol = tol + 2 * U * want.abs()
        else:
            tol = (1 + h) * tol + h * want.abs()
        assert got.shape == want.shape, n
        err = (got.double() - want).abs()
        assert (err <= tol).all(), (n, (err - tol).max(), err.max())


def gradients(q, k, v, how, seed=3):
    g = torch.Generator().manual_seed(seed)
    dout = torch.randn(q.shape, generator=g).to(q.dtype).cuda()
    out, lse = decoder_attention_forward(q, k, v, **how)
    return dout, decoder_attention_backward(dout, q, k, v, out, lse, **how)


@pytest.mark.parametrize("B,Nq,Nk,H,G,D", [
    (1, 1, 1, 1, 1, 64), (2, 5, 3, 2, 2, 64), (1, 128, 128, 2, 1, 64), (1, 129, 257, 3, 3, 64), (1, 900, 900, 4, 4, 64),
    (1, 200, 300, 6, 2, 32), (2, 77, 130, 4, 4, 8), (1, 150, 401, 4, 2, 128), (1, 300, 140, 3, 1, 96), (2, 65, 128, 5, 5, 72),
    (1, 1, 1500, 4, 2, 128), (3, 400, 2, 2, 2, 64),
])
def test_gradients_plain(cuda_device, B, Nq, Nk, H, G, D):
    q, k, v, how = make(B, Nq, Nk, H, G, D)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)


@pytest.mark.parametrize("D", [64, 128])
@pytest.mark.parametrize("pos,slopes", [(1, "head"), (2, "head"), (2, "row"), (0, None)])
@pytest.mark.parametrize("cap", [0.0, 5.0])
def test_gradients_bias_and_cap(cuda_device, D, pos, slopes, cap):
    q, k, v, how = make(2, 190, 333, 4, 2, D, pos=pos, slopes=slopes, cap=cap)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)


@pytest.mark.parametrize("q_ids,k_ids", [
    (ids(300, 80, 20), ids(300, 80, 20)), (ids(128, 128, 128), ids(128, 128, 128)), (ids(10, -5, 200, 1), ids(3, 90, -7, 1)),
    ([i % 3 for i in range(150)], [i % 4 for i in range(290)]), ([-1] * 40, [0] * 60), ([5] * 40, [7] * 500),
])
@pytest.mark.parametrize("k_len", [None, [260, 0]])
def test_gradients_documents(cuda_device, q_ids, k_ids, k_len):
    q, k, v, how = make(2, len(q_ids), len(k_ids), 4, 2, 64, segments=(q_ids, k_ids), k_len=k_len, pos=1)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)


def test_gradients_valid_lengths(cuda_device):
    lens = [0, 1, 127, 128, 129, 600, 700, -3]
    q, k, v, how = make(8, 100, 600, 2, 1, 64, k_len=lens, cap=10.0)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)
    assert not grads[0][0].any() and not grads[1][7].any() and not grads[1][1, 1:].any() and not grads[2][2, 127:].any()


def test_gradients_without_keys_queries_or_batch(cuda_device):
    q, k, v, how = make(2, 5, 3, 2, 1, 64, pos=2)
    full = dict(how)
    how["k_pos"] = full["k_pos"][:, :0]
    _, (dq, dk, dv, ds) = gradients(q, k[:, :0], v[:, :0], how)
    assert not dq.any() and dk.shape == (2, 0, 1, 64) and not ds.any()
    how = dict(full, q_pos=full["q_pos"][:, :0])
    _, (dq, dk, dv, ds) = gradients(q[:, :0], k, v, how)
    assert dq.shape == (2, 0, 2, 64) and not dk.any() and not dv.any() and not ds.any()
    how = dict(full, q_pos=full["q_pos"][:0], k_pos=full["k_pos"][:0])
    _, (dq, dk, dv, ds) = gradients(q[:0], k[:0], v[:0], how)
    assert dk.shape == (0, 3, 1, 64) and not ds.any()


@pytest.mark.parametrize("bad", [math.nan, math.inf])
@pytest.mark.parametrize("D", [64, 128])
def test_gradients_ignore_values_behind_masks(cuda_device, D, bad):
    """Infinities and NaNs in padding, past the valid length and in another document, in keys, values,
    queries and the output's gradient."""
    sizes = ids(150, 60, 90, -20)
    q, k, v, how = make(2, 320, 320, 4, 2, D, segments=(sizes, sizes), k_len=[320, 280], pos=2, slopes="row", cap=20.0)
    dout, clean = gradients(q, k, v, how)
    t = [x.clone() for x in (q, k, v, dout)]
    how = dict(how, q_pos=how["q_pos"].clone(), k_pos=how["k_pos"].clone())
    for x in t + [how["q_pos"], how["k_pos"]]:
        x[:, 300:] = bad                       # padding ids
    for x in (t[1], t[2], how["k_pos"]):
        x[1, 280:] = bad                       # past the valid length
    for x in (t[1], t[3]):
        x[:, 155:170] = bad                    # document 1
    q2, k2, v2, dout2 = t
    out, lse = decoder_attention_forward(q2, k2, v2, **how)
    got = decoder_attention_backward(dout2, q2, k2, v2, out, lse, **how)
    keep = torch.tensor([s in (0, 2) for s in sizes], device="cuda")
    how_ref = dict(how, q_pos=how["q_pos"].nan_to_num(0, 0, 0), k_pos=how["k_pos"].nan_to_num(0, 0, 0))
    ref = reference(*(x.nan_to_num(0, 0, 0) for x in (q2, k2, v2)), **how_ref, dout=dout2.nan_to_num(0, 0, 0))
    for n, g, c in zip(("dq", "dk", "dv", "dslopes"), got, clean):
        assert torch.isfinite(g[:, keep]).all(), n
        want, tol = ref[n][:, keep], ref[n + "_tol"][:, keep]
        if n != "dslopes":
            tol = 1.01 * tol + half_step(torch.bfloat16) * want.abs()
        assert ((g[:, keep].double() - want).abs() <= tol + 2 * U * want.abs()).all(), n
        assert not g[:, 300:].any(), n
    assert not got[1][1, 280:].any() and not got[2][1, 280:].any()
    assert not torch.isfinite(got[0][:, 160]).any()
    for _ in range(40):
        again = decoder_attention_backward(dout2, q2, k2, v2, out, lse, **how)
        assert all(torch.equal(x[:, keep], y[:, keep]) for x, y in zip(again, got))


def test_gradients_strides_expanded_and_parts(cuda_device):
    q, k, v, how = make(2, 100, 150, 4, 4, 64, pos=1)
    dout, want = gradients(q, k, v, how)
    qkv = [x.permute(0, 2, 1, 3).contiguous().permute(0, 2, 1, 3) for x in (q, k, v, dout)]
    out, lse = decoder_attention_forward(*qkv[:3], **how)
    got = decoder_attention_backward(qkv[3], *qkv[:3], out, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(want, got))
    one = decoder_attention_backward(dout[:, :1].expand(-1, 100, -1, -1), q, k, v, out, lse, **how)
    two = decoder_attention_backward(dout[:, :1].expand(-1, 100, -1, -1).contiguous(), q, k, v, out, lse, **how)
    assert all(torch.equal(a, b) for a, b in zip(one, two))
    part = decoder_attention_backward(dout, q, k, v, out, lse, **how, need_dkv=False, need_dslopes=False)
    assert torch.equal(part[0], want[0]) and part[1:] == (None, None, None)


def test_gradients_equal_bits_and_graphs(cuda_device):
    q, k, v, how = make(2, 700, 900, 4, 2, 64, pos=2)
    dout = torch.randn_like(q)

    def step():
        out, lse = decoder_attention_forward(q, k, v, **how)
        return (out, *decoder_attention_backward(dout, q, k, v, out, lse, **how))

    first = [t.clone() for t in step()]
    a, b = capture(step), capture(step)
    for run in (a.replay, step, b.replay, a.replay, b.replay):
        assert all(torch.equal(x, y) for x, y in zip(first, run()))
    dout.neg_()
    assert torch.equal(a.replay()[1], step()[1]) and torch.equal(a.replay()[1], -first[1])


def test_autograd(cuda_device):
    """Through autograd: expanded (shared) keys get the sum of their uses, slopes and leaves the sum of
    two calls; only what requires a gradient gets one."""
    q, k, v, how = make(2, 60, 90, 4, 4, 64, pos=2, cap=8.0)
    dout, want = gradients(q, k, v, how)
    leaves = [t.clone().requires_grad_() for t in (q, k, v, how["slopes"])]
    rest = {n: how[n] for n in ("q_pos", "k_pos", "softcap")}
    (decoder_attention(*leaves[:3], slopes=leaves[3], **rest).float() * dout.float()).sum().backward()
    assert all(torch.equal(t.grad, w) for t, w in zip(leaves, want))
    (decoder_attention(*leaves[:3], slopes=leaves[3], **rest).float() * dout.float()).sum().backward()
    assert torch.allclose(leaves[0].grad.float(), 2 * want[0].float())
    ql = q.clone().requires_grad_()
    decoder_attention(ql, k, v, slopes=how["slopes"], **rest).backward(dout)
    assert torch.equal(ql.grad, want[0])
    kl = k[:, :, :1].clone().requires_grad_()
    decoder_attention(q, kl.expand(-1, -1, 4, -1), v[:, :, :1].expand(-1, -1, 4, -1)).backward(dout)
    ks = k[:, :, :1].clone().requires_grad_()
    decoder_attention(q, ks, v[:, :, :1]).backward(dout)
    # the expanded form rounds four gradients to bf16 and their sum, the shared one its sum once
    big = kl.grad.float().abs().max()
    assert (kl.grad.float() - ks.grad.float()).abs().max() <= 6 * half_step(torch.bfloat16) * 2 * big
    with pytest.raises(TypeError, match="bfloat16"):
        decoder_attention(q.half().requires_grad_(), k.half(), v.half())
    with pytest.raises(ValueError, match="q_pos"):
        decoder_attention(q, k, v, slopes=how["slopes"], q_pos=how["q_pos"].clone().requires_grad_(), k_pos=how["k_pos"])
    with torch.no_grad():
        assert decoder_attention(q.half(), k.half(), v.half()).dtype == torch.float16


def test_gradient_against_differences(cuda_device):
    """The gradient of a loss against central differences of the 64-bit definition, along random
    directions: the definition's derivative is the kernels' up to their own bounds (3 % covers the
    bf16 roundings of a sum of about 10^4 terms of either sign at these sizes)."""
    q, k, v, how = make(1, 40, 50, 2, 1, 64, pos=2, cap=6.0)
    dout, grads = gradients(q, k, v, how)
    g = torch.Generator().manual_seed(9)
    base = dict(q=q.double(), k=k.double(), v=v.double(), slopes=how["slopes"].double())

    def loss(x):
        args = dict(how, slopes=x["slopes"])
        return (reference(x["q"], x["k"], x["v"], **args)["out"] * dout.double()).sum().item()

    for name, got in zip(("q", "k", "v", "slopes"), grads):
        d = torch.randn(base[name].shape, generator=g).double().cuda().sign() * got.double().sign()
        up, down = dict(base), dict(base)
        up[name], down[name] = base[name] + 1e-5 * d, base[name] - 1e-5 * d
        want = (loss(up) - loss(down)) / 2e-5
        have = (got.double() * d).sum().item()
        assert abs(want - have) <= 0.03 * got.double().abs().sum().item(), (name, want, have)


def test_python_refusals(cuda_device):
    q, k, v, how = make(2, 20, 30, 4, 2, 64, pos=2)
    out, lse = decoder_attention_forward(q, k, v, **how)
    f = decoder_attention_forward
    for bad in (lambda: f(q.float(), k.float(), v.float()), lambda: f(q, k.half(), v), lambda: f(q, k, v, k_len=torch.ones(2).cuda()),
                lambda: f(q, k, v, q_segment=torch.ones(2, 20).cuda(), k_segment=torch.ones(2, 30).cuda()),
                lambda: f(q, k, v, **dict(how, slopes=how["slopes"].double())), lambda: f(q, k, v, out=out.half()),
                lambda: f(q, k, v, error_flag=torch.zeros(1, device="cuda"))):
        with pytest.raises(TypeError):
            bad()
    seg = torch.zeros(2, 20, dtype=torch.int32, device="cuda")
    for bad in (lambda: f(q[0], k, v), lambda: f(q, k[:1], v[:1]), lambda: f(q, k, v[:, :5]), lambda: f(q[:, :, :3], k, v),
                lambda: f(q[..., :60], k[..., :60], v[..., :60]), lambda: f(q, k, v, slopes=how["slopes"]),
                lambda: f(q, k, v, q_pos=how["q_pos"]), lambda: f(q, k, v, **dict(how, slopes=how["slopes"][:3])),
                lambda: f(q, k, v, **dict(how, k_pos=how["q_pos"])), lambda: f(q, k, v, q_segment=seg),
                lambda: f(q, k, v, q_segment=seg, k_segment=seg), lambda: f(q, k, v, k_len=seg[0]),
                lambda: f(q, k, v, out=out[:, :, :2]), lambda: f(q, k, v, softcap=-1.0), lambda: f(q, k, v, scale=math.inf),
                lambda: f(q, k.cpu(), v)):
        with pytest.raises(ValueError):
            bad()
    b = decoder_attention_backward
    for bad in (lambda: b(out.half(), q, k, v, out, lse, **how), lambda: b(out, q, k, v, out, lse.double(), **how)):
        with pytest.raises(TypeError):
            bad()
    for bad in (lambda: b(out[:, :5], q, k, v, out, lse, **how), lambda: b(out, q, k, v, out, lse[:, :1], **how),
                lambda: b(out, q, k, v, out.transpose(1, 2).contiguous().transpose(1, 2), lse, **how)):
        with pytest.raises(ValueError):
            bad()


def test_wait_limit_flag_stays_clear_and_step_counts(cuda_device):
    """The error flag is only ever set by a wait that gave up."""
    q, k, v, how = make(3, 500, 700, 4, 2, 128, pos=1, k_len=[700, 0, 333])
    flag = torch.zeros(1, dtype=torch.int32, device="cuda")
    out, lse = decoder_attention_forward(q, k, v, **how, error_flag=flag)
    decoder_attention_backward(torch.randn_like(out), q, k, v, out, lse, **how, error_flag=flag)
    assert flag.item() == 0


@pytest.mark.parametrize("rep", [1, 2, 3, 5, 8, 16, 128, 130])
def test_shared_heads_of_every_kind(cuda_device, rep):
    """Heads a key that divide the 128 rows of a tile and ones that do not, more heads than rows."""
    q, k, v, how = make(1, 9, 140, rep, 1, 64, pos=1, slopes="row")
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)


def test_out_that_shares_memory_and_scales_beyond_fp32_are_rejected(cuda_device):
    buf = torch.randn(3, 2, 64, 4, 64, device="cuda").bfloat16()
    q, k, v = buf
    for bad in (lambda: decoder_attention_forward(q, k, v, out=q), lambda: decoder_attention_forward(q, k, v, out=v),
                lambda: decoder_attention_forward(q, k, v, out=buf.view(-1)[64:64 + q.numel()].view(q.shape)),
                lambda: decoder_attention_forward(q, k, v, scale=1e39), lambda: decoder_attention_forward(q, k, v, softcap=2e3)):
        with pytest.raises(ValueError):
            bad()


@pytest.mark.parametrize("cap", [1024.0, 1e-3])
def test_largest_and_small_caps(cuda_device, cap):
    q, k, v, how = make(1, 100, 150, 2, 2, 64, cap=cap)
    check_forward(q, k, v, how, *decoder_attention_forward(q, k, v, **how))
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)


@pytest.mark.parametrize("D,pos,cap", [(64, 2, 0.0), (64, 0, 20.0), (128, 1, 0.0)])
def test_gradients_do_not_see_the_rounding_of_out(cuda_device, D, pos, cap):
    """delta_i = dO_i . O_i is made from a rounded O.  What it is short of, at most r = (h + h) |dO| P |V| (O
    rounded, and made from rounded P), is taken out of dQ and dK again; left over is r times the
    relative error of the correction: P's rounding h, the scores' 2 e and the sums' N u.  Weights that lie on
    few keys, where dS is small beside r."""
    B, Nq, Nk, H, G = 1, 200, 260, 4, 2
    q, k, v, how = make(B, Nq, Nk, H, G, D, pos=pos, cap=cap)
    q = q * 4
    dout, (dq, dk, dv, ds) = gradients(q, k, v, how)
    r = reference(q, k, v, dout=dout, **how)
    h, n = half_step(q.dtype), max(Nq, Nk) * U
    e = score_error(q, k, None, cap, how.get("slopes"), how.get("q_pos"), how.get("k_pos"))
    scale = D ** -0.5
    tol_q, tol_k = torch.zeros_like(r["dq"]), torch.zeros_like(r["dk"])
    for hd in range(H):
        Q, K, V, dO = q[0, :, hd].double(), k[0, :, hd // 2].double(), v[0, :, hd // 2].double(), dout[0, :, hd].double()
        x = scale * Q @ K.T
        t = torch.tanh(x / cap) if cap else 0 * x
        s = cap * t if cap else x
        if pos:
            dist = (how["q_pos"][0].double()[:, None] - how["k_pos"][0].double()[None]).square().sum(-1).sqrt()
            s = s - how["slopes"][hd].double() * dist
        p = torch.softmax(s, 1)
        dp = dO @ V.T
        dS = p * (dp - (p * dp).sum(1, keepdim=True))
        mag = p * (dO.abs() @ V.abs().T)
        short = p * (2 * h * mag.sum(1, keepdim=True))  # before the correction
        off = (h + 2 * e + (D + 16) * U + n) * dS.abs() + (2 * e + (D + 16) * U + n) * mag + (h + 2 * e + n + 16 * U) * short \
            + p * ((2 * e + n + (D + 16) * U) * mag.sum(1, keepdim=True))
        tol_q[0, :, hd] = scale * off @ K.abs()
        tol_k[0, :, hd // 2] += scale * off.T @ Q.abs()
    for got, name, tol in ((dq, "dq", tol_q), (dk, "dk", tol_k)):
        tol = tol + h * (r[name].abs() + tol) + 1e-30
        assert ((got.double() - r[name]).abs() <= tol).all(), name


@pytest.mark.parametrize("B,Nq,Nk,H,G,D,how", [
    (5, 900, 900, 4, 4, 64, dict(pos=2)),                    # 160 tiles of either kind: twelve are cut in two
    (2, 1700, 1600, 6, 6, 128, dict(cap=20.0)),              # 168 and 156: in four
    (3, 1500, 1500, 16, 4, 64, dict(pos=1, slopes="row", k_len=[1500, 700, 0])),
    (1, 2100, 5, 3, 1, 64, dict(pos=2)),                     # nothing to cut for dq, one tile for dk and dv
    (1, 1024, 1100, 2, 2, 64, dict()),                       # fewer tiles than SMs: all are cut
])
def test_gradients_of_tiles_cut_into_parts(cuda_device, B, Nq, Nk, H, G, D, how):
    """The tiles that do not fill the SMs are cut along the other axis and joined."""
    q, k, v, how = make(B, Nq, Nk, H, G, D, **how)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)
    for _ in range(20):
        again = gradients(q, k, v, how)[1]
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("D,B,groups", [(64, 1, False), (128, 1, False), (64, 3, False), (64, 3, True)])
def test_gradients_of_parts_with_masked_values_that_are_no_numbers(cuda_device, D, B, groups):
    """Valid keys that end inside a tile of some part (without groups), groups (tiles then stay whole), keys and
    queries that nothing sees and hold NaN and infinity, in a captured graph too."""
    N, H = 1200, 6
    ids = torch.arange(N) // 170
    ids[1100:] = -1
    q, k, v, how = make(B, N, N, H, H, D, pos=2, segments=(ids, ids) if groups else None, k_len=[950, 1100, 1000][:B])
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)
    q2, k2, v2, dout2 = (t.clone() for t in (q, k, v, dout))
    for t in (q2, k2, v2, dout2) if groups else (k2, v2):
        t[:, 1100:] = float("nan")
    k2[0, 950:], v2[0, 960:] = float("inf"), float("nan")
    out, lse = decoder_attention_forward(q2, k2, v2, **how)
    run = lambda: decoder_attention_backward(dout2, q2, k2, v2, out, lse, **how)  # noqa: E731
    first = [t.clone() for t in run()]
    check_backward(q, k, v, how, dout, first)
    graph = capture(run)
    for grads in [run() for _ in range(10)] + [graph.replay()]:
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(grads, first))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("B,Nq,Nk,H,G,D,how", [
    (1, 1, 1, 1, 1, 128, {}), (2, 1, 70, 8, 1, 64, dict(pos=1)), (3, 2, 333, 12, 3, 72, dict(cap=12.0)),
    (2, 8, 900, 3, 3, 64, dict(pos=2, slopes="row")), (1, 1, 9000, 4, 2, 40, dict(pos=2)), (2, 3, 64, 4, 2, 128, {}),
    (4, 1, 5000, 8, 8, 128, dict(pos=1, k_len=[5000, 0, 1, 4097])), (2, 9, 500, 2, 2, 128, dict(pos=1)),
])
def test_few_rows(cuda_device, dtype, B, Nq, Nk, H, G, D, how):
    q, k, v, how = make(B, Nq, Nk, H, G, D, dtype, **how)
    out, lse = decoder_attention_forward(q, k, v, **how)
    check_forward(q, k, v, how, out, lse)
    for _ in range(10):
        assert all(torch.equal(a, b) for a, b in zip((out, lse), decoder_attention_forward(q, k, v, **how)))


@pytest.mark.parametrize("Nk", [300, 3000])
@pytest.mark.parametrize("D", [64, 128])
def test_few_rows_with_documents_and_values_that_are_no_numbers(cuda_device, D, Nk):
    """Documents of which a query's own lies in one quarter of a tile, a query of none, and NaN and infinity in
    the others' values and past the valid keys."""
    ks = torch.arange(Nk) // 13
    ks[Nk - 100:] = -1
    q, k, v, how = make(2, 4, Nk, 4, 2, D, pos=2, segments=([0, 3, -1, 7], ks), k_len=[Nk, 95])
    want = decoder_attention_forward(q, k, v, **how)
    check_forward(q, k, v, how, *want)
    k2, v2 = k.clone(), v.clone()
    hidden = ~torch.isin(ks, torch.tensor([0, 3, 7])).cuda()
    k2[:, hidden], v2[:, hidden] = float("nan"), float("inf")
    v2[1, 95:] = float("nan")
    for _ in range(10):
        out, lse = decoder_attention_forward(q, k2, v2, **how)
        check_forward(q, k, v, how, out, lse)


@pytest.mark.parametrize("B,Nq,Nk,H,G,D,how", [
    (1, 1024, 1100, 2, 2, 64, dict(k_len=[100])), (1, 1024, 1100, 2, 2, 64, dict(k_len=[0], pos=2)),
    (1, 1000, 1100, 2, 2, 128, dict(k_len=[100], cap=20.0)), (2, 500, 1100, 2, 2, 128, dict(k_len=[0, 500])),
    (1, 300, 900, 6, 2, 64, dict(k_len=[70], pos=1, slopes="row")),   # Q and dO gathered, not by TMA
    (1, 300, 3100, 2, 2, 64, dict()),                                 # 49 tiles of keys in eight parts of seven
    (1, 3100, 200, 2, 1, 64, dict(pos=1)), (1, 3100, 200, 2, 2, 128, dict(k_len=[130])),
])
def test_gradients_of_parts_without_keys(cuda_device, B, Nq, Nk, H, G, D, how):
    """Own tiles cut into parts of which some have nothing to walk: they add zeros, call after call."""
    q, k, v, how = make(B, Nq, Nk, H, G, D, **how)
    dout, grads = gradients(q, k, v, how)
    check_backward(q, k, v, how, dout, grads)
    for _ in range(30):
        again = gradients(q, k, v, how)[1]
        assert all(a is None and b is None or torch.equal(a, b) for a, b in zip(grads, again))


@pytest.mark.parametrize("dtype", [torch.bfloat16, torch.float16])
@pytest.mark.parametrize("Nq", [1, 4, 5, 70])  # on both sides of eight rows
@pytest.mark.parametrize("D,pos,cap,Nk", [(64, 0, 5.0, 200), (64, 2, 0.0, 200), (128, 0, 0.0, 330), (128, 1, 0.0, 20000),
                                          (64, 0, 0.0, 200)])
@pytest.mark.parametrize("bad", [math.inf, -math.inf, math.nan])
def test_values_that_are_seen_and_no_numbers(cuda_device, D, pos, cap, Nk, Nq, dtype, bad):
    """An infinity in a value that a row sees is that infinity in out, a NaN a NaN, in that column and no other:
    in full tiles and in the ragged last one, whatever the number of rows."""
    q, k, v, how = make(1, Nq, Nk, 2, 1, D, dtype, pos=pos, cap=cap)
    if pos:
        how["slopes"] = how["slopes"] / 20  # no weight underflows
    clean = decoder_attention_forward(q, k, v, **how)
    check_forward(q, k, v, how, *clean)
    hit = {5: 3, 17: D - 1, 70: 9, Nk - 1: 12}  # key: column
    v2 = v.clone()
    for key, col in hit.items():
        v2[:, key, :, col] = bad
    cols = torch.zeros(D, dtype=torch.bool, device="cuda")
    cols[list(hit.values())] = True
    out, lse = decoder_attention_forward(q, k, v2, **how)
    assert torch.equal(lse, clean[1])
    assert torch.isnan(out[..., cols]).all() if math.isnan(bad) else (out[..., cols] == bad).all()
    check_forward(q, k, torch.where(cols, torch.zeros_like(v), v), how, torch.where(cols, torch.zeros_like(out), out), lse)


@pytest.mark.parametrize("Nk", [100, 128, 20000])  # key 80 in a ragged tile, in a full one, in the first of many parts
@pytest.mark.parametrize("Nq", [2, 40])
@pytest.mark.parametrize("D", [64, 128])
def test_seen_values_whose_weight_underflows(cuda_device, D, Nq, Nk):
    """A NaN in a seen value is one in out also when its weight is 0 in fp32, and so is one of a query's output gradient
    in dv: as 0 times NaN is in the definition."""
    q, k, v, how = make(1, Nq, Nk, 1, 1, D, pos=1)
    how["slopes"] = how["slopes"] * 0 + 1
    how["k_pos"][:] = 300.0  # 2^-432 beside the last key
    how["q_pos"][:], how["k_pos"][:, -1] = 0.0, 0.0
    v[:, 80, :, 5] = math.nan
    out, lse = decoder_attention_forward(q, k, v, **how)
    assert torch.isnan(out[..., 5]).all() and torch.isfinite(lse).all()
    keep = torch.arange(D, device="cuda") != 5
    assert torch.equal(out[..., keep], v[:, -1:, :, keep].expand(-1, Nq, -1, -1))
    if Nk <= 128:
        v[:, 80, :, 5] = 0.0
        dout = torch.ones_like(q)
        dout[:, 1, :, 3] = math.nan
        dv = decoder_attention_backward(dout, q, k, v, *decoder_attention_forward(q, k, v, **how), **how)[2]
        assert torch.isnan(dv[..., 3]).all() and torch.isfinite(dv[..., :3]).all() and torch.isfinite(dv[..., 4:]).all()


@pytest.mark.parametrize("B,Nq,Nk,H,G,D,how", [
    (2, 900, 900, 4, 4, 64, dict(pos=2)), (1, 400, 700, 4, 2, 128, dict(cap=20.0)),      # one CTA a row tile
    (1, 3, 300, 6, 2, 64, {}), (1, 130, 2000, 3, 3, 128, dict(pos=1, slopes="row")),     # clusters, parts in the backward pass
    (1, 1, 700, 2, 2, 128, {}), (1, 2, 40000, 2, 1, 64, dict(pos=1)),                    # few rows, few and many parts
    (1, 40, 40000, 1, 1, 64, {}), (2, 500, 500, 2, 2, 64, dict(segments=(ids(300, 200), ids(300, 200)), k_len=[500, 400])),
])
def test_waits_that_run_out(cuda_device, B, Nq, Nk, H, G, D, how):
    """With the limit at 0 the kernels' waits give up and return: the flag's bit is set, and every element of the
    results is a NaN or what it should be; the next call is as ever.  Without a flag the NaNs tell."""
    q, k, v, how = make(B, Nq, Nk, H, G, D, **how)
    lib = lib_decoder.lib()
    out, lse = decoder_attention_forward(q, k, v, **how)
    dout, want = gradients(q, k, v, how)
    clean = (out, lse, *(t for t in want if t is not None))
    flags = torch.zeros(2, dtype=torch.int32, device="cuda")
    leaf = q.clone().requires_grad_()
    prev = lib.s4d_decoder_set_wait_limit_ns(0)
    try:
        got = (*decoder_attention_forward(q, k, v, **how, error_flag=flags[:1]),
               *(t for t in decoder_attention_backward(dout, q, k, v, out, lse, **how, error_flag=flags[1:]) if t is not None))
        y = decoder_attention(leaf, k, v, **how)
        y.backward(dout)
    finally:
        lib.s4d_decoder_set_wait_limit_ns(prev)
    torch.cuda.synchronize()
    assert prev == 2_000_000_000 and flags.tolist() == [S4D_FLAG_WAIT_TIMEOUT] * 2
    for a, b in zip(got, clean):
        gone = torch.isnan(a)
        assert gone.any() and torch.equal(a.masked_fill(gone, 0), b.masked_fill(gone, 0))
    assert torch.isnan(y).any() and torch.isnan(leaf.grad).any()
    flags.zero_()
    again = (*decoder_attention_forward(q, k, v, **how, error_flag=flags[:1]),
             *(t for t in decoder_attention_backward(dout, q, k, v, out, lse, **how, error_flag=flags[1:]) if t is not None))
    assert flags.tolist() == [0, 0] and all(torch.equal(a, b) for a, b in zip(again, clean))


def test_caps_that_are_zero_in_fp32_are_rejected(cuda_device):
    """A positive cap that fp32 rounds to 0 means the opposite of no cap: all scores equal."""
    q, k, v, _ = make(1, 5, 9, 2, 1, 64)
    out, lse = decoder_attention_forward(q, k, v)
    for call in (lambda: decoder_attention_forward(q, k, v, softcap=1e-50), lambda: decoder_attention(q, k, v, softcap=1e-50),
                 lambda: decoder_attention_backward(out, q, k, v, out, lse, softcap=1e-50)):
        with pytest.raises(ValueError, match="softcap"):
            call()
    one = decoder_attention_forward(q, k, v, scale=1e-50)[0]  # a scale that small makes them equal
    assert torch.equal(one, decoder_attention_forward(q, k, v, scale=0.0)[0])


@pytest.mark.parametrize("batch,queries", [(0, 5), (2, 0)])
def test_slopes_gradient_of_no_rows_is_written(cuda_device, batch, queries):
    """The C entry's sum over no rows is 0, whatever dslopes held."""
    ds, x, dk, dv = torch.full((6,), 7.0, device="cuda"), *(torch.zeros(4096, device="cuda") for _ in range(3))
    a = x.data_ptr()
    args = lib_decoder.ATTENTION_ARGS.pack(batch, queries, 3, 6, 2, 8, 1, a, a, a, *(1024, 48, 8), *(1024, 16, 8), *(1024, 16, 8), a,
                                           a, a, 0, 0, 1, a, a, 0, 0, 0, 0, 0, 0, 0.5, 0.0, 1, 0, a, 1024, 48, 8, a,
                                           dk.data_ptr(), dv.data_ptr(), ds.data_ptr())
    lib_decoder.check("s4d_attention_backward", lib_decoder.lib().s4d_attention_backward(args, lib_decoder.stream_ptr(0)))
    assert not ds.any()
