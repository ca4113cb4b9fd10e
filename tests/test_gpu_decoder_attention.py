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
from sparse4d_tt_b200 import decoder_attention_forward
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
def test_values_behind_masks_do_not_reach_out(cuda_device, bad, Nq):
    """Keys past the valid length, padding and another document hold infinities and NaNs: the rows that do
    not see them are bit-equal to the ones without; the rows that do are not numbers."""
    sizes = ids(150, 60, 90, -20)
    qid = [sizes[i * len(sizes) // Nq] for i in range(Nq)]
    q, k, v, how = make(2, Nq, len(sizes), 4, 2, 64, segments=(qid, sizes), k_len=[320, 280], pos=2, cap=20.0)
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
