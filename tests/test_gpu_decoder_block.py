"""The decoder operators together: a training block (norm, attention with a learned distance bias over
groups, residual, norm) against the same block in 64 bits, as an eager step and as a captured one; and
the decoder head with its attention on decoder_attention_forward."""
import math

import pytest
import torch
import torch.nn.functional as F

from helpers import pcc
from oracle import head_torch as oh
from sparse4d_tt_b200 import _lib_decoder as lib_decoder
from sparse4d_tt_b200 import (decoder_attention, decoder_attention_backward, decoder_attention_forward, decoder_norm,
                              decoder_norm_backward, decoder_norm_forward, ops)
from sparse4d_tt_b200 import synthetic as syn
from sparse4d_tt_b200.graph import capture
from sparse4d_tt_b200.head import HeadGraph, Sparse4DHead, preprocess_head_parameters

pytestmark = pytest.mark.gpu

B, N, H, D = 2, 230, 4, 64
E = H * D


def block_inputs():
    g = torch.Generator().manual_seed(11)
    r = lambda *s: torch.randn(*s, generator=g)  # noqa: E731
    p = {"w1": 1 + 0.2 * r(E), "b1": 0.1 * r(E), "wqkv": r(3 * E, E) / math.sqrt(E), "wo": r(E, E) / math.sqrt(E),
         "slopes": 0.05 + 0.1 * torch.rand(H, generator=g), "w2": 1 + 0.2 * r(E), "b2": 0.1 * r(E)}
    x, dy = r(B, N, E), r(B, N, E)
    pos = torch.rand(B, N, 2, generator=g) * 40
    group = torch.tensor([0] * 150 + [1] * 40 + [2] * 30 + [-1] * 10, dtype=torch.int32).expand(B, -1).contiguous()
    return {k: v.cuda() for k, v in p.items()}, x.cuda(), dy.cuda(), pos.cuda(), group.cuda()


def block(p, x, pos, group):
    y = decoder_norm(x, p["w1"], p["b1"])
    q, k, v = F.linear(y, p["wqkv"]).bfloat16().view(B, N, 3, H, D).unbind(2)
    o = decoder_attention(q, k, v, softcap=15.0, slopes=p["slopes"], q_pos=pos, k_pos=pos, q_segment=group,
                          k_segment=group)
    return decoder_norm(x + F.linear(o.float().reshape(B, N, E), p["wo"]), p["w2"], p["b2"])


def block64(p, x, pos, group):
    y = F.layer_norm(x, (E,), p["w1"], p["b1"], 1e-5)
    q, k, v = (t.transpose(1, 2) for t in F.linear(y, p["wqkv"]).view(B, N, 3, H, D).unbind(2))
    s = 15.0 * torch.tanh(q @ k.transpose(-1, -2) / math.sqrt(D) / 15.0)
    # positions have no gradient, and a root's derivative at 0 is none either
    dist = (pos[:, :, None] - pos[:, None]).square().sum(-1).sqrt()
    s = s - p["slopes"][None, :, None, None] * dist[:, None]
    ok = ((group[:, :, None] == group[:, None]) & (group[:, :, None] >= 0))[:, None]
    w = torch.where(ok.any(-1, keepdim=True), torch.softmax(s.masked_fill(~ok, -1e300), -1), torch.zeros_like(s))
    o = (w @ v).transpose(1, 2).reshape(B, N, E)
    return F.layer_norm(x + F.linear(o, p["wo"]), (E,), p["w2"], p["b2"], 1e-5)


def test_block_trains_like_its_64_bit_form(cuda_device):
    """Up to six bf16 roundings (q, k, v, P, out, dS) of at most 2^-8 of a norm each lie behind every
    gradient: 2.4e-2 relative in the 2-norm."""
    p, x, dy, pos, group = block_inputs()
    leaves = {k: v.clone().requires_grad_() for k, v in p.items()}
    xl = x.clone().requires_grad_()
    out = block(leaves, xl, pos, group)
    out.backward(dy)
    l64 = {k: v.double().requires_grad_() for k, v in p.items()}
    x64 = x.double().requires_grad_()
    ref = block64(l64, x64, pos.double(), group)
    ref.backward(dy.double())
    err = lambda a, b: ((a.double() - b).norm() / b.norm()).item()  # noqa: E731
    assert err(out.detach(), ref.detach()) <= 2.4e-2
    assert err(xl.grad, x64.grad) <= 2.4e-2
    for k in p:
        assert err(leaves[k].grad, l64[k].grad) <= 2.4e-2, (k, err(leaves[k].grad, l64[k].grad))


def test_block_step_captured(cuda_device):
    """A whole step (forward and gradients) in a CUDA graph equals the eager one bit for bit, replay after
    replay, with new data in its inputs.  No eager graph of the same leaves is alive while it is captured."""
    p, x, dy, pos, group = block_inputs()

    def step():
        leaves = {k: v.detach().requires_grad_() for k, v in p.items()}
        xl = x.detach().requires_grad_()
        out = block(leaves, xl, pos, group)
        return (out.detach(), *torch.autograd.grad(out, [xl, *leaves.values()], dy))

    call = capture(step)
    for _ in range(2):
        want = [t.clone() for t in step()]
        got = call.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(want, got))
        x.copy_(x.flip(1))
        dy.neg_()


# ---- the head ------------------------------------------------------------------------------------------


@pytest.fixture(scope="module")
def head_case():
    head = oh.build_head(42)
    cfg = syn.DFAConfig(bs=2)
    ins = syn.make_inputs(cfg, 9, feature_dtype=torch.bfloat16)
    d = torch.device("cuda:0")
    packed = ops.pack_feature_maps([m.to(d) for m in ins.feature_maps], dtype=torch.bfloat16)
    return preprocess_head_parameters(head), cfg, ins, packed


BASE = {"FEATURE_DTYPE": torch.bfloat16, "MATMUL_PRECISION": "tf32", "ATTENTION_DTYPE": torch.bfloat16}


def run(gh, case, **kw):
    _, cfg, ins, packed = case
    d = torch.device("cuda:0")
    anchor = kw.pop("anchor", ins.anchor.to(d))
    return gh.forward(packed, ins.projection_mat.to(d), ins.image_wh.to(d), cfg.spatial_shapes, cfg.bs, anchor=anchor,
                      **kw)["prediction"]


def steps_agree(a, b, anchor, least):
    prev_a, prev_b = anchor, anchor
    for x, y in zip(a, b):
        assert pcc((x - prev_a).cpu(), (y - prev_b).cpu()) >= least
        prev_a, prev_b = x, y


def test_head_on_the_decoder_kernel_follows_sdpa(cuda_device, head_case):
    """Without bias and masks the two kernels compute the same attention up to bf16 roundings: the decoders'
    refinement steps agree as the bf16 head does with the fp32 oracle."""
    params = head_case[0]
    a = run(Sparse4DHead("cuda:0", params, BASE), head_case)
    b = run(Sparse4DHead("cuda:0", params, dict(BASE, ATTENTION_KERNEL="decoder")), head_case)
    steps_agree(a, b, head_case[2].anchor.cuda(), 0.999)


def test_head_attention_has_the_gradients_of_sdpa(cuda_device, head_case):
    """The attention layer's gradients in its input and in the value, on either kernel: both round P, dS and the
    results to bf16 a few times, 2^-8 of a norm each.  What has no gradient is refused, not left out."""
    params = head_case[0]
    heads = [Sparse4DHead("cuda:0", params, dict(BASE, ATTENTION_KERNEL=kind)) for kind in ("sdpa", "decoder")]
    layer = heads[0].operation_order.index("gnn")
    g = torch.Generator().manual_seed(4)
    query, value, dout = (torch.randn(2, 300, n, generator=g).cuda() for n in (512, 512, 256))
    anchor = torch.randn(2, 300, 11, generator=g).cuda()
    got = []
    for gh in heads:
        x, v = query.clone().requires_grad_(), value.clone().requires_grad_()
        out = gh._attention(gh.layers[layer], x, v, anchor, None)
        got.append(torch.autograd.grad(out, (x, v), dout))
    for a, b in zip(*got):
        assert b.norm() > 0 and (a - b).norm() <= 2.4e-2 * a.norm()
    biased = Sparse4DHead("cuda:0", params, dict(BASE, ATTENTION_KERNEL="decoder", ATTENTION_DISTANCE_SLOPES=[0.1] * 8))
    with pytest.raises(ValueError, match="no gradient"):
        biased._attention(biased.layers[layer], query, value, anchor.clone().requires_grad_(), None)
    half = Sparse4DHead("cuda:0", params, dict(BASE, ATTENTION_KERNEL="decoder", ATTENTION_DTYPE=torch.float16))
    with pytest.raises(TypeError, match="bfloat16"):
        half._attention(half.layers[layer], query.clone().requires_grad_(), value, anchor, None)


class PlainHead(Sparse4DHead):
    """The head with its attention written out in fp32 on the same rounded q, k and v."""

    def _attention(self, p, query, value, anchor, group):
        bs, n, e = query.shape
        heads = p["num_heads"]
        v_in = query if value is None else value
        w, b = p["in_proj_weight"].chunk(3, dim=0), p["in_proj_bias"].chunk(3, dim=0)
        q, k, v = (F.linear(t, w[i], b[i]).view(bs, n, heads, -1).transpose(1, 2).bfloat16().float()
                   for i, t in enumerate((query, query, v_in)))
        s = q @ k.transpose(-1, -2) * (e // heads) ** -0.5
        s = self.attention_softcap * torch.tanh(s / self.attention_softcap)
        xy = anchor[..., :2]
        s = s - self.attention_slopes[None, :, None, None] * (xy[:, :, None] - xy[:, None]).norm(dim=-1)[:, None]
        ok = (group[:, :, None] == group[:, None])[:, None]
        o = (torch.softmax(s.masked_fill(~ok, -math.inf), -1) @ v).transpose(1, 2).reshape(bs, n, e)
        return F.linear(query + F.linear(o, p["out_proj_weight"], p["out_proj_bias"]), self.fc_after)


def test_head_with_bias_cap_and_groups(cuda_device, head_case):
    params, cfg, ins, packed = head_case
    d = torch.device("cuda:0")
    conf = dict(BASE, ATTENTION_KERNEL="decoder", ATTENTION_DISTANCE_SLOPES=[0.2 * 2.0 ** -i for i in range(8)],
                ATTENTION_SOFTCAP=20.0)
    group = (torch.arange(900) >= 700).int().expand(cfg.bs, -1).contiguous().cuda()
    gh = Sparse4DHead("cuda:0", params, conf)
    a = [t.clone() for t in run(gh, head_case, instance_group=group)]
    steps_agree(a, run(PlainHead("cuda:0", params, conf), head_case, instance_group=group), ins.anchor.cuda(), 0.999)
    # one group's anchors do not reach the other's predictions, and do reach their own
    moved = ins.anchor.cuda().clone()
    moved[:, 700:, :3] += 3.0
    b = run(gh, head_case, instance_group=group, anchor=moved)
    assert all(torch.equal(x[:, :700], y[:, :700]) for x, y in zip(a, b))
    assert not torch.equal(a[-1][:, 700:], b[-1][:, 700:])
    graph = HeadGraph(gh, cfg.bs, cfg.spatial_shapes, instance_group=group)
    out = graph.run(packed[0], ins.projection_mat.to(d), ins.image_wh.to(d), ins.anchor.to(d), group)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(out["prediction"], a))


def test_head_option_checks(cuda_device, head_case):
    params = head_case[0]
    for bad in ({"ATTENTION_KERNEL": "flash"}, {"ATTENTION_KERNEL": "decoder", "ATTENTION_DTYPE": torch.float32},
                {"ATTENTION_SOFTCAP": 5.0}, {"ATTENTION_DISTANCE_SLOPES": [0.1] * 8}):
        with pytest.raises(ValueError):
            Sparse4DHead("cuda:0", params, dict(BASE, **bad))
    with pytest.raises(ValueError, match="instance_group"):
        run(Sparse4DHead("cuda:0", params, BASE), head_case,
            instance_group=torch.zeros(2, 900, dtype=torch.int32, device="cuda"))


def test_calls_module_and_python_path_agree(cuda_device, monkeypatch):
    """What the calls module takes, and what it leaves to the Python path, gives the same bits; what it cannot
    take it leaves."""
    g = torch.Generator().manual_seed(5)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    x, dy, w, b = r(3, 40, 96), r(3, 40, 96), r(96), r(96)
    q, k, v = r(2, 30, 4, 64).bfloat16(), r(2, 90, 2, 64).bfloat16(), r(2, 90, 2, 64).bfloat16()
    how = dict(softcap=9.0, slopes=torch.rand(4, generator=g).cuda(), q_pos=r(2, 30, 2), k_pos=r(2, 90, 2),
               q_segment=torch.randint(-1, 3, (2, 30), generator=g).int().cuda(),
               k_segment=torch.randint(-1, 3, (2, 90), generator=g).int().cuda(),
               k_len=torch.tensor([90, 50], dtype=torch.int32).cuda())
    long = r(1, 1, 8, 128).bfloat16(), r(1, 20000, 1, 128).bfloat16(), r(1, 20000, 1, 128).bfloat16()
    row = dict(how, slopes=torch.rand(2, 30, 4, generator=g).cuda())

    def everything():
        out = []
        for t, p in ((x, (w, b)), (x.half(), (w, None)), (x.bfloat16(), (w.bfloat16(), b.bfloat16())), (x, (None, None)),
                     (x[:, :0], (w, b)), (x[0, 0], (w, b))):
            y, mean, rstd = decoder_norm_forward(t, *p)
            d = dy.to(t.dtype)[:, :t.shape[1]] if t.dim() == 3 else dy[0, 0]
            out += [y, mean, rstd, *decoder_norm_backward(d.contiguous(), t, p[0], mean, rstd),
                    *decoder_norm_backward(d.contiguous(), t, p[0], mean, rstd, need_dx=False, need_dbias=False)]
        for a in ((q, k, v), long, (q[:0], k[:0], v[:0]), (q.half(), k.half(), v.half())):
            out += decoder_attention_forward(*a)
        for kw in (how, dict(row, scale=0.5), {}, dict(k_len=how["k_len"])):
            o, lse = decoder_attention_forward(q, k, v, **kw)
            out += [o, lse, *decoder_attention_backward(o, q, k, v, o, lse, **kw),
                    *decoder_attention_backward(o.transpose(1, 2).contiguous().transpose(1, 2), q, k, v, o, lse, **kw,
                                                need_dkv=False, need_dslopes=False)]
        return out

    class Leaves:
        def __getattr__(self, name):
            return lambda *a: None

    taken = []

    class Counts:
        def __getattr__(self, name):
            def call(*a):
                done = getattr(calls, name)(*a)
                taken.append(done is not None)
                return done
            return call

    calls = lib_decoder.calls()
    monkeypatch.setattr(lib_decoder, "_calls", Counts())
    first = everything()
    assert all(taken) and len(taken) == 34
    monkeypatch.setattr(lib_decoder, "_calls", Leaves())
    for a, b_ in zip(first, everything(), strict=True):
        assert (a is None) == (b_ is None)
        if a is not None:
            assert a.shape == b_.shape and a.dtype == b_.dtype and a.is_contiguous() and torch.equal(a, b_)
    monkeypatch.setattr(lib_decoder, "_calls", calls)
    c = calls
    for bad in (lambda: c.norm_forward(x.transpose(0, 1), w, b, 1e-5), lambda: c.norm_forward(x, w[:5], b, 1e-5),
                lambda: c.norm_forward(x, w, b.half(), 1e-5), lambda: c.norm_forward(x.double(), None, None, 1e-5),
                lambda: c.norm_forward(x, w.cpu(), b, 1e-5), lambda: c.norm_forward(x, w, b, float("nan")),
                lambda: c.norm_backward(dy[:, :5], x, w, x[..., 0].contiguous(), x[..., 0].contiguous(), True, True, True),
                lambda: c.norm_backward(dy, x, w, x[..., 0], x[..., 0], True, True, True),
                lambda: c.attention_forward(q, k, v.half(), None, 0.0, *[None] * 6),
                lambda: c.attention_forward(q[..., ::2], k[..., ::2], v[..., ::2], None, 0.0, *[None] * 6),
                lambda: c.attention_forward(q, k, v, None, 0.0, how["slopes"], *[None] * 5),
                lambda: c.attention_forward(q, k, v, None, 0.0, None, how["q_pos"], *[None] * 4),
                lambda: c.attention_forward(q, k, v, None, 0.0, how["slopes"], how["q_pos"], how["q_pos"], *[None] * 3),
                lambda: c.attention_forward(q, k, v, None, 0.0, None, None, None, how["q_segment"], None, None),
                lambda: c.attention_forward(q, k, v, None, 5e3, *[None] * 6),
                lambda: c.attention_forward(q, k, v, q, 0.0, *[None] * 6),
                lambda: c.attention_backward(q, q, k, v, q, x, None, 0.0, *[None] * 6, True, True),
                lambda: c.attention_backward(q.half(), q, k, v, q, x, None, 0.0, *[None] * 6, True, True),
                lambda: c.attention_backward(q, q, k, v, q, None, None, 0.0, *[None] * 6, True, True),
                lambda: c.attention_backward(q, q, k, v)):
        assert bad() is None


def test_views_that_stand_for_the_negative_of_their_memory(cuda_device):
    """The imaginary part of a conjugate is such a view; every argument may be one, and an out may not."""
    g = torch.Generator().manual_seed(8)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    neg = lambda t: torch.complex(t * 0, -t).conj().imag if t.dtype == torch.float32 else torch._neg_view(-t)  # noqa: E731
    assert neg(r(3)).is_neg()
    q, k, v, dout = (r(1, n, 2, 64).bfloat16() for n in (20, 30, 30, 20))
    how = dict(slopes=r(2).abs(), q_pos=r(1, 20, 2), k_pos=r(1, 30, 2))
    out, lse = decoder_attention_forward(q, k, v, **how)
    grads = decoder_attention_backward(dout, q, k, v, out, lse, **how)
    nhow = {n: neg(t) for n, t in how.items()}
    nout, nlse = decoder_attention_forward(neg(q), neg(k), neg(v), **nhow)
    assert torch.equal(nout, out) and torch.equal(nlse, lse)
    got = decoder_attention_backward(neg(dout), neg(q), neg(k), neg(v), neg(out), torch._neg_view(-lse), **nhow)
    assert all(torch.equal(a, b) for a, b in zip(got, grads))
    with pytest.raises(ValueError, match="out"):
        decoder_attention_forward(q, k, v, out=torch._neg_view(out))
    for width in (1, 24):
        x, dy, w, b = r(7, width), r(7, width), r(width), r(width)
        y, mean, rstd = decoder_norm_forward(x, w, b)
        want = decoder_norm_backward(dy, x, w, mean, rstd)
        flat = lambda t: torch._neg_view(-t)  # noqa: E731
        for f in (neg, flat):
            ny = decoder_norm_forward(f(x), flat(w), flat(b))
            assert all(torch.equal(a, c) for a, c in zip(ny, (y, mean, rstd)))
            got = decoder_norm_backward(f(dy), f(x), flat(w), flat(mean), flat(rstd))
            assert all(torch.equal(a, c) for a, c in zip(got, want))
        with pytest.raises(ValueError, match="out"):
            decoder_norm_forward(x, out=flat(y))


def test_needs_that_have_no_truth_value(cuda_device):
    """What Python refuses to take for true or false is refused as Python does it."""
    x = torch.randn(6, 32, device="cuda")
    _, mean, rstd = decoder_norm_forward(x)
    q = torch.randn(1, 6, 2, 64, device="cuda").bfloat16()
    out, lse = decoder_attention_forward(q, q, q)
    pos = dict(slopes=torch.ones(2, device="cuda"), q_pos=torch.zeros(1, 6, 1, device="cuda"),
               k_pos=torch.zeros(1, 6, 1, device="cuda"))
    two = torch.ones(2)
    for call in (lambda: decoder_norm_backward(x, x, None, mean, rstd, need_dx=two),
                 lambda: decoder_norm_backward(x, x, None, mean, rstd, need_dbias=two),
                 lambda: decoder_attention_backward(q, q, q, q, out, lse, need_dkv=two),
                 lambda: decoder_attention_backward(q, q, q, q, out, lse, need_dslopes=two, **pos)):
        with pytest.raises(RuntimeError, match="ambiguous"):
            call()
    assert decoder_norm_backward(x, x, None, mean, rstd, need_dx=0, need_dweight=torch.ones(1))[0] is None


def test_head_graph_over_other_groups(cuda_device, head_case):
    """A captured pass reads the groups that it is handed, as an eager pass on them does."""
    params, cfg, ins, packed = head_case
    d = torch.device("cuda:0")
    gh = Sparse4DHead("cuda:0", params, dict(BASE, ATTENTION_KERNEL="decoder", ATTENTION_DISTANCE_SLOPES=[0.1] * 8))
    groups = [(torch.arange(900) >= at).int().expand(cfg.bs, -1).contiguous().cuda() for at in (900, 600, 128)]
    graph = HeadGraph(gh, cfg.bs, cfg.spatial_shapes, instance_group=groups[0])
    feed = (packed[0], ins.projection_mat.to(d), ins.image_wh.to(d), ins.anchor.to(d))
    seen = []
    for group in groups + groups[1:2]:
        got = [t.clone() for t in graph.run(*feed, group)["prediction"]]
        assert all(torch.equal(x, y) for x, y in zip(got, run(gh, head_case, instance_group=group)))
        seen.append(got[-1])
    assert torch.equal(seen[1], seen[3]) and not torch.equal(seen[0], seen[1]) and not torch.equal(seen[1], seen[2])


def test_two_threads_and_streams_at_once(cuda_device):
    """Calls from two host threads on two streams, each with launches of clusters (few rows, cut tiles) and without,
    give the bits that they give alone."""
    import threading

    g = torch.Generator().manual_seed(3)
    r = lambda *s: torch.randn(*s, generator=g).cuda()  # noqa: E731
    sets = []
    for n, keys, dim in ((2, 4000, 64), (900, 900, 64), (1, 9000, 128), (700, 1100, 128)):
        q, k, v = r(1, n, 4, dim).bfloat16(), r(1, keys, 2, dim).bfloat16(), r(1, keys, 2, dim).bfloat16()
        sets.append((q, k, v, dict(slopes=r(4).abs() / 8, q_pos=r(1, n, 2), k_pos=r(1, keys, 2))))
    x, w, b = r(3000, 300), r(300), r(300)

    def work(order):
        out = {}
        for i in order:
            q, k, v, how = sets[i]
            o, lse = decoder_attention_forward(q, k, v, **how)
            out[i] = (o, lse, *decoder_attention_backward(o, q, k, v, o, lse, **how))
            y, mean, rstd = decoder_norm_forward(x, w, b)
            out[i] += (y, *decoder_norm_backward(y, x, w, mean, rstd))
        return out

    want = work(range(4))
    torch.cuda.synchronize()
    results, errors = [], []

    def thread(order):
        try:
            with torch.cuda.stream(torch.cuda.Stream()):
                for _ in range(25):
                    results.append(work(order))
                torch.cuda.current_stream().synchronize()
        except Exception as e:  # noqa: BLE001
            errors.append(e)

    threads = [threading.Thread(target=thread, args=(o,)) for o in ((0, 1, 2, 3), (3, 0, 2, 1))]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert not errors and len(results) == 50
    for got in results:
        assert all(torch.equal(a, c) for i in range(4) for a, c in zip(got[i], want[i]))
