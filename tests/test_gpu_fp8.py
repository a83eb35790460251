"""GPU: e4m3 rows, the e4m3 linear layer and the e4m3 (routed) gated MLP against their definitions in 64 bits.

* quantised rows: values and scales must be equal bit for bit (the kernel rounds as exact division does);
* linear: every product of two e4m3 values is exact in fp32, so an output's error is at most that of fp32 sums
  of 128 terms (per K block) and of the K blocks, two roundings of the scales' product and one of the output:
  (128 + blocks + 3) * 2^-23 of the sum of magnitudes (2^-23, not 2^-24: the tensor core may truncate), plus half a
  step of the output type relative to the value;
* gated MLP: an activation within that error of a border between two e4m3 values may round to the other one.
  The error is below 2e-5 of the block's maximum for the K here, an e4m3 step is 2^-4 .. 2^-3 of a value, so at most
  about 1e-3 of the values flip, by 2^-3 each: sqrt(1e-3) * 2^-3 / 2 = 2e-3 of the result (2-norm)."""
import os
import subprocess
import sys
import types

import numpy as np
import pytest
import torch

import exl3_dense
import exl3_fp8
import exl3_grouped_runtime as rt
import exl3_router
import synth

pytestmark = pytest.mark.gpu
LIMIT = 7.0
MLP_REL = 2e-3


def ref_quant(x, pow2=False):
    """(q values, scales) in 64 bits; the scale is a 32-bit number by definition."""
    x = x.double()
    T, K = x.shape
    nb = -(-K // 128)
    xb = torch.nn.functional.pad(x, (0, nb * 128 - K)).view(T, nb, 128)
    amax = xb.abs().amax(-1).clamp(min=2.0 ** -64)
    if pow2:
        s = torch.ldexp(torch.ones_like(amax), torch.frexp(amax).exponent - 10)
        for _ in range(3):
            s = torch.where(s * 448 < amax, 2 * s, s)
    else:
        s = (amax / torch.full_like(amax, 448.0)).float().double()
    v = xb / s[..., None]
    unit = torch.ldexp(torch.ones_like(v), torch.frexp(v.abs()).exponent.clamp(min=-5) - 4)
    return (torch.round(v / unit) * unit).view(T, -1)[:, :K], s


def spread(s, n, k):
    return s.double().repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]


def deq_weight(w, s):
    return w.float().double() * spread(s, w.shape[-2], w.shape[-1])


def deq_rows(x):
    q, s = ref_quant(x)
    return q * s.repeat_interleave(128, 1)[:, :x.shape[1]]


def make_weight(shape, seed, dev):
    g = torch.Generator(device=dev).manual_seed(seed)
    return exl3_fp8.quantize_weight(torch.randn(*shape, generator=g, device=dev) / shape[-1] ** 0.5)


def make_layer(E, d, f, seed, dev):
    L = types.SimpleNamespace(_exl3_intermediate_local=f)
    L.w13_fp8, L.w13_scale = make_weight((E, 2 * f, d), seed, dev)
    L.w2_fp8, L.w2_scale = make_weight((E, d, f), seed + 1, dev)
    return L


def rows(T, K, dtype, dev, seed):
    g = torch.Generator(device=dev).manual_seed(seed)
    x = torch.randn(T, K, generator=g, device=dev)
    x[:, ::97] *= 20
    return x.to(dtype)


def ref_mlp(x, L, e):
    f = L.w2_fp8.shape[2]
    gu = deq_rows(x) @ deq_weight(L.w13_fp8[e], L.w13_scale[e]).t()
    g, u = gu[:, :f].clamp(max=LIMIT), gu[:, f:].clamp(-LIMIT, LIMIT)
    return deq_rows(g * torch.sigmoid(g) * u) @ deq_weight(L.w2_fp8[e], L.w2_scale[e]).t()


def ref_experts(x, ids, w, L):
    out = torch.zeros(x.shape, dtype=torch.float64, device=x.device)
    for e in range(L.w13_fp8.shape[0]):
        t, j = (ids == e).nonzero(as_tuple=True)
        if t.numel():
            out.index_add_(0, t, ref_mlp(x[t], L, e) * w[t, j].double()[:, None])
    return out


def rel(a, b):
    return float((a.double() - b).norm() / b.norm())


# ------------------------------------------------------------------------------------ quantised rows
@pytest.mark.parametrize("pow2", [False, True])
@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("T,K", [(1, 1), (1, 128), (3, 200), (33, 4096), (257, 144), (5, 130), (1000, 1536)])
def test_quantize_rows_is_exact(ext, cuda_device, T, K, dtype, pow2):
    x = rows(T, K, dtype, cuda_device, T + K)
    if T > 2:
        x[1] = 0.0
        x[2, :64] *= 1e-6
    q, s = exl3_fp8.quantize_rows(x, pow2=pow2)
    want_q, want_s = ref_quant(x, pow2)
    assert torch.equal(s.double(), want_s)
    assert torch.equal(q.double(), want_q)


def test_quantize_rows_borders(ext, cuda_device):
    """Quotients on and next to every border between e4m3 values, for scales that divide badly."""
    dev = cuda_device
    v = torch.arange(0, 127, device=dev, dtype=torch.uint8).view(torch.float8_e4m3fn).double()     # 0 .. 448
    mid = (v[1:] + v[:-1]) / 2
    for amax in (448.0, 1.0, 3.1415927, 0.013, 5e4):
        s = float(torch.tensor(amax / 448.0).float())
        x = torch.cat([mid * s, v * s]).float()
        x = torch.cat([x, x.nextafter(torch.zeros_like(x)), x.nextafter(torch.full_like(x, 1e9))]).clamp(max=amax)
        n = -(-x.numel() // 127)
        x = torch.nn.functional.pad(x, (0, n * 127 - x.numel())).view(n, 127)
        x = torch.cat([x, torch.full((n, 1), amax, device=dev)], 1)
        x = torch.cat([x, -x], 0).contiguous()
        q, sc = exl3_fp8.quantize_rows(x)
        want_q, want_s = ref_quant(x)
        assert torch.equal(sc.double(), want_s) and torch.equal(q.double(), want_q)


def test_quantize_rows_strides_and_specials(ext, cuda_device):
    dev = cuda_device
    wide = rows(40, 1000, torch.bfloat16, dev, 1)
    for part in (wide[:, 8:776], wide[:, 3:259], wide[::3, :512]):
        q, s = exl3_fp8.quantize_rows(part)
        want_q, want_s = ref_quant(part)
        assert torch.equal(s.double(), want_s) and torch.equal(q.double(), want_q)
    x = rows(4, 256, torch.float32, dev, 2)
    x[0, 5] = float("nan")
    x[1, 200] = float("inf")
    x[2, 130] = 3e38
    q, s = exl3_fp8.quantize_rows(x)
    deq = q.float() * s.repeat_interleave(128, 1)
    assert torch.isnan(deq[0, :128]).all() and torch.isfinite(deq[0, 128:]).all()
    assert torch.isnan(deq[1, 128:]).all() and torch.isfinite(deq[1, :128]).all()
    assert torch.isfinite(deq[2:]).all()
    q, s = exl3_fp8.quantize_rows(torch.empty(0, 256, device=dev))
    assert q.shape == (0, 256) and s.shape == (0, 2)


# ------------------------------------------------------------------------------------ linear
def check_linear(x, w, ws, out_dtype, got, base=None):
    q, s = ref_quant(x)
    xd = q * s.repeat_interleave(128, 1)[:, :x.shape[1]]
    wd = deq_weight(w, ws)
    want = xd @ wd.t()
    bound = (128 + s.shape[1] + 3) * 2.0 ** -23 * (xd.abs() @ wd.abs().t())
    if base is not None:
        want = want + base.double()
        bound = bound + 2.0 ** -24 * want.abs()
    bound = bound * (1 + torch.finfo(out_dtype).eps) + torch.finfo(out_dtype).eps / 2 * want.abs() + 1e-30
    assert got.dtype == out_dtype and got.shape == want.shape
    assert bool(((got.double() - want).abs() <= bound).all())


@pytest.mark.parametrize("T,N,K", [
    (1, 1, 16), (1, 4096, 4096), (2, 130, 128), (5, 576, 1536), (8, 256, 400), (16, 200, 2064), (17, 384, 256), (31, 129, 144),
    (32, 300, 512), (33, 257, 512), (64, 1024, 1024), (100, 72, 4096), (127, 640, 272), (129, 513, 384), (300, 576, 1024),
    (777, 576, 4096), (1025, 1536, 512)])
def test_linear(ext, cuda_device, T, N, K):
    dev = cuda_device
    w, ws = make_weight((N, K), T + N, dev)
    for i, (dt, odt) in enumerate([(torch.bfloat16, torch.float32), (torch.float16, torch.float16),
                                   (torch.float32, torch.bfloat16)]):
        x = rows(T, K, dt, dev, i)
        check_linear(x, w, ws, odt, exl3_fp8.fp8_linear(x, w, ws, out_dtype=odt))
    assert ext.read_status(dev) == 0


def test_linear_strides_accumulate_and_untouched_rows(ext, cuda_device):
    dev = cuda_device
    T, N, K = 70, 200, 384
    w, ws = make_weight((N, K), 3, dev)
    x = rows(T, 1000, torch.bfloat16, dev, 4)[:, 100:100 + K]
    whole = torch.full((T + 4, N + 8), 7.0, device=dev)
    out = whole[2:2 + T, 4:4 + N]
    base = out.clone()
    exl3_fp8.fp8_linear(x, w, ws, out=out)
    check_linear(x, w, ws, torch.float32, out, base)
    whole[2:2 + T, 4:4 + N] = 7.0
    assert bool((whole == 7.0).all())
    big, bs = make_weight((N, 512), 5, dev)                   # a view of a wider weight: strided rows and scales
    xs = rows(T, 256, torch.float16, dev, 6)
    check_linear(xs, big[:, 256:], bs[:, 2:], torch.float32, exl3_fp8.fp8_linear(xs, big[:, 256:], bs[:, 2:]))


def test_linear_nan_stays_in_its_row(ext, cuda_device):
    dev = cuda_device
    for T in (6, 200):
        w, ws = make_weight((300, 512), 3, dev)
        x = rows(T, 512, torch.float32, dev, 4)
        clean = exl3_fp8.fp8_linear(x, w, ws)
        x[T // 2, 7] = float("inf")
        got = exl3_fp8.fp8_linear(x, w, ws)
        assert torch.isnan(got[T // 2]).all()
        keep = torch.arange(T, device=dev) != T // 2
        assert torch.equal(got[keep], clean[keep])


def test_linear_no_rows(ext, cuda_device):
    w, ws = make_weight((64, 128), 1, cuda_device)
    assert exl3_fp8.fp8_linear(torch.empty(0, 128, device=cuda_device), w, ws).shape == (0, 64)


# ------------------------------------------------------------------------------------ gated MLP and experts
@pytest.mark.parametrize("T,d,f", [(1, 384, 256), (2, 640, 384), (3, 384, 256), (7, 384, 256),
                                   (8, 1280, 384), (16, 384, 256), (17, 384, 256), (32, 384, 256), (33, 384, 256), (128, 384, 256),
                                   (200, 384, 256), (40, 1024, 1024), (130, 1152, 640), (300, 2048, 512)])
def test_mlp(ext, cuda_device, T, d, f):
    dev = cuda_device
    L = make_layer(1, d, f, 11, dev)
    x = rows(T, d, torch.bfloat16, dev, T)
    want = ref_mlp(x, L, 0)
    assert rel(exl3_fp8.fp8_mlp_prefill(x, L, LIMIT), want) <= MLP_REL
    base = torch.randn(T, d, device=dev)
    out = exl3_dense.dense_mlp_prefill(x, L, LIMIT, out=base.clone())
    assert rel(out - base, want) <= MLP_REL + 1e-5
    assert ext.read_status(dev) == 0


@pytest.mark.parametrize("T,E,d,f,k,kind", [
    (1, 1, 128, 128, 1, "uniform"), (1, 288, 512, 256, 8, "uniform"), (3, 8, 256, 384, 8, "uniform"),
    (40, 16, 256, 128, 2, "zipf"), (256, 16, 1024, 512, 4, "uniform"), (300, 5, 384, 256, 3, "zipf"),
    (4, 4, 512, 256, 2, "uniform"), (16, 16, 512, 256, 2, "zipf"), (2100, 8, 256, 128, 2, "zipf"),
    (20, 4, 1024, 512, 2, "uniform"), (90, 3, 1280, 1152, 2, "zipf"), (1000, 8, 256, 256, 2, "skewed"), (5, 1024, 128, 128, 4, "uniform")])
def test_experts(ext, cuda_device, T, E, d, f, k, kind):
    dev = cuda_device
    L = make_layer(E, d, f, 21, dev)
    ids, w = (t.to(dev) for t in (synth.routing_skewed(T, E, k, 5, hot=2) if kind == "skewed"
                                  else synth.routing(kind, T, E, k, seed=5)))
    x = rows(T, d, torch.float16, dev, 8)
    want = ref_experts(x, ids, w, L)
    out = exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT)
    assert rel(out, want) <= MLP_REL
    assert torch.equal(out, exl3_fp8.fp8_prefill(x, ids.int(), w, L, LIMIT))          # bit-repeatable
    half = exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT, out_dtype=torch.bfloat16)
    assert torch.equal(half, out.to(torch.bfloat16))
    assert torch.equal(rt.grouped_prefill(x, ids, w, L, LIMIT), out)
    assert ext.read_status(dev) == 0


def test_experts_unrouted_slots_and_repeated_experts(ext, cuda_device):
    dev = cuda_device
    T, E, d, f, k = 50, 6, 256, 128, 4
    L = make_layer(E, d, f, 31, dev)
    x = rows(T, d, torch.bfloat16, dev, 1)
    ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
    ids[0] = -1                                              # a token without experts
    ids[1, 2:] = 99
    ids[2] = 3                                               # the same expert in every slot
    ids[3:20, 0] = -1
    for wt in (w, w.half(), w.bfloat16()):
        out = exl3_fp8.fp8_prefill(x, ids, wt, L, LIMIT)
        assert rel(out, ref_experts(x, ids, wt, L)) <= MLP_REL
        assert bool((out[0] == 0).all())
    base = torch.randn(T, d, device=dev)
    acc = exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT, out=base.clone())
    assert torch.equal(acc[0], base[0]) and rel(acc - base, ref_experts(x, ids, w, L)) <= MLP_REL + 1e-5
    ids[:] = -1                                              # nothing routed at all
    assert bool((exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT) == 0).all())
    assert exl3_fp8.fp8_prefill(x[:0], ids[:0], w[:0], L, LIMIT).shape == (0, d)


def test_block_from_logits_with_8_bit_layers(ext, cuda_device):
    """The operators together: logits -> routing -> 8-bit experts + 8-bit shared expert; and an 8-bit shared expert
    beside trellis experts."""
    dev = cuda_device
    T, E, d, f = 60, 16, 256, 128
    L, S = make_layer(E, d, f, 41, dev), make_layer(1, d, f, 43, dev)
    x = rows(T, d, torch.bfloat16, dev, 3)
    logits = torch.randn(T, E, device=dev)
    r = exl3_router.LogitsRouter(4, scoring="softmax", n_group=4, topk_group=2, group_top=1)
    out, ids, w = exl3_router.moe_prefill_from_logits(x, logits, r, L, LIMIT, shared=S, return_routing=True)
    assert rel(out, ref_experts(x, ids, w, L) + ref_mlp(x, S, 0)) <= MLP_REL
    trellis = synth.layer_to(synth.make_layer(E, d, f, seed=31, sv_scale=0.05), dev)
    names = []
    mixed = exl3_dense.moe_block_prefill(x, ids, w, trellis, S, LIMIT, stage_hook=names.append)
    alone = rt.grouped_prefill(x, ids, w, trellis, LIMIT)
    assert rel(mixed - alone, ref_mlp(x, S, 0)) <= MLP_REL + 1e-5
    assert names[-2:] == ["shared_fp8_mlp", "end"]


def test_graphed_small_batches_and_the_hidden_state_router(ext, cuda_device):
    import exl3_decode
    dev = cuda_device
    E, d, f, k = 16, 256, 128, 4
    L, S = make_layer(E, d, f, 61, dev), make_layer(1, d, f, 63, dev)
    graphed = exl3_decode.GraphedPrefill(L, LIMIT, k, max_tokens=16)
    for T in (1, 3, 16):
        ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=T))
        x = rows(T, d, torch.bfloat16, dev, T)
        assert rel(graphed(x, ids, w), ref_experts(x, ids, w, L)) <= MLP_REL
    g = torch.Generator(device=dev).manual_seed(7)
    router = exl3_router.NoauxTcRouter(torch.randn(E, d, generator=g, device=dev) / d ** 0.5, topk=k)
    x = rows(50, d, torch.float16, dev, 9)
    out, ids, w = exl3_router.moe_prefill_from_hidden(x, router, L, LIMIT, shared=S, return_routing=True)
    assert rel(out, ref_experts(x, ids, w, L) + ref_mlp(x, S, 0)) <= MLP_REL
    assert ext.read_status(dev) == 0


def test_two_graphs_on_two_streams(ext, cuda_device):
    """Two captured calls share nothing: replayed side by side they give the eager results."""
    dev = cuda_device
    L = make_layer(8, 256, 256, 51, dev)
    xs, outs, graphs, eager = [], [], [], []
    streams = [torch.cuda.Stream() for _ in range(2)]
    for i, T in enumerate((12, 300)):
        ids, w = (t.to(dev) for t in synth.routing("uniform", T, 8, 2, seed=i))
        x = rows(T, 256, torch.bfloat16, dev, i)
        eager.append(exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT))
        torch.cuda.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.stream(streams[i]), torch.cuda.graph(g, stream=streams[i]):
            outs.append(exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT))
        graphs.append(g)
        xs.append((x, ids, w))
    torch.cuda.synchronize()
    for _ in range(5):
        for g, s in zip(graphs, streams):
            with torch.cuda.stream(s):
                g.replay()
    torch.cuda.synchronize()
    for o, e in zip(outs, eager):
        assert torch.equal(o, e)
    assert ext.read_status(dev) == 0


@pytest.mark.parametrize("T", [1, 2, 9, 40, 300])
def test_non_finite_tokens_stay_in_their_rows(ext, cuda_device, T):
    """One value of a token is NaN or inf: its outputs are NaN, every other token's stay as they were."""
    dev = cuda_device
    E, d, f, k = 24, 256, 128, 2
    L, S = make_layer(E, d, f, 71, dev), make_layer(1, d, f, 73, dev)
    ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
    x = rows(T, d, torch.float32, dev, 2)
    bad = T // 2
    keep = torch.arange(T, device=dev) != bad
    calls = [lambda v: exl3_fp8.fp8_linear(v, S.w13_fp8[0], S.w13_scale[0]), lambda v: exl3_fp8.fp8_mlp_prefill(v, S, LIMIT),
             lambda v: exl3_fp8.fp8_prefill(v, ids, w, L, LIMIT)]
    for value in (float("nan"), float("inf"), -float("inf")):
        y = x.clone()
        y[bad, 131] = value
        for call in calls:
            got = call(y)
            assert bool(torch.isnan(got[bad]).all()) and torch.equal(got[keep], call(x)[keep])
    big = x.clone()
    big[bad] *= 1e30                                         # finite: the activations stop at the limit
    assert bool(torch.isfinite(exl3_fp8.fp8_mlp_prefill(big, S, LIMIT)).all())


@pytest.mark.parametrize("T", [1, 2, 9, 40, 300])
def test_output_added_to_the_input(ext, cuda_device, T):
    """x += mlp(x) in place gives what separate tensors give; a linear layer of one token refuses it."""
    dev = cuda_device
    E, d, k = 24, 256, 2
    L, S = make_layer(E, d, 128, 81, dev), make_layer(1, d, 128, 83, dev)
    w, ws = make_weight((d, d), 85, dev)
    ids, rw = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
    x = rows(T, d, torch.float32, dev, 2)
    calls = [lambda v, o: exl3_fp8.fp8_mlp_prefill(v, S, LIMIT, out=o), lambda v, o: exl3_fp8.fp8_prefill(v, ids, rw, L, LIMIT, out=o)]
    if T > 1:
        calls.append(lambda v, o: exl3_fp8.fp8_linear(v, w, ws, out=o))
    else:
        with pytest.raises(RuntimeError, match="overlaps x"):
            exl3_fp8.fp8_linear(x, w, ws, out=x)
    for call in calls:
        want, same = call(x, x.clone()), x.clone()
        assert call(same, same) is same and torch.equal(same, want)


def test_products_give_up_then_recover(ext, cuda_device):
    """With a wait limit of 0 every wait that is not over yet gives up: the tcgen05 product records a timeout, drains what
    it issued and returns; the next calls are right.  Wide and thin tiles, stored and activated outputs."""
    dev = cuda_device
    # nothing waits before a CTA's five stages are full, so a tile needs more than five K blocks: here eight and more
    # (at 400 x 1024 x 1024 K is split into parts of four blocks, and no wait gives up)
    E, d, f, k, T = 4, 1024, 4096, 2, 400
    L = make_layer(E, d, f, 91, dev)
    x = rows(T, d, torch.float16, dev, 3)
    ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
    linear = lambda: exl3_fp8.fp8_linear(x, L.w13_fp8[0], L.w13_scale[0])
    experts = lambda: exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT)
    want = [linear(), experts()]
    ext.read_status(dev)
    for call, right in zip((linear, experts), want):
        prev = ext.set_wait_limit_ns(0)
        try:
            call()
            torch.cuda.synchronize()
        finally:
            ext.set_wait_limit_ns(prev)
        assert ext.read_status(dev) == 1
        assert torch.equal(call(), right) and torch.equal(call(), right)
        torch.cuda.synchronize()
        assert ext.read_status(dev) == 0


def test_offsets_past_32_bits(ext, cuda_device):
    """The last rows of inputs, outputs and workspaces of more than 2^31 elements."""
    dev = cuda_device
    T, N = 70000, 32768                                      # 2.3e9 outputs
    w, ws = make_weight((N, 128), 101, dev)
    x = rows(T, 128, torch.float16, dev, 4)
    out = exl3_fp8.fp8_linear(x, w, ws, out_dtype=torch.float16)
    check_linear(x[-5:], w, ws, torch.float16, out[-5:])
    q, s = exl3_fp8.quantize_rows(out)                       # 2.3e9 inputs
    q1, s1 = exl3_fp8.quantize_rows(out[-5:])
    assert torch.equal(q[-5:].view(torch.uint8), q1.view(torch.uint8)) and torch.equal(s[-5:], s1)
    del out, q, s
    d, f, k = 8192, 128, 4                                   # 2.3e9 values in the routes' rows
    L = make_layer(3, d, f, 103, dev)
    ids, rw = (t.to(dev) for t in synth.routing("uniform", T, 3, k - 1, seed=5))
    ids, rw = torch.cat([ids, ids[:, :1]], 1), torch.cat([rw, rw[:, :1]], 1)
    x = rows(T, d, torch.bfloat16, dev, 6)
    got = exl3_fp8.fp8_prefill(x, ids, rw, L, LIMIT, out_dtype=torch.bfloat16)
    # (half a bf16 step on top: 2^-8)
    assert rel(got[-6:], ref_experts(x[-6:], ids[-6:], rw[-6:], L)) <= MLP_REL + 2.0 ** -8
    assert ext.read_status(dev) == 0


@pytest.mark.parametrize("T", [8, 9, 16, 17])
def test_both_sides_of_the_rule_for_few_tokens(ext, cuda_device, T):
    """9..16 tokens take one path or the other by the weight's shape: long rows (K > 2 N), and square ones."""
    dev = cuda_device
    for N, K in ((100, 1024), (512, 512)):
        w, ws = make_weight((N, K), 111, dev)
        x = rows(T, K, torch.bfloat16, dev, 2)
        check_linear(x, w, ws, torch.bfloat16, exl3_fp8.fp8_linear(x, w, ws, out_dtype=torch.bfloat16))
    for d, f in ((1280, 256), (256, 640), (512, 512)):
        L = make_layer(1, d, f, 113, dev)
        x = rows(T, d, torch.bfloat16, dev, 3)
        assert rel(exl3_fp8.fp8_mlp_prefill(x, L, LIMIT), ref_mlp(x, L, 0)) <= MLP_REL
    assert ext.read_status(dev) == 0


@pytest.mark.parametrize("dtype", [torch.float16, torch.bfloat16])
def test_quantize_rows_non_finite_halves(ext, cuda_device, dtype):
    """16-bit rows with a NaN or inf of either sign in one place of a block: that block has no finite value, the others
    stay exact."""
    dev = cuda_device
    clean = rows(24, 512, dtype, dev, 5)
    want_q, want_s = exl3_fp8.quantize_rows(clean)
    for value in (float("nan"), float("inf"), -float("inf")):
        x = clean.clone()
        for r in range(24):
            x[r, 128 + (r * 53) % 128] = value
        q, s = exl3_fp8.quantize_rows(x)
        deq = q.float() * s.repeat_interleave(128, 1)
        assert bool(torch.isnan(deq[:, 128:256]).all())
        keep = torch.ones(512, dtype=torch.bool, device=dev)
        keep[128:256] = False
        assert torch.equal(q.view(torch.uint8)[:, keep], want_q.view(torch.uint8)[:, keep])
        assert torch.equal(s[:, [0, 2, 3]], want_s[:, [0, 2, 3]])


def _at_16(t):
    """A copy of `t` that starts 16 bytes behind a 32-byte boundary."""
    flat = torch.empty(t.numel() + 64, dtype=torch.uint8, device=t.device)
    start = (16 - flat.data_ptr()) % 32
    view = flat[start:start + t.numel()].view(t.dtype).view(t.shape)
    view.copy_(t)
    assert view.data_ptr() % 32 == 16 and view.is_contiguous()
    return view


@pytest.mark.parametrize("T", [1, 3, 12, 40])
def test_weights_aligned_to_16_bytes(ext, cuda_device, T):
    """Weights cut out of one flat buffer start on 16 bytes, not 32: every path gives the same bits."""
    dev = cuda_device
    E, d, f, k = 24, 384, 256, 2
    for bank in (make_layer(E, d, f, 121, dev), make_layer(1, d, f, 123, dev)):
        n = bank.w13_fp8.shape[0]
        ids, w = (t.to(dev) for t in synth.routing("uniform", T, n, min(k, n), seed=5))
        for names in (("w13_fp8",), ("w2_fp8",), ("w13_fp8", "w2_fp8")):
            moved = types.SimpleNamespace(**vars(bank))
            for name in names:
                setattr(moved, name, _at_16(getattr(bank, name)))
            for dt in (torch.float32, torch.float16, torch.bfloat16):
                x = rows(T, d, dt, dev, 2)
                want = exl3_fp8.fp8_prefill(x, ids, w, bank, LIMIT)
                assert rel(want, ref_experts(x, ids, w, bank)) <= MLP_REL
                assert torch.equal(exl3_fp8.fp8_prefill(x, ids, w, moved, LIMIT), want)
                if n == 1:
                    assert torch.equal(exl3_fp8.fp8_mlp_prefill(x, moved, LIMIT), exl3_fp8.fp8_mlp_prefill(x, bank, LIMIT))
                assert torch.equal(exl3_fp8.fp8_linear(x, moved.w13_fp8[0], bank.w13_scale[0]),
                                   exl3_fp8.fp8_linear(x, bank.w13_fp8[0], bank.w13_scale[0]))
    assert ext.read_status(dev) == 0


@pytest.mark.parametrize("shift", [16, 48, 240])
def test_workspaces_aligned_to_16_bytes(ext, cuda_device, shift):
    """The C calls take a workspace at any multiple of 16 and write nothing past the size they asked for.  Wide tiles with
    activations (whole-sector stores), split products, and the kernels for few tokens."""
    dev, lib = cuda_device, ext.load()
    stream = torch.cuda.current_stream(dev).cuda_stream
    status = ext.status_tensor(dev).data_ptr()

    def shifted(need):
        flat = torch.full((need + 1024,), 85, dtype=torch.uint8, device=dev)
        start = -flat.data_ptr() % 256 + shift
        return flat, start, flat.data_ptr() + start

    for T, d, f, E, k in ((300, 256, 128, 4, 2), (60, 1024, 512, 2, 2), (9, 256, 128, 2, 2)):
        L = make_layer(E, d, f, 131, dev)
        x = rows(T, d, torch.float32, dev, 4)
        ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
        one = types.SimpleNamespace(w13_fp8=L.w13_fp8[:1], w13_scale=L.w13_scale[:1], w2_fp8=L.w2_fp8[:1], w2_scale=L.w2_scale[:1])
        ptrs = [t.data_ptr() for t in (L.w13_fp8, L.w13_scale, L.w2_fp8, L.w2_scale)]
        calls = [(exl3_fp8.fp8_mlp_prefill(x, one, LIMIT), lib.exl3_fp8_mlp_workspace(T, d, f),
                  lambda out, ws, n: lib.exl3_fp8_mlp(x.data_ptr(), 0, T, d, d, *ptrs, f, LIMIT, out, 0, d, 0, ws, n, status,
                                                      stream)),
                 (exl3_fp8.fp8_prefill(x, ids, w, L, LIMIT), lib.exl3_fp8_experts_workspace(T, k, E, d, f),
                  lambda out, ws, n: lib.exl3_fp8_experts(x.data_ptr(), 0, T, d, d, ids.data_ptr(), 1, w.data_ptr(), 0, k, E,
                                                          *ptrs, f, LIMIT, out, 0, d, 0, ws, n, status, stream)),
                 (exl3_fp8.fp8_linear(x, L.w13_fp8[0], L.w13_scale[0]), lib.exl3_fp8_linear_workspace(T, d, 2 * f),
                  lambda out, ws, n: lib.exl3_fp8_linear(x.data_ptr(), 0, T, d, d, ptrs[0], d, ptrs[1], d // 128, 2 * f, out, 0,
                                                         2 * f, 0, ws, n, status, stream))]
        assert w.dtype == torch.float32 and ids.dtype == torch.int64
        for want, need, call in calls:
            flat, start, ws = shifted(need)
            out = torch.empty_like(want)
            assert call(out.data_ptr(), ws, need) == 0, lib.exl3_last_error()
            assert torch.equal(out, want)
            assert bool((flat[:start] == 85).all()) and bool((flat[start + need:] == 85).all())
    assert ext.read_status(dev) == 0


def test_shared_entry_points_take_any_float_type_and_strides(ext, cuda_device):
    """grouped_prefill and its kin take 8-bit layers on the inputs that they take trellis layers on: 64-bit values and
    weights, strided columns, broadcast rows."""
    dev = cuda_device
    T, E, d, f, k = 30, 6, 256, 128, 2
    L, S = make_layer(E, d, f, 141, dev), make_layer(1, d, f, 143, dev)
    ids, w = (t.to(dev) for t in synth.routing("uniform", T, E, k, seed=5))
    x = rows(T, d, torch.float32, dev, 4)
    want = exl3_dense.moe_block_prefill(x, ids, w, L, S, LIMIT)
    assert rel(want, ref_experts(x, ids, w, L) + ref_mlp(x, S, 0)) <= MLP_REL
    for same in (x.double(), x.t().contiguous().t()):
        assert torch.equal(exl3_dense.moe_block_prefill(same, ids, w.double(), L, S, LIMIT), want)
    one = x[:1].expand(T, d)
    assert torch.equal(exl3_dense.moe_block_prefill(one, ids, w, L, S, LIMIT),
                       exl3_dense.moe_block_prefill(one.contiguous(), ids, w, L, S, LIMIT))


def test_a_capture_as_the_first_call_keeps_the_status_word(ext, cuda_device):
    """In a process whose first call is captured: the word exists, zeroed, outside the graph, and a replay does not reset
    what an earlier launch recorded."""
    code = """
import sys
sys.path.insert(0, {pkg!r})
import torch, b200_ext, exl3_fp8
dev = torch.device("cuda", 0)
w, ws = exl3_fp8.quantize_weight(torch.randn(256, 256, generator=torch.Generator().manual_seed(1)))
w, ws, x = w.to(dev), ws.to(dev), torch.ones(40, 256, device=dev)
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    out = exl3_fp8.fp8_linear(x, w, ws)
torch.cuda.synchronize()
assert b200_ext.read_status(dev) == 0
b200_ext.status_tensor(dev).fill_(1)
graph.replay()
torch.cuda.synchronize()
assert b200_ext.read_status(dev) == 1, "the replay reset the word"
graph.replay()
assert torch.equal(out, exl3_fp8.fp8_linear(x, w, ws)) and b200_ext.read_status(dev) == 0
"""
    pkg = os.path.dirname(os.path.abspath(exl3_fp8.__file__))
    r = subprocess.run([sys.executable, "-c", code.format(pkg=pkg)], capture_output=True, text=True, timeout=120)
    assert r.returncode == 0, r.stderr[-2000:]
