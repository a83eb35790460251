"""GPU: routing from logits against the definition in 64 bits.

ids must be equal everywhere: the kernel ranks as exact arithmetic does (no case here has two 64-bit scores
closer than their own rounding).  Weights: a sigmoid or softmax in fp32 is a few roundings and at most 32 terms
of a sum, under 2^-18 relative (expf within 2 units, a sum over E / 32 + 5 terms, two divisions, one product;
softmax also rounds l - max, at most 2^-24 * 100 of the exponent here)."""
import numpy as np
import pytest
import torch

import exl3_router
import synth

pytestmark = pytest.mark.gpu
W_REL = 2.0 ** -17


@np.errstate(over="ignore", invalid="ignore")
def reference(logits, bias, k, softmax, n_group, topk_group, group_top, norm, scale):
    """The definition, one token at a time, in Python floats (64 bits)."""
    l = logits.double().cpu().numpy()
    b = None if bias is None else bias.double().cpu().numpy()
    T, E = l.shape
    ids, ws = np.full((T, k), -1, np.int64), np.zeros((T, k))
    per = E // n_group
    for t in range(T):
        ok = l[t] > -np.inf                                  # False for NaN
        s = np.zeros(E)
        if softmax and ok.any():
            e = np.where(l[t][ok] == l[t][ok].max(), 1.0, np.exp(l[t][ok] - l[t][ok].max()))
            s[ok] = e / e.sum()
        elif ok.any():
            s[ok] = 1.0 / (1.0 + np.exp(-l[t][ok]))
        c = np.where(ok, (l[t] if b is None else s + b), -np.inf)
        g = np.where(ok, s if b is None else s + b, -np.inf)
        if topk_group < n_group:
            gs = [np.sort(g[i * per:(i + 1) * per])[::-1][:group_top].sum() for i in range(n_group)]
            kept = sorted(range(n_group), key=lambda i: (-gs[i], i))[:topk_group]
            c = np.where(np.isin(np.arange(E) // per, kept), c, -np.inf)
        order = sorted((e for e in range(E) if c[e] > -np.inf), key=lambda e: (-c[e], e))[:k]
        ids[t, :len(order)] = order
        w = s[order]
        ws[t, :len(order)] = (w / (w.sum() + 1e-20) if norm else w) * scale
    return ids, ws


def check(logits, bias, k, scoring="sigmoid", n_group=1, topk_group=1, group_top=2, norm=True, scale=2.5):
    r = exl3_router.LogitsRouter(k, scoring=scoring, bias=bias, n_group=n_group, topk_group=topk_group,
                                 group_top=group_top, norm=norm, scale=scale)
    ids, w = r.route(logits)
    want_ids, want_w = reference(logits, bias, k, scoring == "softmax", n_group, topk_group, group_top, norm, scale)
    assert np.array_equal(ids.cpu().numpy(), want_ids)
    got = w.double().cpu().numpy()
    assert np.all(np.abs(got - want_w) <= W_REL * np.abs(want_w) + 1e-37)
    return ids, w


def _logits(T, E, dtype, dev, seed, std=1.5):
    g = torch.Generator(device=dev).manual_seed(seed)
    return (torch.randn(T, E, generator=g, device=dev) * std).to(dtype), 0.1 * torch.randn(E, generator=g, device=dev)


@pytest.mark.parametrize("dtype", [torch.float32, torch.float16, torch.bfloat16])
@pytest.mark.parametrize("scoring", ["sigmoid", "softmax"])
@pytest.mark.parametrize("T,E,k,G,keep,gtop,with_bias", [
    (1, 1, 1, 1, 1, 1, True), (3, 7, 7, 1, 1, 1, True), (65, 33, 4, 1, 1, 2, False), (130, 288, 8, 1, 1, 2, True),
    (40, 256, 8, 8, 4, 2, True), (40, 256, 8, 8, 3, 1, False), (33, 90, 6, 5, 2, 2, False), (20, 320, 16, 32, 7, 2, True),
    (17, 1024, 32, 4, 2, 2, True), (9, 500, 10, 1, 1, 2, True), (64, 62, 31, 31, 31, 2, True)])
def test_matches_the_definition(ext, cuda_device, T, E, k, G, keep, gtop, with_bias, scoring, dtype):
    logits, bias = _logits(T, E, dtype, cuda_device, seed=T + E)
    check(logits, bias if with_bias else None, k, scoring, G, keep, gtop, norm=T % 2 == 1)


@pytest.mark.parametrize("G,keep", [(1, 1), (4, 2)])
def test_masked_logits_and_empty_rows(ext, cuda_device, G, keep):
    logits, bias = _logits(12, 48, torch.float32, cuda_device, seed=4)
    logits[0] = -float("inf")                                # nothing left
    logits[1] = float("nan")
    logits[2, 3:] = -float("inf")                            # fewer than topk left
    logits[3, ::2] = float("nan")
    logits[4, 5] = float("inf")
    logits[5] = torch.finfo(torch.float32).min               # the lowest finite value is not a mask
    logits[6, 10:] = -torch.inf
    logits[7] = 0.0                                          # ties everywhere: the lowest ids
    logits[7, 24:] = -0.0
    for scoring in ("sigmoid", "softmax"):
        for b in (None, bias, torch.zeros_like(bias)):
            ids, w = check(logits, b, 6, scoring, G, keep)
            assert ids[0].tolist() == [-1] * 6 and w[0].tolist() == [0.0] * 6


@pytest.mark.parametrize("G,keep", [(1, 1), (4, 2)])
def test_masked_biases(ext, cuda_device, G, keep):
    """A bias of -inf or NaN keeps its expert from being chosen; one of +inf puts it first."""
    logits, bias = _logits(40, 48, torch.float32, cuda_device, seed=14)
    bias[3], bias[20:30], bias[47] = float("nan"), -float("inf"), float("inf")
    logits[1, 4:47] = -float("inf")                          # experts 0, 1, 2 and 47 are left
    logits[2:20] = logits[2] + 1e-7 * logits[2:20]           # near-ties: the ranking in 64 bits
    bias[:3] = 0.25
    logits[2:20, :3] = 0.5
    assert bool(bias.isnan().any())
    masked = logits.clone()
    masked[:, 3] = float("nan")
    masked[:, 20:30] = -float("inf")
    finite = bias.clone()
    finite[3] = 0
    finite[20:30] = 0
    finite[47] = 1e30
    ids, _ = check(masked, finite, 6, "sigmoid", G, keep)    # the sigmoid has no sum that a bias could change
    r = exl3_router.LogitsRouter(6, bias=bias, n_group=G, topk_group=keep, scale=2.5)
    got, w = r.route(logits)
    assert torch.equal(got, ids)
    for softmax in ("sigmoid", "softmax"):
        got, w = exl3_router.LogitsRouter(6, softmax, bias, G, keep).route(logits)
        chosen = got[got >= 0]
        assert not bool(((chosen == 3) | ((chosen >= 20) & (chosen < 30))).any()) and bool(torch.isfinite(w).all())
        assert all(len(set(row)) == len(row) for row in ([e for e in t if e >= 0] for t in got.tolist()))
        first = (got == 47).any(1)                           # (alone in its group, it has no sum of two in row 1)
        assert bool(first[torch.arange(40, device=cuda_device) != 1].all()) and bool(first[1]) == (G == 1)
        assert got[1].tolist().count(-1) >= 2


def test_near_ties_are_decided_exactly(ext, cuda_device):
    """Scores plus bias that 32 bits cannot tell apart (gaps of 1e-9 .. 1e-7 around equal sums)."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(9)
    E = 64
    logits = torch.randn(200, E, generator=g, device=dev)
    base = torch.sigmoid(logits[0].double())
    bias = (0.7 - base + 1e-8 * torch.randn(E, generator=g, device=dev)).float()
    logits[1:100] = logits[0] + 1e-7 * torch.randn(99, E, generator=g, device=dev)
    check(logits, bias, 8)
    check(logits, bias, 8, n_group=8, topk_group=3)
    check(logits, bias, 8, scoring="softmax", n_group=8, topk_group=3)
    check(logits, None, 8, n_group=8, topk_group=3)


def test_strided_rows_other_stream_and_graph(ext, cuda_device):
    dev = cuda_device
    wide, bias = _logits(50, 320, torch.float32, dev, seed=6)
    part = wide[:, 16:304]
    ids, w = check(part, bias[:288].contiguous(), 8)
    r = exl3_router.LogitsRouter(8, bias=bias[:288].contiguous(), scale=2.5)
    s = torch.cuda.Stream()
    s.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(s):
        graph = torch.cuda.CUDAGraph()
        r.route(part)
        with torch.cuda.graph(graph, stream=s):
            gi, gw = r.route(part)
    torch.cuda.current_stream().wait_stream(s)
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gi, ids) and torch.equal(gw, w)
    wide.copy_(wide.flip(0))
    graph.replay()
    torch.cuda.synchronize()
    assert torch.equal(gi, ids.flip(0)) and torch.equal(gw, w.flip(0))


def test_no_tokens(ext, cuda_device):
    ids, w = exl3_router.LogitsRouter(4).route(torch.empty(0, 16, device=cuda_device))
    assert ids.shape == (0, 4) and w.shape == (0, 4)


def test_moe_from_logits_is_the_block_on_its_routing(ext, cuda_device):
    import exl3_dense
    dev = cuda_device
    layer = synth.layer_to(synth.make_layer(16, 256, 128, seed=31, sv_scale=0.05), dev)
    x = synth.make_x(40, 256, seed=3, device=dev)
    logits, bias = _logits(40, 16, torch.bfloat16, dev, seed=2)
    r = exl3_router.LogitsRouter(4, bias=bias, n_group=4, topk_group=2)
    out, ids, w = exl3_router.moe_prefill_from_logits(x, logits, r, layer, 7.0, return_routing=True)
    ref = exl3_dense.moe_block_prefill(x, ids, w, layer, None, 7.0)
    assert float((out - ref).norm() / ref.norm()) < 1e-6      # the trellis down stage adds in any order


def test_offsets_past_32_bits(ext, cuda_device):
    dev = cuda_device
    T, E = 9_000_000, 256                                    # 2.3e9 logits
    logits = torch.empty(T, E, dtype=torch.bfloat16, device=dev).normal_(generator=torch.Generator(device=dev).manual_seed(3))
    ids, w = exl3_router.LogitsRouter(2).route(logits)
    tail_ids, tail_w = exl3_router.LogitsRouter(2).route(logits[-7:])
    assert torch.equal(ids[-7:], tail_ids) and torch.equal(w[-7:], tail_w)
    check(logits[-7:], None, 2)


@pytest.mark.parametrize("G,keep", [(1, 1), (4, 2)])
def test_missing_slots_come_last_whatever_the_scores(ext, cuda_device, G, keep):
    """Fewer experts than slots, with scores plus bias at or below zero, tied and not: experts first, then -1."""
    E, k = 48, 6
    few = [(1, 3), (0, 5, 9), (2, 4, 7, 11), (1, 2, 3, 4, 5)]
    logits = torch.full((8, E), -float("inf"), device=cuda_device)
    for t in range(8):
        live = torch.tensor(few[t % 4], device=cuda_device)
        logits[t, live] = 0.25 if t < 4 else torch.linspace(-1, 1, live.numel(), device=cuda_device)
    flat = torch.full((E,), -1.0, device=cuda_device)
    tied_above = flat.clone()                                # a tie of positive scores before a negative one
    tied_above[1:3] = 0.5
    sunk = logits.clone()                                    # scores of exactly zero
    sunk[logits > -float("inf")] = -1e4
    for scoring in ("sigmoid", "softmax"):
        for l, b in ((logits, flat), (logits, tied_above), (logits, -0.25 - torch.arange(E, device=cuda_device) / 64),
                     (sunk, torch.zeros_like(flat))):
            ids, w = check(l, b.float(), k, scoring, G, keep)
            assert ids[0].tolist()[2:] == [-1] * 4 and w[0].tolist()[2:] == [0.0] * 4


def test_group_scores_of_cancelling_biases(ext, cuda_device):
    """The two best of a group have large biases of opposite sign: their sum is small and its rounding is not."""
    dev = cuda_device
    g = torch.Generator(device=dev).manual_seed(19)
    noise = torch.randn(300, 16, generator=g, device=dev)
    for sizes in ([64.0] * 8, [1000.0] * 8, [0.0, 64.0, 1000.0, 3e4, 0.0, 64.0, 1000.0, 3e4]):
        bias = torch.tensor([v for s in sizes for v in (s, -s)], device=dev)
        for spread in (1e-5, 1e-4, 1e-3):                    # about the rounding of the addends, and on both sides of it
            for scoring in ("sigmoid", "softmax"):
                check(0.3 + spread * noise, bias, 5, scoring, n_group=8, topk_group=3)


def test_group_scores_past_the_largest_float(ext, cuda_device):
    """Sums of two biases that fp32 does not hold: groups keep their order, and finite ones stay above empty ones."""
    dev = cuda_device
    logits, bias = _logits(30, 16, torch.float32, dev, seed=23)
    high = bias.clone()
    high[0:4] = torch.tensor([3e38, 2e38, 1.0, 1.0], device=dev)
    high[8:12] = torch.tensor([3e38, 2.5e38, 2.5e38, 1.0], device=dev)
    low = bias.clone()
    low[4:8], low[8:12] = torch.finfo(torch.float32).min, -3e38
    empty = logits.clone()
    empty[:, :4] = -float("inf")
    for l in (logits, empty):
        for b in (high, low):
            for keep in (1, 2, 3):
                check(l, b, 3, n_group=4, topk_group=keep)
