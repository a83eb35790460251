"""CPU: refusals of the routing and 8-bit entry points, and the load-time weight quantiser."""
import ctypes
import types

import pytest
import torch

import b200_ext
import ep
import exl3_dense
import exl3_fp8
import exl3_router

P = ctypes.c_void_p
A = P(256)                                                    # never dereferenced: every case fails before a launch


@pytest.fixture(scope="module")
def lib():
    return b200_ext.load()


def refused(lib, rc, text):
    assert rc not in (0, None) and text in lib.exl3_last_error().decode(), lib.exl3_last_error()


def test_route_logits_refusals(lib):
    def call(logits=A, dtype=0, T=4, E=16, stride=16, G=1, keep=1, gtop=1, k=4, scale=1.0, ids=A):
        return lib.exl3_route_logits(logits, dtype, T, E, stride, None, 0, G, keep, gtop, k, 1, scale, ids, A, None)
    refused(lib, call(dtype=3), "float32, float16 or bfloat16")
    refused(lib, call(E=1025, stride=1025), "too many experts")
    refused(lib, call(E=0), "too many experts")
    refused(lib, call(T=-1), "invalid routing shape")
    refused(lib, call(stride=15), "rows overlap")
    refused(lib, call(G=3), "divide the number of experts")
    refused(lib, call(G=33, E=33, stride=33), "n_group must be 1..32")
    refused(lib, call(G=4, keep=5), "topk_group")
    refused(lib, call(gtop=3), "group_top")
    refused(lib, call(G=16, keep=8, gtop=2), "group_top")
    refused(lib, call(k=17), "topk must be")
    refused(lib, call(k=0), "topk must be")
    refused(lib, call(G=4, keep=1, k=5), "topk must be")
    refused(lib, call(E=64, stride=64, k=33), "topk must be 1..32")
    refused(lib, call(scale=float("nan")), "scale must be finite")
    refused(lib, call(logits=None), "CUDA")
    refused(lib, call(ids=None), "CUDA")
    assert call(logits=None, T=0) == 0


def test_quantize_refusals(lib):
    def call(x=A, dtype=1, T=4, K=256, xs=256, q=A, qs=256, s=A):
        return lib.exl3_fp8_quantize_rows(x, dtype, T, K, xs, 0, q, qs, s, 2, 1, None)
    refused(lib, call(dtype=-1), "unknown dtype")
    refused(lib, call(T=-1), "invalid row count")
    refused(lib, call(K=0), "invalid row length")
    refused(lib, call(xs=255), "rows overlap")
    refused(lib, call(qs=255), "output rows overlap")
    refused(lib, call(q=None), "CUDA")
    assert call(x=None, T=0) == 0


def test_linear_refusals(lib):
    need = lib.exl3_fp8_linear_workspace(4, 256, 64)
    assert need >= 4 * 256 + 4 * 2 * 4 and lib.exl3_fp8_linear_workspace(4, 100, 64) == -1

    def call(T=4, K=256, xs=256, w=A, wstride=256, wss=2, N=64, out=A, odt=0, ostride=64, ws=A, nbytes=need):
        return lib.exl3_fp8_linear(A, 1, T, K, xs, w, wstride, A, wss, N, out, odt, ostride, 0, ws, nbytes, None, None)
    refused(lib, call(K=100, xs=100), "multiple of 16")
    refused(lib, call(N=0), "weight rows")
    refused(lib, call(odt=3), "output dtype")
    refused(lib, call(ostride=63), "output rows overlap")
    refused(lib, call(w=P(264)), "16-byte aligned")
    refused(lib, call(wstride=248), "16-byte aligned")
    refused(lib, call(wss=1), "weight scales")
    refused(lib, call(nbytes=need - 1), "workspace must hold")
    refused(lib, call(ws=P(8)), "workspace must hold")
    refused(lib, call(out=None), "CUDA")
    assert call(T=0, out=None, ws=None) == 0


def test_experts_refusals(lib):
    need = lib.exl3_fp8_experts_workspace(4, 2, 8, 256, 128)
    assert need > 0
    assert lib.exl3_fp8_experts_workspace(4, 2, 1025, 256, 128) == -1
    assert lib.exl3_fp8_mlp_workspace(4, 256, 100) == -1

    def call(T=4, d=256, k=2, E=8, f=128, limit=7.0, wdt=0, w13=A, out=A, ostride=256, nbytes=need, ids=A):
        return lib.exl3_fp8_experts(A, 1, T, d, d, ids, 1, A, wdt, k, E, w13, A, A, A, f, limit, out, 0, ostride, 0, A,
                                    nbytes, None, None)
    refused(lib, call(E=0), "too many experts")
    refused(lib, call(k=33), "topk must be 1..32")
    refused(lib, call(d=200), "d must be a multiple of 128")
    refused(lib, call(f=64), "f must be a multiple of 128")
    refused(lib, call(T=1 << 30), "invalid routing shape")
    refused(lib, call(limit=0.0), "limit must be positive")
    refused(lib, call(limit=float("nan")), "limit must be positive")
    refused(lib, call(wdt=5), "weight dtype")
    refused(lib, call(w13=P(8)), "16-byte aligned")
    refused(lib, call(ostride=255), "output rows overlap")
    refused(lib, call(nbytes=need - 1), "workspace must hold")
    refused(lib, call(ids=None), "CUDA")
    assert call(T=0, out=None) == 0
    rc = lib.exl3_fp8_mlp(A, 1, 4, 256, 256, A, A, A, A, 128, -1.0, A, 0, 256, 0, A, 1 << 20, None, None)
    refused(lib, rc, "limit must be positive")
    rc = lib.exl3_fp8_mlp(A, 1, 4, 256, 256, A, A, A, A, 128, 7.0, A, 0, 256, 0, A, 16, None, None)
    refused(lib, rc, "workspace must hold")


def test_python_refusals(lib):
    e4 = torch.float8_e4m3fn
    x = torch.zeros(4, 256)
    w, ws = torch.zeros(64, 256, dtype=e4), torch.ones(1, 2)
    for bad, text in [(lambda: exl3_fp8.fp8_linear(x, w[:, :128], ws), "K mismatch"),
                      (lambda: exl3_fp8.fp8_linear(x, w.float(), ws), "weight e4m3"),
                      (lambda: exl3_fp8.fp8_linear(x, w, ws[:, :1]), "weight_scale"),
                      (lambda: exl3_fp8.fp8_linear(x.double(), w, ws), "float32, float16 or bfloat16"),
                      (lambda: exl3_fp8.fp8_linear(x.t().contiguous().t(), w, ws), "contiguous, separate rows"),
                      (lambda: exl3_fp8.fp8_linear(x[:1].expand(4, 256), w, ws), "contiguous, separate rows"),
                      (lambda: exl3_fp8.fp8_linear(x, w, ws), "CUDA"),
                      (lambda: exl3_fp8.quantize_rows(x[0]), r"\[T, K\]"),
                      (lambda: exl3_fp8.quantize_rows(x), "CUDA"),
                      (lambda: exl3_router.LogitsRouter(2, scoring="relu"), "scoring"),
                      (lambda: exl3_router.LogitsRouter(2).route(x[0]), r"\[T, E\]"),
                      (lambda: exl3_router.LogitsRouter(2).route(x), "CUDA"),
                      (lambda: exl3_router.LogitsRouter(2, bias=torch.zeros(3)).route(x), "bias"),
                      (lambda: exl3_router.LogitsRouter(2).route(x.int()), "float32, float16 or bfloat16")]:
        with pytest.raises(RuntimeError, match=text):
            bad()
    L = types.SimpleNamespace(w13_fp8=torch.zeros(2, 256, 256, dtype=e4), w13_scale=torch.ones(2, 2, 2),
                              w2_fp8=torch.zeros(2, 256, 128, dtype=e4), w2_scale=torch.ones(2, 2, 1))
    ids, rw = torch.zeros(4, 2, dtype=torch.int64), torch.ones(4, 2)
    with pytest.raises(RuntimeError, match="CUDA"):
        exl3_fp8.fp8_prefill(x, ids, rw, L, 7.0)
    with pytest.raises(RuntimeError, match="CUDA|one expert"):
        exl3_dense.dense_mlp_prefill(x, L, 7.0)
    L.w2_scale = torch.ones(2, 1, 2)
    with pytest.raises(RuntimeError, match="w2_scale"):
        exl3_fp8.fp8_prefill(x, ids, rw, L, 7.0)
    L.w13_fp8 = L.w13_fp8[:, :200]
    with pytest.raises(RuntimeError, match="w13_fp8"):
        exl3_fp8.fp8_prefill(x, ids, rw, L, 7.0)


def test_broadcast_weight_scales_are_refused(lib):
    """Scales with a row stride of 0 would be read past their end: refused before a launch."""
    x = torch.zeros(4, 256)
    w = torch.zeros(300, 256, dtype=torch.float8_e4m3fn)
    for scale in (torch.ones(1, 2).expand(3, 2), torch.ones(1).expand(3, 2), torch.ones(2, 3).t()):
        with pytest.raises(RuntimeError, match="weight_scale"):
            exl3_fp8.fp8_linear(x, w, scale)


def test_one_token_linear_refuses_an_output_that_overlaps_its_input(lib):
    def call(T, x, out, ws=None, nbytes=0):
        return lib.exl3_fp8_linear(P(x), 1, T, 256, 256, A, 256, A, 2, 64, P(out), 0, 64, 1, ws, nbytes, None, None)
    for x, out in [(4096, 4096), (4096, 4096 + 511), (4096 + 255, 4096), (4096, 4096 - 255)]:
        refused(lib, call(1, x, out), "overlaps x")


def test_workspace_sizes_name_their_refusal(lib):
    assert lib.exl3_fp8_linear_workspace(4, 0, 64) == -1
    assert "fp8_linear: invalid sizes" in lib.exl3_last_error().decode()
    assert lib.exl3_fp8_mlp_workspace(4, 256, 64) == -1
    assert "f must be a multiple of 128" in lib.exl3_last_error().decode()


def test_layers_that_do_not_fit_are_refused():
    L = types.SimpleNamespace(w13_fp8=torch.zeros(2, 256, 256, dtype=torch.float8_e4m3fn))
    with pytest.raises(RuntimeError, match="number of experts"):
        exl3_router.moe_prefill_from_logits(torch.zeros(4, 256), torch.zeros(4, 3), exl3_router.LogitsRouter(1), L, 7.0)
    for call in (lambda: ep.layer_slice(L, 0, 1), lambda: ep.layer_take(L, [0])):
        with pytest.raises(RuntimeError, match="trellis layers"):
            call()


def test_packed_calls_reach_their_entry_points(lib):
    """Every argument of a packed call arrives: the refusals are those of the entry point itself."""
    def call(packer, *args):
        return lib.exl3_call(packer(*args))
    ok = [4096, 0, 4, 16, 16, 0, 0, 1, 1, 1, 4, 1, 1.0, 4096, 4096, 0]
    for i, bad, text in [(1, 3, "float32, float16"), (3, 1025, "too many experts"), (4, 15, "rows overlap"), (7, 3, "divide"),
                         (10, 17, "topk must be"), (12, float("inf"), "scale must be finite"), (13, 0, "CUDA")]:
        refused(lib, call(b200_ext._ROUTE_LOGITS, *[bad if j == i else a for j, a in enumerate(ok)]), text)
    assert call(b200_ext._ROUTE_LOGITS, *[0 if j == 2 else a for j, a in enumerate(ok)]) == 0
    refused(lib, call(b200_ext._QUANTIZE_ROWS, 4096, 1, 4, 256, 256, 0, 4096, 255, 4096, 2, 1, 0), "output rows overlap")
    refused(lib, call(b200_ext._LINEAR, 4096, 1, 4, 256, 256, 4096, 256, 4096, 2, 64, 4096, 0, 64, 0, 4096, 16, 0, 0), "workspace must")
    refused(lib, call(b200_ext._MLP, 4096, 1, 4, 256, 256, 4096, 4096, 4096, 4096, 128, -1.0, 4096, 0, 256, 0, 4096, 16, 0, 0),
            "limit must be positive")
    refused(lib, call(b200_ext._EXPERTS, 4096, 1, 4, 256, 256, 4096, 1, 4096, 0, 2, 8, 4096, 4096, 4096, 4096, 128, 7.0, 4096, 0,
                      256, 0, 4096, 16, 0, 0), "workspace must hold")
    refused(lib, lib.exl3_call(None), "no arguments")
    refused(lib, lib.exl3_call((1 + 256 * 3).to_bytes(8, "little") + bytes(64)), "number of arguments")
    refused(lib, lib.exl3_call((99).to_bytes(8, "little")), "unknown call")


@pytest.mark.parametrize("shape", [(128, 128), (1, 16), (200, 300), (3, 130, 256)])
def test_quantize_weight(shape):
    w = torch.randn(*shape, generator=torch.Generator().manual_seed(1))
    w.view(-1)[:5] = 0
    q, s = exl3_fp8.quantize_weight(w)
    n, k = shape[-2:]
    assert q.shape == w.shape and s.shape == (*shape[:-2], -(-n // 128), -(-k // 128))
    full = s.repeat_interleave(128, -2)[..., :n, :].repeat_interleave(128, -1)[..., :k]
    # half a step of e4m3 (2^-4 of the value; 2^-10 of the scale's unit below 2^-6), and the fp32 division's rounding
    assert bool(((q.float() * full - w).abs() <= w.abs() * (2.0 ** -4 + 2.0 ** -20) + full * 2.0 ** -10).all())
    for b in range(s.shape[-1]):
        block = w[..., :128, b * 128:(b + 1) * 128]
        assert torch.allclose(s[..., 0, b] * 448, block.abs().amax(dim=(-2, -1)), rtol=1e-6, atol=1e-15)
    with pytest.raises(RuntimeError, match="NaN or inf"):
        exl3_fp8.quantize_weight(torch.full((2, 16), float("nan")))


@pytest.mark.parametrize("rows", [3, 5])
def test_routing_of_other_tokens_is_refused(lib, rows):
    """Logits (or ids) for another number of tokens than the hidden states have, with either kind of layer."""
    x = torch.zeros(4, 256)
    fp8 = types.SimpleNamespace(w13_fp8=torch.zeros(8, 256, 256, dtype=torch.float8_e4m3fn), w13_scale=torch.ones(8, 2, 2),
                                w2_fp8=torch.zeros(8, 256, 128, dtype=torch.float8_e4m3fn), w2_scale=torch.ones(8, 2, 1))
    trellis = types.SimpleNamespace(w13_trellis=torch.zeros(8, 2, 16, 8, 64, dtype=torch.int16))
    for layer in (fp8, trellis):
        with pytest.raises(RuntimeError, match="number of tokens"):
            exl3_router.moe_prefill_from_logits(x, torch.zeros(rows, 8), exl3_router.LogitsRouter(2), layer, 7.0)
        for ids in (torch.zeros(rows, 2, dtype=torch.int64), torch.zeros(4, dtype=torch.int64)):
            with pytest.raises(RuntimeError, match=r"\[T, topk\]"):
                exl3_dense.moe_block_prefill(x, ids, torch.ones(ids.shape), layer, None, 7.0)


def test_two_threads_share_one_status_word(monkeypatch):
    """First calls from two threads at once: both get the word that read_status reads (its address is kept)."""
    import threading
    together, made = threading.Barrier(2, timeout=20), torch.zeros

    def zeros(*args, **kwargs):
        together.wait()
        return made(*args, **kwargs)
    monkeypatch.setattr(b200_ext.torch, "zeros", zeros)
    monkeypatch.setattr(b200_ext, "_status", {})
    dev, got = torch.device("cpu", 0), []
    threads = [threading.Thread(target=lambda: got.append(b200_ext.status_tensor(dev))) for _ in range(2)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(got) == 2 and got[0] is got[1] and got[0] is b200_ext.status_tensor(dev)
