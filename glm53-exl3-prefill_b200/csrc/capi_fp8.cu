// capi_fp8.cu — the extern "C" boundary of routing from logits and of the 8-bit (e4m3) layers: argument
// checks, the workspace's layout, and the order of the launches.  Nothing here allocates or synchronises.
#include <cstdint>
#include <cstring>
#include <type_traits>
#include <utility>

#include <cuda_runtime.h>

#include "exl3_internal.h"
#include "../../include/exl3_b200.h"

using namespace exl3b;

namespace {

cudaStream_t as_stream(void* s) { return reinterpret_cast<cudaStream_t>(s); }
bool aligned16(const void* p) { return reinterpret_cast<uintptr_t>(p) % 16 == 0; }
int64_t up256(int64_t n) { return (n + 255) & ~int64_t(255); }
int64_t blocks128(int64_t n) { return (n + 127) / 128; }
bool is_dtype(int64_t d) { return d >= EXL3_DTYPE_F32 && d <= EXL3_DTYPE_BF16; }
int64_t bytes_of(int64_t dtype) { return dtype == EXL3_DTYPE_F32 ? 4 : 2; }
bool overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes)
{
    const uintptr_t x = reinterpret_cast<uintptr_t>(a), y = reinterpret_cast<uintptr_t>(b);
    return x < y + (uintptr_t) b_bytes && y < x + (uintptr_t) a_bytes;
}

constexpr int64_t kMaxDim = 0x7fffff00;

// Pieces of the caller's workspace (null: only their sizes), 256-byte aligned whatever the workspace's own alignment of 16
// bytes or more: kernels store whole 32-byte sectors into them.
constexpr int64_t kAlignSlack = 256 - 16;
struct Carver {
    uint8_t* base;
    int64_t used = 0;
    explicit Carver(void* workspace)
        : base(reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(workspace) + 255) & ~uintptr_t(255))) {}
    int64_t bytes() const { return used ? used + kAlignSlack : 0; }
    template <class T> T* take(int64_t n)
    {
        uint8_t* p = base ? base + used : nullptr;
        used += up256(n * (int64_t) sizeof(T));
        return reinterpret_cast<T*>(p);
    }
};

// Quantised rows: e4m3 [rows, k] and scales [k / 128][rows], so that a K block's scales lie side by side.
struct Rows8 {
    uint8_t* q;
    float* s;
};

Rows8 take_rows(Carver& c, int64_t rows, int64_t k)
{
    Rows8 r;
    r.q = c.take<uint8_t>(rows * k);
    r.s = c.take<float>(rows * blocks128(k));
    return r;
}

// Partial sums of a product whose K is split (parts > 1): fp32 [parts][rows][ld].
struct Parts {
    int n;
    int64_t ld, stride;
    float* p;
};

Parts take_parts(Carver& c, int64_t rows, int64_t E, int64_t N, int64_t K)
{
    Parts r{fp8_gemm_splits(rows, (int) E, (int) N, (int) K), (N + 7) / 8 * 8, 0, nullptr};
    r.stride = rows * r.ld;
    if (r.n > 1) r.p = c.take<float>(r.n * r.stride);
    return r;
}

// The product of a problem that stores its sums, with K split into parts.
int run_split(Fp8GemmProblem p, const Parts& parts, cudaStream_t stream)
{
    p.swiglu = 0;
    p.out = parts.p; p.out_stride = parts.ld; p.out_dtype = EXL3_DTYPE_F32; p.accumulate = 0;
    p.splits = parts.n; p.split_stride = parts.stride;
    return launch_fp8_gemm(p, stream);
}

// Whether rows are quantised once per token and copied to their routes (two launches), or once per route (one).  At 4096
// columns and 8 routes a token, per route and per token: 8192 tokens 190 and 95 us, 2048 55 and 30, 512 16 and 14.
bool many_routes(int64_t R, int64_t topk) { return topk > 1 && R >= 4096; }

struct ExpertBuffers {
    int64_t* slot;
    void* weight_sorted;
    int32_t *expert_of_row, *counts, *row0, *meta, *scratch;
    Rows8 tokens;                   // quantised once per token, if that pays
    Rows8 x, h;
    Parts gu;                       // gate | up sums, if split
    Parts y;                        // the routes' rows: one part at least
};

ExpertBuffers take_experts(Carver& c, int64_t T, int64_t topk, int64_t E, int64_t d, int64_t f)
{
    const int64_t R = T * topk;
    ExpertBuffers b{};
    b.slot = c.take<int64_t>(R);
    b.weight_sorted = c.take<uint16_t>(R);
    b.expert_of_row = c.take<int32_t>(R);
    b.counts = c.take<int32_t>(E);
    b.row0 = c.take<int32_t>(E);
    b.meta = c.take<int32_t>(2);
    b.scratch = c.take<int32_t>(route_sort_scratch_elems(R, (int) E));
    if (many_routes(R, topk)) b.tokens = take_rows(c, T, d);
    b.x = take_rows(c, R, d);
    b.h = take_rows(c, R, f);
    b.gu = take_parts(c, R, E, 2 * f, d);
    b.y = take_parts(c, R, E, d, f);
    if (b.y.n == 1) b.y.p = c.take<float>(b.y.stride);
    return b;
}

// Routes whose products each read their expert's weights for themselves (fp8_small.cu), activations [R, f] in the workspace.
// With 288 experts of 4096 x 1536 (every route another expert), 8 / 16 / 32 / 64 routes: 39 / 72 / 126 / 257 us, and 58 / 95 /
// 138 / 203 us by the tiles of fp8_gemm.cu.  Where routes share experts the tiles read their weights once, hence the second bound:
// small experts gain up to it (1024 x 512: 24 routes over 24 experts 18.5 us, by tiles 30, which need 28 to start up; 2048 x 768:
// 32 over 48 48 and 50 us), large ones only to about R * R = 12 E (4096 x 1536: 8 over 4 38 and 41 us, 16 over 8 68 and 56,
// 32 over 16 126 and 86).
bool few_routes(int64_t R, int64_t E) { return R <= 32 && R <= 2 * E; }

// Tokens whose product streams the weights through fp8_small.cu rather than in tiles.  Up to 8 tokens it is never slower: 6.5
// against 14.0 us for 4096 x 4096, 23.4 against 24.3 for 24576 x 4096, 14.5 against 17.8 for 2048 x 16384.  9..16 tokens take
// twice the instructions: 9.6 against 15.0 us for 4096 x 4096 and 16.4 against 16.8 for 8192 x 4096, but 22.1 against 19.2 for
// 12288 x 4096, and 28.7 against 18.4 for 2048 x 16384, whose rows are long and few.
bool few_tokens(int64_t T, int64_t N, int64_t K)
{
    return T <= 8 || (T <= kFp8FewTokens && N * K <= (1 << 25) && K <= 2 * N);
}
bool few_mlp_tokens(int64_t T, int64_t d, int64_t f) { return few_tokens(T, 2 * f, d) && few_tokens(T, d, f); }

int check_rows(const char* what, int64_t dtype, int64_t rows, int64_t K, int64_t stride)
{
    if (!is_dtype(dtype)) return set_error("%s: unknown dtype", what);
    if (rows < 0 || rows > kMaxDim) return set_error("%s: invalid row count", what);
    if (K < 1 || K > kMaxDim) return set_error("%s: invalid row length", what);
    if (rows > 1 && stride < K) return set_error("%s: rows overlap (row stride below the row length)", what);
    return EXL3_OK;
}

int check_experts_shape(const char* what, int64_t T, int64_t topk, int64_t E, int64_t d, int64_t f)
{
    if (E <= 0 || E > kMaxExperts) return set_error("too many experts");
    if (topk < 1 || topk > 32) return set_error("%s: topk must be 1..32", what);
    if (T < 0 || T > kMaxDim || T * topk > kMaxDim) return set_error("invalid routing shape");
    if (d <= 0 || d % 128 != 0 || d > (1 << 24)) return set_error("%s: d must be a multiple of 128", what);
    if (f <= 0 || f % 128 != 0 || f > (1 << 24)) return set_error("%s: f must be a multiple of 128", what);
    return EXL3_OK;
}

int check_out(const char* what, const void* out, int64_t out_dtype, int64_t T, int64_t n, int64_t stride)
{
    if (!is_dtype(out_dtype)) return set_error("%s: unknown output dtype", what);
    if (T > 1 && stride < n) return set_error("%s: output rows overlap", what);
    if (!out) return set_error("tensors must be CUDA");
    return EXL3_OK;
}

// Both products of the gated MLP over quantised rows x [rows, d]: gate | up into h, then down's sums into `y` (its parts, if
// it has several), or into `out` if y has one.
int run_mlp(const Rows8& x, const Rows8& h, const Parts& gu, const Parts& y, int64_t rows, int64_t d, int64_t f, int64_t E,
            const int32_t* counts, const int32_t* row0, const int32_t* rows_dev, const void* w13, const float* w13_scale,
            const void* w2, const float* w2_scale, double limit, void* out, int64_t out_stride, int64_t out_dtype,
            int accumulate, const int64_t* slot, int32_t* status, cudaStream_t stream)
{
    Fp8GemmProblem p{};
    p.x = x.q; p.rows = rows; p.x_stride = d; p.K = (int) d;
    p.sx = x.s; p.sx_row = 1; p.sx_blk = rows;
    p.w = w13; p.w_stride = d; p.w_expert = 2 * f * d; p.N = (int) (2 * f); p.n_experts = (int) E;
    p.sw = w13_scale; p.sw_n = blocks128(d); p.sw_expert = blocks128(2 * f) * p.sw_n;
    p.counts = counts; p.row0 = row0;
    p.swiglu = 1; p.limit = (float) limit;
    p.h = h.q; p.h_stride = f; p.hs = h.s; p.hs_row = 1; p.hs_blk = rows;
    p.status = status;
    int rc = gu.n > 1 ? run_split(p, gu, stream) : launch_fp8_gemm(p, stream);
    if (rc) return rc;
    if (gu.n > 1)
    {
        rc = launch_fp8_act(gu.p, gu.n, gu.stride, gu.ld, rows, rows_dev, (int) f, (float) limit, h.q, f, h.s, 1, rows, stream);
        if (rc) return rc;
    }
    Fp8GemmProblem q{};
    q.x = h.q; q.rows = rows; q.x_stride = f; q.K = (int) f;
    q.sx = h.s; q.sx_row = 1; q.sx_blk = rows;
    q.w = w2; q.w_stride = f; q.w_expert = d * f; q.N = (int) d; q.n_experts = (int) E;
    q.sw = w2_scale; q.sw_n = blocks128(f); q.sw_expert = blocks128(d) * q.sw_n;
    q.counts = counts; q.row0 = row0;
    q.slot = slot; q.status = status;
    if (y.n > 1) return run_split(q, y, stream);
    q.out = out; q.out_stride = out_stride; q.out_dtype = (int) out_dtype; q.accumulate = accumulate;
    return launch_fp8_gemm(q, stream);
}

template <class A>
A argument(const int64_t* word)
{
    if constexpr (std::is_pointer_v<A>) return reinterpret_cast<A>(*word);
    else if constexpr (std::is_same_v<A, double>)
    {
        double d;
        std::memcpy(&d, word, sizeof d);
        return d;
    }
    else return static_cast<A>(*word);
}

template <class... A, size_t... I>
int call_with(int (*fn)(A...), const int64_t* args, std::index_sequence<I...>)
{
    return fn(argument<A>(args + I)...);
}

template <class... A>
int call_packed(int (*fn)(A...), const int64_t* words)
{
    if (words[0] >> 8 != (int64_t) sizeof...(A)) return set_error("exl3_call: wrong number of arguments");
    return call_with(fn, words + 1, std::index_sequence_for<A...>());
}

}  // namespace

extern "C" {

int exl3_route_logits(const void* logits, int64_t dtype, int64_t T, int64_t E, int64_t row_stride, const float* bias,
                      int64_t softmax, int64_t n_group, int64_t topk_group, int64_t group_top, int64_t topk,
                      int64_t norm, double scale, int64_t* ids, float* weights, void* stream)
{
    if (!is_dtype(dtype)) return set_error("route_logits: logits must be float32, float16 or bfloat16");
    if (E <= 0 || E > kMaxExperts) return set_error("too many experts");
    if (T < 0 || T > kMaxDim) return set_error("invalid routing shape");
    if (T > 1 && row_stride < E) return set_error("route_logits: rows overlap (row stride below the number of experts)");
    if (n_group < 1 || n_group > 32 || E % n_group != 0)
        return set_error("route_logits: n_group must be 1..32 and divide the number of experts");
    if (topk_group < 1 || topk_group > n_group) return set_error("route_logits: topk_group must be 1..n_group");
    if (group_top < 1 || group_top > 2 || group_top > E / n_group)
        return set_error("route_logits: group_top must be 1 or 2 and at most the experts of a group");
    if (topk < 1 || topk > 32 || topk > topk_group * (E / n_group))
        return set_error("route_logits: topk must be 1..32 and at most the experts of the kept groups");
    if (!(scale >= -3.0e38 && scale <= 3.0e38)) return set_error("route_logits: scale must be finite");
    if (T == 0) return EXL3_OK;
    if (!logits || !ids || !weights) return set_error("tensors must be CUDA");
    return launch_route_logits(logits, (int) dtype, T, (int) E, row_stride, bias, softmax ? 1 : 0, (int) n_group,
                               (int) topk_group, (int) group_top, (int) topk, norm ? 1 : 0, (float) scale, ids, weights,
                               as_stream(stream));
}

int exl3_fp8_quantize_rows(const void* x, int64_t dtype, int64_t rows, int64_t K, int64_t x_stride, int64_t pow2,
                           void* q, int64_t q_stride, float* scale, int64_t s_row, int64_t s_blk, void* stream)
{
    const int rc = check_rows("fp8_quantize_rows", dtype, rows, K, x_stride);
    if (rc) return rc;
    if (rows > 1 && q_stride < K) return set_error("fp8_quantize_rows: output rows overlap");
    if (rows == 0) return EXL3_OK;
    if (!x || !q || !scale) return set_error("tensors must be CUDA");
    return launch_fp8_quantize(x, (int) dtype, rows, (int) K, x_stride, pow2 ? 1 : 0, q, q_stride, scale, s_row, s_blk,
                               nullptr, 1, nullptr, false, as_stream(stream));
}

int64_t exl3_fp8_linear_workspace(int64_t T, int64_t K, int64_t N)
{
    if (T < 0 || T > kMaxDim || K < 16 || K % 16 != 0 || K > (1 << 24) || N < 1 || N > (1 << 24))
    {
        set_error("fp8_linear: invalid sizes (K must be a multiple of 16, K and N 1..2^24)");
        return -1;
    }
    if (T <= 1) return 0;                               // one row is quantised on the way
    Carver c(nullptr);
    take_rows(c, T, K);
    if (!few_tokens(T, N, K)) take_parts(c, T, 1, N, K);
    return c.bytes();
}

int exl3_fp8_linear(const void* x, int64_t dtype, int64_t T, int64_t K, int64_t x_stride, const void* w, int64_t w_stride,
                    const float* w_scale, int64_t w_scale_stride, int64_t N, void* out, int64_t out_dtype,
                    int64_t out_stride, int accumulate, void* workspace, int64_t workspace_bytes, int32_t* status,
                    void* stream)
{
    int rc = check_rows("fp8_linear", dtype, T, K, x_stride);
    if (rc) return rc;
    if (K % 16 != 0 || K > (1 << 24)) return set_error("fp8_linear: K must be a multiple of 16");
    if (N < 1 || N > (1 << 24)) return set_error("fp8_linear: invalid number of weight rows");
    if (T == 0) return EXL3_OK;
    if ((rc = check_out("fp8_linear", out, out_dtype, T, N, out_stride))) return rc;
    if (!x || !w || !w_scale || (!workspace && T > 1)) return set_error("tensors must be CUDA");
    if (!aligned16(w) || w_stride % 16 != 0 || w_stride < K)
        return set_error("fp8_linear: the weight's rows must be 16-byte aligned");
    if (w_scale_stride < blocks128(K)) return set_error("fp8_linear: weight scales [ceil(N / 128), ceil(K / 128)]");
    if (!aligned16(workspace) || workspace_bytes < exl3_fp8_linear_workspace(T, K, N))
        return set_error("fp8_linear: workspace must hold exl3_fp8_linear_workspace() bytes");
    if (T == 1 && overlap(x, K * bytes_of(dtype), out, N * bytes_of(out_dtype)))
        return set_error("fp8_linear: out overlaps x (one token is read while out is written)");
    if (T == 1)
        return launch_fp8_linear_token(x, (int) dtype, (int) K, w, w_stride, w_scale, w_scale_stride, (int) N, out,
                                       (int) out_dtype, accumulate ? 1 : 0, as_stream(stream));
    Carver c(workspace);
    const Rows8 r = take_rows(c, T, K);
    rc = launch_fp8_quantize(x, (int) dtype, T, (int) K, x_stride, 0, r.q, K, r.s, 1, T, nullptr, 1, nullptr,
                             false, as_stream(stream));
    if (rc) return rc;
    Fp8GemmProblem p{};
    p.x = r.q; p.rows = T; p.x_stride = K; p.K = (int) K;
    p.sx = r.s; p.sx_row = 1; p.sx_blk = T;
    p.w = w; p.w_stride = w_stride; p.w_expert = w_stride * N; p.N = (int) N; p.n_experts = 1;
    p.sw = w_scale; p.sw_n = w_scale_stride; p.sw_expert = 0;
    p.out = out; p.out_stride = out_stride; p.out_dtype = (int) out_dtype; p.accumulate = accumulate ? 1 : 0;
    p.status = status;
    if (few_tokens(T, N, K)) return launch_fp8_linear_tokens(p, as_stream(stream));
    const Parts parts = take_parts(c, T, 1, N, K);
    if (parts.n == 1) return launch_fp8_gemm(p, as_stream(stream));
    if ((rc = run_split(p, parts, as_stream(stream)))) return rc;
    return launch_fp8_join(parts.p, parts.n, parts.stride, parts.ld, T, (int) N, accumulate ? 1 : 0, out, (int) out_dtype,
                           out_stride, as_stream(stream));
}

int64_t exl3_fp8_mlp_workspace(int64_t T, int64_t d, int64_t f)
{
    if (check_experts_shape("fp8_mlp", T, 1, 1, d, f)) return -1;
    Carver c(nullptr);
    take_rows(c, T, d);
    take_rows(c, T, f);
    if (few_mlp_tokens(T, d, f))
    {
        c.take<float>(T * 2 * f);
        return c.bytes();
    }
    take_parts(c, T, 1, 2 * f, d);
    take_parts(c, T, 1, d, f);
    return c.bytes();
}

int exl3_fp8_mlp(const void* x, int64_t dtype, int64_t T, int64_t d, int64_t x_stride, const void* w13,
                 const float* w13_scale, const void* w2, const float* w2_scale, int64_t f, double limit, void* out,
                 int64_t out_dtype, int64_t out_stride, int accumulate, void* workspace, int64_t workspace_bytes,
                 int32_t* status, void* stream)
{
    int rc = check_rows("fp8_mlp", dtype, T, d, x_stride);
    if (rc || (rc = check_experts_shape("fp8_mlp", T, 1, 1, d, f))) return rc;
    if (!(limit > 0.0)) return set_error("fp8_mlp: limit must be positive");
    if (T == 0) return EXL3_OK;
    if ((rc = check_out("fp8_mlp", out, out_dtype, T, d, out_stride))) return rc;
    if (!x || !w13 || !w13_scale || !w2 || !w2_scale || !workspace) return set_error("tensors must be CUDA");
    if (!aligned16(w13) || !aligned16(w2)) return set_error("fp8_mlp: weights must be 16-byte aligned");
    if (!aligned16(workspace) || workspace_bytes < exl3_fp8_mlp_workspace(T, d, f))
        return set_error("fp8_mlp: workspace must hold exl3_fp8_mlp_workspace() bytes");
    Carver c(workspace);
    const Rows8 xr = take_rows(c, T, d), hr = take_rows(c, T, f);
    if (few_mlp_tokens(T, d, f))
    {
        // the same four steps by the kernels for few tokens: rows, gate | up sums, activations, down
        float* sums = c.take<float>(T * 2 * f);
        rc = launch_fp8_quantize(x, (int) dtype, T, (int) d, x_stride, 0, xr.q, d, xr.s, 1, T, nullptr, 1, nullptr, false,
                                 as_stream(stream));
        if (rc) return rc;
        Fp8GemmProblem p{};
        p.x = xr.q; p.rows = T; p.x_stride = d; p.K = (int) d; p.sx = xr.s; p.sx_row = 1; p.sx_blk = T;
        p.w = w13; p.w_stride = d; p.N = (int) (2 * f); p.sw = w13_scale; p.sw_n = blocks128(d);
        p.out = sums; p.out_stride = 2 * f; p.out_dtype = EXL3_DTYPE_F32;
        if ((rc = launch_fp8_linear_tokens(p, as_stream(stream)))) return rc;
        rc = launch_fp8_act(sums, 1, 0, 2 * f, T, nullptr, (int) f, (float) limit, hr.q, f, hr.s, 1, T, as_stream(stream));
        if (rc) return rc;
        p.x = hr.q; p.x_stride = f; p.K = (int) f; p.sx = hr.s;
        p.w = w2; p.w_stride = f; p.N = (int) d; p.sw = w2_scale; p.sw_n = blocks128(f);
        p.out = out; p.out_stride = out_stride; p.out_dtype = (int) out_dtype; p.accumulate = accumulate ? 1 : 0;
        return launch_fp8_linear_tokens(p, as_stream(stream));
    }
    const Parts gu = take_parts(c, T, 1, 2 * f, d), y = take_parts(c, T, 1, d, f);
    rc = launch_fp8_quantize(x, (int) dtype, T, (int) d, x_stride, 0, xr.q, d, xr.s, 1, T, nullptr, 1, nullptr,
                             false, as_stream(stream));
    if (rc) return rc;
    rc = run_mlp(xr, hr, gu, y, T, d, f, 1, nullptr, nullptr, nullptr, w13, w13_scale, w2, w2_scale, limit, out, out_stride,
                 out_dtype, accumulate ? 1 : 0, nullptr, status, as_stream(stream));
    if (rc || y.n == 1) return rc;
    return launch_fp8_join(y.p, y.n, y.stride, y.ld, T, (int) d, accumulate ? 1 : 0, out, (int) out_dtype, out_stride,
                           as_stream(stream));
}

int64_t exl3_fp8_experts_workspace(int64_t T, int64_t topk, int64_t E, int64_t d, int64_t f)
{
    if (check_experts_shape("fp8_experts", T, topk, E, d, f)) return -1;
    if (few_routes(T * topk, E)) return up256(T * topk * f * (int64_t) sizeof(float));
    Carver c(nullptr);
    take_experts(c, T, topk, E, d, f);
    return c.bytes();
}

int exl3_fp8_experts(const void* x, int64_t dtype, int64_t T, int64_t d, int64_t x_stride, const void* ids,
                     int ids_is_int64, const void* weights, int64_t weight_dtype, int64_t topk, int64_t E,
                     const void* w13, const float* w13_scale, const void* w2, const float* w2_scale, int64_t f,
                     double limit, void* out, int64_t out_dtype, int64_t out_stride, int accumulate, void* workspace,
                     int64_t workspace_bytes, int32_t* status, void* stream)
{
    int rc = check_rows("fp8_experts", dtype, T, d, x_stride);
    if (rc || (rc = check_experts_shape("fp8_experts", T, topk, E, d, f))) return rc;
    if (!is_dtype(weight_dtype)) return set_error("unknown weight dtype");
    if (!(limit > 0.0)) return set_error("fp8_experts: limit must be positive");
    if (T == 0) return EXL3_OK;
    if ((rc = check_out("fp8_experts", out, out_dtype, T, d, out_stride))) return rc;
    if (!x || !ids || !weights || !w13 || !w13_scale || !w2 || !w2_scale || !workspace)
        return set_error("tensors must be CUDA");
    if (!aligned16(w13) || !aligned16(w2)) return set_error("fp8_experts: weights must be 16-byte aligned");
    if (!aligned16(workspace) || workspace_bytes < exl3_fp8_experts_workspace(T, topk, E, d, f))
        return set_error("fp8_experts: workspace must hold exl3_fp8_experts_workspace() bytes");
    cudaStream_t st = as_stream(stream);
    const int64_t R = T * topk;
    if (few_routes(R, E))
        return launch_fp8_experts_small(x, (int) dtype, (int) T, (int) d, x_stride, ids, ids_is_int64 ? 1 : 0, weights,
                                        (int) weight_dtype, (int) topk, (int) E, w13, w13_scale, w2, w2_scale, (int) f,
                                        (float) limit, static_cast<float*>(workspace), out, (int) out_dtype, out_stride,
                                        accumulate ? 1 : 0, st);
    Carver c(workspace);
    const ExpertBuffers b = take_experts(c, T, topk, E, d, f);
    // sorted by routing slot t * topk + j, so that each row knows both its token and its place in y
    rc = launch_route_sort(ids, ids_is_int64 ? 1 : 0, weights, (int) weight_dtype, R, 1, (int) E, 0, b.slot,
                           b.weight_sorted, b.expert_of_row, b.counts, b.row0, nullptr, nullptr, b.meta, nullptr,
                           b.scratch, st);
    if (rc) return rc;
    if (many_routes(R, topk))
    {
        rc = launch_fp8_quantize(x, (int) dtype, T, (int) d, x_stride, 0, b.tokens.q, d, b.tokens.s, 1, T, nullptr, 1,
                                 nullptr, true, st);
        if (rc) return rc;
        rc = launch_fp8_gather(b.tokens.q, b.tokens.s, T, b.slot, (int) topk, (int) d, b.meta + 1, b.x.q, b.x.s, R, st);
    }
    else
        rc = launch_fp8_quantize(x, (int) dtype, R, (int) d, x_stride, 0, b.x.q, d, b.x.s, 1, R, b.slot, (int) topk,
                                 b.meta + 1, true, st);
    if (rc) return rc;
    rc = run_mlp(b.x, b.h, b.gu, b.y, R, d, f, E, b.counts, b.row0, b.meta + 1, w13, w13_scale, w2, w2_scale, limit, b.y.p,
                 b.y.ld, EXL3_DTYPE_F32, 0, b.slot, status, st);
    if (rc) return rc;
    return launch_fp8_combine(b.y.p, b.y.ld, b.y.n, b.y.stride, ids, ids_is_int64 ? 1 : 0, weights, (int) weight_dtype, T,
                              (int) topk, (int) E, (int) d, accumulate ? 1 : 0, out, (int) out_dtype, out_stride, st);
}

int exl3_call(const void* words)
{
    const int64_t* w = static_cast<const int64_t*>(words);
    if (!w) return set_error("exl3_call: no arguments");
    switch (w[0] & 255)
    {
        case EXL3_CALL_ROUTE_LOGITS: return call_packed(exl3_route_logits, w);
        case EXL3_CALL_FP8_QUANTIZE_ROWS: return call_packed(exl3_fp8_quantize_rows, w);
        case EXL3_CALL_FP8_LINEAR: return call_packed(exl3_fp8_linear, w);
        case EXL3_CALL_FP8_MLP: return call_packed(exl3_fp8_mlp, w);
        case EXL3_CALL_FP8_EXPERTS: return call_packed(exl3_fp8_experts, w);
        default: return set_error("exl3_call: unknown call");
    }
}

}  // extern "C"
