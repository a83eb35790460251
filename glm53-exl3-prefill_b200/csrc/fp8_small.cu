// fp8_small.cu — the 8-bit products for a few tokens, where reading the weights is all the time there is.
//
// A warp takes 16 weight rows and streams them from global memory straight into the A fragments of
// mma.sync m16n8k32 (e4m3, fp32 sums): lane (g, t) = (lane / 4, lane % 4) reads the 32 bytes t of a row's 128-byte K
// block, for rows g and g + 8, and the K order inside a block is permuted alike for both operands, so a fragment
// is what one 32-byte load brings.  No shared memory and no barrier before the sums; a row tile's K blocks are dealt in runs
// to a CTA's warps, whose sums are added in a fixed order at the end.  What counts is the number of warps that wait for memory:
// one block in flight in each of 32 warps per SM beats four in each of 16 (6.4 against 8.4 us for one token,
// 4096 x 4096, whose bytes take 2.6 us); neither rows copied to shared memory by the bulk-copy engine nor fp16
// products were faster, and prefetching a CTA's weight rows into L2 was slower (eight routes 45 us instead of 39).
//   one token of a projection, routes   rows are quantised on the way: a warp reads a block's 128 values (4 a lane), takes their
//               maximum, rounds them, and hands the words to the lanes whose fragment they belong to;
//   up to 16 tokens, plain MLPs         rows are quantised by their own kernel first and read as fragments from L2.
// The tcgen05 kernel needs 128 x 256 tiles and a pipeline to start up: 13 us for two tokens and 4096 x 4096 (5.7 here), whose
// bytes take 2.6 us.
#include "fp8_common.cuh"

namespace exl3b {

namespace {

using namespace fp8;

constexpr int S_WARPS = 8;                      // gate and up
constexpr int S_THREADS = S_WARPS * 32;
constexpr int T_WARPS = 16;                     // linear, down: a warp has half as many rows
constexpr int T_THREADS = T_WARPS * 32;

__device__ __forceinline__ void mma_e4m3(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                         uint32_t b1)
{
    asm volatile("mma.sync.aligned.m16n8k32.row.col.f32.e4m3.e4m3.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, "
                 "{%0, %1, %2, %3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

// The lane's 32 bytes of a row's K block `kb`: bytes 32 t .. 32 t + 31, zeros past K (a multiple of 16).  CONST: memory that
// nothing writes while the kernel runs (weights), for the read-only path.
template <bool ALIGNED32, bool CONST>
__device__ __forceinline__ void load_frag(const uint8_t* row, int kb, int t, int K, uint32_t (&w)[8])
{
    const int k = kb * kBlock + 32 * t;
    if (ALIGNED32 && k + 32 <= K)
    {
        if constexpr (CONST)
            asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(row + k));
        else
            asm volatile("ld.global.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                         : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                         : "l"(row + k) : "memory");
        return;
    }
    #pragma unroll
    for (int i = 0; i < 2; ++i)
    {
        uint4 v = make_uint4(0, 0, 0, 0);
        if (k + 16 * i < K) v = reinterpret_cast<const uint4*>(row + k)[i];
        w[4 * i] = v.x; w[4 * i + 1] = v.y; w[4 * i + 2] = v.z; w[4 * i + 3] = v.w;
    }
}

// Four consecutive values of a block (columns 4 lane .. 4 lane + 3 of block kb), zeros past K.  `vec`: 4-value loads.
template <class T>
__device__ __forceinline__ void load_values(const T* x, int kb, int lane, int K, bool vec, float (&v)[4])
{
    const int k = kb * kBlock + 4 * lane;
    if (vec && k + 4 <= K)
    {
        if constexpr (sizeof(T) == 4)
        {
            const float4 f = *reinterpret_cast<const float4*>(x + k);
            v[0] = f.x; v[1] = f.y; v[2] = f.z; v[3] = f.w;
        }
        else
        {
            const uint2 w = *reinterpret_cast<const uint2*>(x + k);
            const T* h = reinterpret_cast<const T*>(&w);
            #pragma unroll
            for (int i = 0; i < 4; ++i) v[i] = to_float(h[i]);
        }
        return;
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = k + i < K ? to_float(x[k + i]) : 0.0f;
}

// One block of a token's row, held four values a lane, quantised by the warp: its scale, and the fragment words of
// lane (g, t): column 0 is the token (g = 0), the other columns are zero.
__device__ __forceinline__ float quantize_block(const float (&v)[4], int lane, uint32_t (&b)[8])
{
    uint32_t m = 0;
    #pragma unroll
    for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
    const float s = block_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, m)), false), inv = reciprocal(s);
    float q[4];
    #pragma unroll
    for (int i = 0; i < 4; ++i) q[i] = quotient(v[i], s, inv);
    const uint32_t w = to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
    #pragma unroll
    for (int j = 0; j < 8; ++j)
    {
        const uint32_t x = __shfl_sync(0xffffffffu, w, 8 * (lane & 3) + j);
        b[j] = lane < 4 ? x : 0u;
    }
    return s;
}

// sums (c0: row g, c2: row g + 8, columns 2 t, 2 t + 1) of one 16-row tile and one K block
__device__ __forceinline__ void block_sums(const uint32_t (&lo)[8], const uint32_t (&hi)[8], const uint32_t (&b)[8],
                                           float (&c)[4])
{
    float o[4] = {0.0f, 0.0f, 0.0f, 0.0f};                  // two chains of two: half the latency
    c[0] = c[1] = c[2] = c[3] = 0.0f;
    #pragma unroll
    for (int i = 0; i < 4; i += 2)
    {
        mma_e4m3(c, lo[2 * i], hi[2 * i], lo[2 * i + 1], hi[2 * i + 1], b[2 * i], b[2 * i + 1]);
        mma_e4m3(o, lo[2 * i + 2], hi[2 * i + 2], lo[2 * i + 3], hi[2 * i + 3], b[2 * i + 2], b[2 * i + 3]);
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) c[i] += o[i];
}

// One token by NR tiles of 16 weight rows, K blocks kb0 <= kb < kb1: acc[r][0], acc[r][1] = rows g and g + 8 of tile r, in
// the lanes with t = 0.  row[r][i]: this lane's weight rows; sw[r]: the tile's scales by K block.  One block of weights is
// in flight per warp; the first of them before the launch this one depends on has ended (x is only read after it).
template <int NR, bool ALIGNED32, class T>
__device__ __forceinline__ void stream_token(const uint8_t* const (&row)[NR][2], const float* const (&sw)[NR], const T* x,
                                             bool vec, int K, int kb0, int kb1, int lane, float (&acc)[NR][2])
{
    const int t = lane & 3;
    uint32_t a[NR][2][8];
    float f[NR], v[4];
    auto load_w = [&](int kb) {
        if (kb >= kb1) return;
        #pragma unroll
        for (int r = 0; r < NR; ++r)
        {
            #pragma unroll
            for (int i = 0; i < 2; ++i) load_frag<ALIGNED32, true>(row[r][i], kb, t, K, a[r][i]);
            f[r] = __ldg(sw[r] + kb);
        }
    };
    #pragma unroll
    for (int r = 0; r < NR; ++r) acc[r][0] = acc[r][1] = 0.0f;
    load_w(kb0);
    wait_for_previous_launch();
    if (kb0 < kb1) load_values(x, kb0, lane, K, vec, v);
    for (int kb = kb0; kb < kb1; ++kb)
    {
        uint32_t b[8];
        const float s = quantize_block(v, lane, b);
        #pragma unroll
        for (int r = 0; r < NR; ++r)
        {
            float c[4];
            block_sums(a[r][0], a[r][1], b, c);
            acc[r][0] = fmaf(c[0], s * f[r], acc[r][0]);
            acc[r][1] = fmaf(c[2], s * f[r], acc[r][1]);
        }
        load_w(kb + 1);
        if (kb + 1 < kb1) load_values(x, kb + 1, lane, K, vec, v);
    }
}

// ------------------------------------------------------------------------------------ linear, one token
struct SmallLinearArgs {
    const void* x;
    int vec;
    const uint8_t* q; int64_t q_stride;         // 1..16 tokens: quantised rows and their scales
    const float* sx; int64_t sx_row, sx_blk;
    int T, N, K;
    const uint8_t* w; int64_t w_stride;
    const float* sw; int64_t sw_n;
    void* out; int64_t out_stride; int out_dtype, accumulate;
};

__device__ __forceinline__ void put(void* out, int dtype, int64_t at, float v, bool accumulate)
{
    if (dtype == 0)
    {
        float* o = reinterpret_cast<float*>(out) + at;
        *o = accumulate ? *o + v : v;
    }
    else if (dtype == 1)
    {
        __half* o = reinterpret_cast<__half*>(out) + at;
        *o = __float2half_rn(accumulate ? __half2float(*o) + v : v);
    }
    else
    {
        __nv_bfloat16* o = reinterpret_cast<__nv_bfloat16*>(out) + at;
        *o = __float2bfloat16_rn(accumulate ? __bfloat162float(*o) + v : v);
    }
}

template <bool ALIGNED32, class T>
__global__ __launch_bounds__(T_THREADS, 2)
void linear_token_kernel(const SmallLinearArgs p)
{
    __shared__ float s_sum[T_WARPS][16];
    let_next_launch_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * 16, g = lane >> 2;
    const int nkb = (p.K + kBlock - 1) / kBlock;
    const uint8_t* const row[1][2] = {{p.w + (int64_t) min(n0 + g, p.N - 1) * p.w_stride,
                                       p.w + (int64_t) min(n0 + g + 8, p.N - 1) * p.w_stride}};
    const float* const sw[1] = {p.sw + (n0 / kBlock) * p.sw_n};
    float acc[1][2];
    stream_token<1, ALIGNED32>(row, sw, reinterpret_cast<const T*>(p.x), p.vec != 0, p.K, warp * nkb / T_WARPS,
                                   (warp + 1) * nkb / T_WARPS, lane, acc);
    if ((lane & 3) == 0)
    {
        s_sum[warp][g] = acc[0][0];
        s_sum[warp][g + 8] = acc[0][1];
    }
    __syncthreads();
    const int n = n0 + threadIdx.x;
    if (threadIdx.x < 16 && n < p.N)
    {
        float v = 0.0f;
        #pragma unroll
        for (int w = 0; w < T_WARPS; ++w) v += s_sum[w][threadIdx.x];
        put(p.out, p.out_dtype, n, v, p.accumulate != 0);
    }
}

// 1..16 tokens: NG groups of 8 columns.
template <int NG, int WARPS, bool ALIGNED32>
__global__ __launch_bounds__(WARPS * 32, 2)
void linear_tokens_kernel(const SmallLinearArgs p)
{
    constexpr int DEPTH = NG;                              // blocks of weights in flight per warp
    __shared__ float s_sum[WARPS][16][NG * 8];
    let_next_launch_start();
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n0 = blockIdx.x * 16, g = lane >> 2, t = lane & 3;
    const int nkb = (p.K + kBlock - 1) / kBlock;
    const uint8_t* row0 = p.w + (int64_t) min(n0 + g, p.N - 1) * p.w_stride;
    const uint8_t* row1 = p.w + (int64_t) min(n0 + g + 8, p.N - 1) * p.w_stride;
    const float* sw = p.sw + (n0 / kBlock) * p.sw_n;
    float acc[NG][4];
    #pragma unroll
    for (int j = 0; j < NG; ++j) acc[j][0] = acc[j][1] = acc[j][2] = acc[j][3] = 0.0f;
    const int kb0 = warp * nkb / WARPS, kb1 = (warp + 1) * nkb / WARPS;
    uint32_t a[DEPTH][2][8];
    float f[DEPTH];
    auto load_w = [&](int u, int kb) {
        if (kb >= kb1) return;
        load_frag<ALIGNED32, true>(row0, kb, t, p.K, a[u][0]);
        load_frag<ALIGNED32, true>(row1, kb, t, p.K, a[u][1]);
        f[u] = __ldg(sw + kb);
    };
    #pragma unroll
    for (int u = 0; u < DEPTH; ++u) load_w(u, kb0 + u);
    wait_for_previous_launch();
    for (int kb = kb0; kb < kb1; kb += DEPTH)
    {
        #pragma unroll
        for (int u = 0; u < DEPTH; ++u)
        {
            const int k = kb + u;
            if (k >= kb1) break;
            #pragma unroll
            for (int j = 0; j < NG; ++j)
            {
                // a column past the last token repeats it; its sums are not stored
                uint32_t b[8];
                load_frag<ALIGNED32, false>(p.q + (int64_t) min(8 * j + g, p.T - 1) * p.q_stride, k, t, p.K, b);
                const float f0 = p.sx[min(8 * j + 2 * t, p.T - 1) * p.sx_row + k * p.sx_blk] * f[u];
                const float f1 = p.sx[min(8 * j + 2 * t + 1, p.T - 1) * p.sx_row + k * p.sx_blk] * f[u];
                float c[4];
                block_sums(a[u][0], a[u][1], b, c);
                acc[j][0] = fmaf(c[0], f0, acc[j][0]);
                acc[j][1] = fmaf(c[1], f1, acc[j][1]);
                acc[j][2] = fmaf(c[2], f0, acc[j][2]);
                acc[j][3] = fmaf(c[3], f1, acc[j][3]);
            }
            load_w(u, k + DEPTH);
        }
    }
    #pragma unroll
    for (int j = 0; j < NG; ++j)
    {
        s_sum[warp][g][8 * j + 2 * t] = acc[j][0];
        s_sum[warp][g][8 * j + 2 * t + 1] = acc[j][1];
        s_sum[warp][g + 8][8 * j + 2 * t] = acc[j][2];
        s_sum[warp][g + 8][8 * j + 2 * t + 1] = acc[j][3];
    }
    __syncthreads();
    if (threadIdx.x < 16 * NG * 8)
    {
        const int n = n0 + (threadIdx.x & 15), m = threadIdx.x >> 4;
        if (n < p.N && m < p.T)
        {
            float v = 0.0f;
            #pragma unroll
            for (int w = 0; w < WARPS; ++w) v += s_sum[w][threadIdx.x & 15][m];
            put(p.out, p.out_dtype, m * p.out_stride + n, v, p.accumulate != 0);
        }
    }
}

// ------------------------------------------------------------------------------------ routed experts, a few routes
struct SmallExpertArgs {
    const void* x; int64_t x_stride; int vec;
    const void* ids; int ids_i64;
    const void* weights; int wdtype;
    int T, topk, E, d, f;
    const uint8_t* w13; const float* s13;
    const uint8_t* w2; const float* s2;
    float limit;
    float* act;                                 // [T * topk, f]
    void* out; int64_t out_stride; int out_dtype, accumulate;
};

__device__ __forceinline__ int64_t route_expert(const SmallExpertArgs& p, int64_t slot)
{
    return p.ids_i64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + slot)
                     : (int64_t) __ldg(reinterpret_cast<const int*>(p.ids) + slot);
}

__device__ __forceinline__ float weight_of(const SmallExpertArgs& p, int64_t slot)
{
    if (p.wdtype == 0) return __ldg(reinterpret_cast<const float*>(p.weights) + slot);
    if (p.wdtype == 1) return __half2float(reinterpret_cast<const __half*>(p.weights)[slot]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(p.weights)[slot]);
}

// Gate and up rows n0 .. n0 + 15 of the expert of route blockIdx.y: act = silu(min(g, L)) * clamp(u, -L, L), fp32.
// Two CTAs an SM, without spills: 8 / 16 routes of 4096 x 1536 in 39.1 / 72.4 us; three, with spills, 39.4 / 74.0; gate and up
// rows in different warps, four CTAs, 40.5 / 70.  ALIGNED32: the weights start on 32 bytes (rows are multiples of 128).
template <bool ALIGNED32, class T>
__global__ __launch_bounds__(S_THREADS, 2)
void gate_up_token_kernel(const SmallExpertArgs p)
{
    __shared__ float s_sum[S_WARPS][32];
    const int64_t slot = blockIdx.y;
    const int64_t e = route_expert(p, slot);
    let_next_launch_start();
    if (e < 0 || e >= p.E) return;                                  // no expert: the combine leaves the route out
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int n0 = blockIdx.x * 16, nkb = p.d / kBlock;
    const uint8_t* w = p.w13 + e * 2 * p.f * p.d;
    const float* s = p.s13 + e * (2 * p.f / kBlock) * nkb;
    const uint8_t* const row[2][2] = {{w + (int64_t) (n0 + g) * p.d, w + (int64_t) (n0 + g + 8) * p.d},
                                      {w + (int64_t) (p.f + n0 + g) * p.d, w + (int64_t) (p.f + n0 + g + 8) * p.d}};
    const float* const sw[2] = {s + (n0 / kBlock) * nkb, s + ((p.f + n0) / kBlock) * nkb};
    float acc[2][2];
    stream_token<2, ALIGNED32>(row, sw, reinterpret_cast<const T*>(p.x) + slot / p.topk * p.x_stride, p.vec != 0, p.d,
                             warp * nkb / S_WARPS, (warp + 1) * nkb / S_WARPS, lane, acc);
    if ((lane & 3) == 0)
        #pragma unroll
        for (int r = 0; r < 2; ++r)
        {
            s_sum[warp][16 * r + g] = acc[r][0];
            s_sum[warp][16 * r + g + 8] = acc[r][1];
        }
    __syncthreads();
    if (threadIdx.x < 16)
    {
        float gate = 0.0f, up = 0.0f;
        #pragma unroll
        for (int i = 0; i < S_WARPS; ++i)
        {
            gate += s_sum[i][threadIdx.x];
            up += s_sum[i][16 + threadIdx.x];
        }
        p.act[slot * p.f + n0 + threadIdx.x] = clamped_swiglu(gate, up, p.limit);
    }
}

// Output columns n0 .. n0 + 15 of token blockIdx.y: the activations quantised on the way, every route's product, and their
// weighted sum in slot order.  The (route, part of K) units of a token are dealt to the warps.
template <bool ALIGNED32>
__global__ __launch_bounds__(T_THREADS, 2)
void down_token_kernel(const SmallExpertArgs p)
{
    __shared__ float s_sum[32][16];                                 // [unit][row]: topk * parts units, at most 32
    const int64_t t = blockIdx.y;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2;
    const int n0 = blockIdx.x * 16, nkb = p.f / kBlock;
    const int parts = (T_WARPS + p.topk - 1) / p.topk;
    for (int u = warp; u < p.topk * parts; u += T_WARPS)
    {
        const int64_t slot = t * p.topk + u / parts;
        const int64_t e = route_expert(p, slot);
        if (e < 0 || e >= p.E) continue;
        const uint8_t* w = p.w2 + e * p.d * p.f;
        const uint8_t* const row[1][2] = {{w + (int64_t) (n0 + g) * p.f, w + (int64_t) (n0 + g + 8) * p.f}};
        const float* const sw[1] = {p.s2 + (e * (p.d / kBlock) + n0 / kBlock) * nkb};
        float acc[1][2];
        stream_token<1, ALIGNED32>(row, sw, p.act + slot * p.f, true, p.f, u % parts * nkb / parts,
                                   (u % parts + 1) * nkb / parts, lane, acc);
        if ((lane & 3) == 0)
        {
            s_sum[u][g] = acc[0][0];
            s_sum[u][g + 8] = acc[0][1];
        }
    }
    wait_for_previous_launch();                                     // (a warp without a unit has not)
    __syncthreads();
    if (threadIdx.x < 16)
    {
        float sum = 0.0f;
        for (int j = 0; j < p.topk; ++j)
        {
            const int64_t slot = t * p.topk + j;
            const int64_t e = route_expert(p, slot);
            if (e < 0 || e >= p.E) continue;
            float y = 0.0f;
            for (int i = 0; i < parts; ++i) y += s_sum[j * parts + i][threadIdx.x];
            sum = fmaf(weight_of(p, slot), y, sum);
        }
        put(p.out, p.out_dtype, t * p.out_stride + n0 + threadIdx.x, sum, p.accumulate != 0);
    }
}

}  // namespace

int launch_fp8_linear_token(const void* x, int dtype, int K, const void* w, int64_t w_stride, const float* sw, int64_t sw_n,
                            int N, void* out, int out_dtype, int accumulate, cudaStream_t stream)
{
    SmallLinearArgs p{};
    p.x = x; p.T = 1; p.N = N; p.K = K;
    p.vec = reinterpret_cast<uintptr_t>(x) % (dtype == 0 ? 16 : 8) == 0;
    p.w = static_cast<const uint8_t*>(w); p.w_stride = w_stride; p.sw = sw; p.sw_n = sw_n;
    p.out = out; p.out_stride = N; p.out_dtype = out_dtype; p.accumulate = accumulate;
    const bool a32 = reinterpret_cast<uintptr_t>(w) % 32 == 0 && w_stride % 32 == 0;
    const unsigned grid = (unsigned) ((N + 15) / 16);
    auto go = [&](auto v) {
        using T = decltype(v);
        if (a32) linear_token_kernel<true, T><<<grid, T_THREADS, 0, stream>>>(p);
        else linear_token_kernel<false, T><<<grid, T_THREADS, 0, stream>>>(p);
    };
    if (dtype == 0) go(float{});
    else if (dtype == 1) go(__half{});
    else go(__nv_bfloat16{});
    return check_launch("fp8_linear (one token)");
}

int launch_fp8_linear_tokens(const Fp8GemmProblem& q, cudaStream_t stream)
{
    SmallLinearArgs p{};
    p.q = static_cast<const uint8_t*>(q.x); p.q_stride = q.x_stride; p.sx = q.sx; p.sx_row = q.sx_row; p.sx_blk = q.sx_blk;
    p.T = (int) q.rows; p.N = q.N; p.K = q.K;
    p.w = static_cast<const uint8_t*>(q.w); p.w_stride = q.w_stride; p.sw = q.sw; p.sw_n = q.sw_n;
    p.out = q.out; p.out_stride = q.out_stride; p.out_dtype = q.out_dtype; p.accumulate = q.accumulate;
    const bool a32 = reinterpret_cast<uintptr_t>(q.w) % 32 == 0 && q.w_stride % 32 == 0 &&
                     reinterpret_cast<uintptr_t>(q.x) % 32 == 0 && q.x_stride % 32 == 0;
    const unsigned grid = (unsigned) ((q.N + 15) / 16);
    // two groups of columns need twice the registers, so half the warps with twice the blocks in flight
    const char* what = "fp8_linear (few tokens)";
    if (q.rows <= 8)
        return a32 ? launch_after(what, linear_tokens_kernel<1, T_WARPS, true>, dim3(grid), T_THREADS, 0, stream, p)
                   : launch_after(what, linear_tokens_kernel<1, T_WARPS, false>, dim3(grid), T_THREADS, 0, stream, p);
    return a32 ? launch_after(what, linear_tokens_kernel<2, S_WARPS, true>, dim3(grid), S_THREADS, 0, stream, p)
               : launch_after(what, linear_tokens_kernel<2, S_WARPS, false>, dim3(grid), S_THREADS, 0, stream, p);
}

int launch_fp8_experts_small(const void* x, int dtype, int T, int d, int64_t x_stride, const void* ids, int ids_i64,
                             const void* weights, int wdtype, int topk, int E, const void* w13, const float* s13,
                             const void* w2, const float* s2, int f, float limit, float* act, void* out, int out_dtype,
                             int64_t out_stride, int accumulate, cudaStream_t stream)
{
    SmallExpertArgs p{};
    p.x = x; p.x_stride = x_stride;
    p.vec = (reinterpret_cast<uintptr_t>(x) | (uintptr_t) (x_stride * (dtype == 0 ? 4 : 2))) % (dtype == 0 ? 16 : 8) == 0;
    p.ids = ids; p.ids_i64 = ids_i64; p.weights = weights; p.wdtype = wdtype;
    p.T = T; p.topk = topk; p.E = E; p.d = d; p.f = f;
    p.w13 = static_cast<const uint8_t*>(w13); p.s13 = s13; p.w2 = static_cast<const uint8_t*>(w2); p.s2 = s2;
    p.limit = limit; p.act = act;
    p.out = out; p.out_dtype = out_dtype; p.out_stride = out_stride; p.accumulate = accumulate;
    // (weights are 16-byte aligned, like those of the products by tiles)
    const dim3 grid((unsigned) (f / 16), (unsigned) (T * topk));
    const bool a13 = reinterpret_cast<uintptr_t>(w13) % 32 == 0, a2 = reinterpret_cast<uintptr_t>(w2) % 32 == 0;
    auto go = [&](auto v) {
        using Tx = decltype(v);
        if (a13) gate_up_token_kernel<true, Tx><<<grid, S_THREADS, 0, stream>>>(p);
        else gate_up_token_kernel<false, Tx><<<grid, S_THREADS, 0, stream>>>(p);
    };
    if (dtype == 0) go(float{});
    else if (dtype == 1) go(__half{});
    else go(__nv_bfloat16{});
    int rc = check_launch("fp8_experts (gate and up, few routes)");
    if (rc) return rc;
    return launch_after("fp8_experts (down, few routes)", a2 ? down_token_kernel<true> : down_token_kernel<false>,
                        dim3((unsigned) (d / 16), (unsigned) T), T_THREADS, 0, stream, p);
}

}  // namespace exl3b
