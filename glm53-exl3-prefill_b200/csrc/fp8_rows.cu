// fp8_rows.cu — the row kernels of the 8-bit layers: quantising rows, and summing a token's routes.
#include "fp8_common.cuh"

namespace exl3b {

namespace {

using namespace fp8;

// ------------------------------------------------------------------------------------ quantised rows
//     s[r, b] = max(max_k |x[r, k]|, 2^-64) / 448   (or the least power of two at or above that)
//     q[r, k] = e4m3(x[r, k] / s[r, k / 128])       b = k / 128
// bound by bytes: a row is read once (2 or 4 bytes a value) and written once (1 byte).  Eight lanes hold a block,
// 16 values each, so loads are whole 32-byte sectors, the store is 16 bytes a lane, and a block's maximum is three shuffles.
// 8192 x 12288: fp16 to powers of two 53 us (47 by bytes), bf16 with exact scales 70 us, where the seven operations of quotient()
// for every value share the bound with the bytes.
struct QuantArgs {
    const void* x;
    int64_t x_stride;                // elements
    int K, n_blocks;
    uint8_t* q;
    int64_t q_stride;
    float* scale;
    int64_t s_row, s_blk;            // element strides of the scales
    int64_t rows;
    // gather (optional): row r holds x[slot[r] / topk]; only the first *rows_dev rows exist
    const int64_t* slot;
    int topk;
    const int32_t* rows_dev;
};

constexpr int Q_THREADS = 256;

// 32 bytes from a 32-byte (16-byte) aligned address.
template <bool ALIGNED32>
__device__ __forceinline__ void load32(const void* src, uint32_t* w)
{
    if constexpr (ALIGNED32)
        asm volatile("ld.global.nc.v8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
                     : "=r"(w[0]), "=r"(w[1]), "=r"(w[2]), "=r"(w[3]), "=r"(w[4]), "=r"(w[5]), "=r"(w[6]), "=r"(w[7])
                     : "l"(src));
    else
    {
        reinterpret_cast<uint4*>(w)[0] = __ldg(reinterpret_cast<const uint4*>(src));
        reinterpret_cast<uint4*>(w)[1] = __ldg(reinterpret_cast<const uint4*>(src) + 1);
    }
}

// ALIGN: 32 or 16 bytes (rows and K allow vectors), 0: element by element.  Index: type of a (row, block) number.
template <class T, int ALIGN, bool POW2, class Index>
__global__ __launch_bounds__(Q_THREADS)
void quantize_rows_kernel(const QuantArgs p)
{
    let_next_launch_start();
    wait_for_previous_launch();
    const int lane8 = threadIdx.x & 7;
    const int64_t rows = p.rows_dev ? min(p.rows, (int64_t) *p.rows_dev) : p.rows;
    const Index units = (Index) (rows * p.n_blocks);                // (row, block) pairs, blocks fastest
    const Index step = (Index) gridDim.x * (Q_THREADS / 8);
    // whole warps take part in the shuffles: the bound is rounded up to the warp's four units
    const Index first = ((Index) blockIdx.x * Q_THREADS + threadIdx.x) >> 3;
    for (Index u = first; u - (first & 3) < units; u += step)
    {
        const bool live = u < units;
        const Index row = live ? u / (Index) p.n_blocks : 0;
        const int b = live ? (int) (u - row * (Index) p.n_blocks) : 0;
        const int64_t r = (int64_t) row;
        const int64_t src = p.slot && live ? (int64_t) ((uint32_t) __ldg(p.slot + r) / (uint32_t) p.topk) : r;
        const int k0 = b * kBlock + lane8 * 16;
        const T* x = reinterpret_cast<const T*>(p.x) + src * p.x_stride + k0;
        float v[16];
        uint32_t m = 0;                                             // magnitudes as integers: NaN is the largest
        if (live && ALIGN && k0 < p.K)                              // K % 16 == 0
        {
            __align__(16) uint32_t w[4 * sizeof(T)];
            #pragma unroll
            for (int j = 0; j < (int) sizeof(T) / 2; ++j)
                load32<ALIGN == 32>(reinterpret_cast<const uint8_t*>(x) + 32 * j, w + 8 * j);
            const T* h = reinterpret_cast<const T*>(w);
            #pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = to_float(h[i]);
            if constexpr (sizeof(T) == 2)
            {
                // 16-bit magnitudes two at a time: 12 instructions instead of 32
                uint32_t m2 = 0;
                #pragma unroll
                for (int i = 0; i < 8; i += 2) m2 = __vimax3_u16x2(m2, w[i] & 0x7fff7fffu, w[i + 1] & 0x7fff7fffu);
                const uint16_t top = (uint16_t) max(m2 & 0xffffu, m2 >> 16);
                T t;
                memcpy(&t, &top, 2);
                m = __float_as_uint(to_float(t));
            }
        }
        else
        {
            #pragma unroll
            for (int i = 0; i < 16; ++i) v[i] = !ALIGN && live && k0 + i < p.K ? to_float(x[i]) : 0.0f;
        }
        if (!ALIGN || sizeof(T) == 4)
            #pragma unroll
            for (int i = 0; i < 16; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        #pragma unroll
        for (int o = 1; o < 8; o <<= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (!live) continue;
        const float s = block_scale(__uint_as_float(m), POW2);
        const float inv = POW2 ? 1.0f / s : reciprocal(s);
        uint32_t w[4];
        #pragma unroll
        for (int i = 0; i < 16; ++i) v[i] = POW2 ? v[i] * inv : quotient(v[i], s, inv);    // powers of two: exact
        #pragma unroll
        for (int j = 0; j < 4; ++j) w[j] = to_e4m3x2(v[4 * j], v[4 * j + 1]) | to_e4m3x2(v[4 * j + 2], v[4 * j + 3]) << 16;
        uint8_t* q = p.q + r * p.q_stride + k0;
        if (ALIGN)
        {
            if (k0 < p.K) *reinterpret_cast<uint4*>(q) = make_uint4(w[0], w[1], w[2], w[3]);
        }
        else
        {
            #pragma unroll
            for (int i = 0; i < 16; ++i)
                if (k0 + i < p.K) q[i] = (uint8_t) (w[i >> 2] >> (8 * (i & 3)));
        }
        if (lane8 == 0) p.scale[r * p.s_row + b * p.s_blk] = s;
    }
}

// ------------------------------------------------------------------------------------ rows by route
// Quantised rows of tokens copied to their routes' places: row r of q, s is token slot[r] / topk's.  With many routes per
// token this is cheaper than quantising every route's copy (65536 routes of 4096 columns from 8192 tokens: 206 us).
struct GatherArgs {
    const uint8_t* q;
    const float* s;                  // [blocks][tokens]
    int64_t tokens;
    const int64_t* slot;
    int topk, d;
    const int32_t* rows_dev;
    uint8_t* q_out;
    float* s_out;                    // [blocks][rows]
    int64_t rows;
};

__global__ __launch_bounds__(256)
void gather_rows_kernel(const GatherArgs p)
{
    let_next_launch_start();
    wait_for_previous_launch();
    const int lane = threadIdx.x & 31;
    const int64_t rows = min(p.rows, (int64_t) *p.rows_dev), n = p.d / 16;
    for (int64_t r = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5); r < rows; r += (int64_t) gridDim.x * 8)
    {
        const int64_t t = (int64_t) ((uint32_t) p.slot[r] / (uint32_t) p.topk);
        const uint4* src = reinterpret_cast<const uint4*>(p.q + t * p.d);
        uint4* dst = reinterpret_cast<uint4*>(p.q_out + r * p.d);
        for (int64_t i = lane; i < n; i += 128)
        {
            uint4 v[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + 32 * j < n) v[j] = src[i + 32 * j];
            #pragma unroll
            for (int j = 0; j < 4; ++j)
                if (i + 32 * j < n) dst[i + 32 * j] = v[j];
        }
        for (int b = lane; b < p.d / kBlock; b += 32) p.s_out[b * p.rows + r] = p.s[b * p.tokens + t];
    }
}

// ------------------------------------------------------------------------------------ sum over a token's routes
//     out[t] = (accumulate ? out[t] : 0) + sum over j ascending, ids[t, j] in [0, E), of w[t, j] * y[t * topk + j]
// in fp32 and a fixed order (no atomics), rounded once to out's type.  Bound by reading y, which is fp32 so that a result has one
// rounding: 65536 rows of 4096 (1.07 GB, part of it still to be written back) take 270 us.
struct CombineArgs {
    const float* y;
    int64_t y_stride;
    int parts;                       // y is the sum of this many, part_stride elements apart
    int64_t part_stride;
    const void* ids;
    int ids_i64;
    const void* weights;
    int wdtype;
    int64_t T;
    int topk, E, d, accumulate;
    void* out;
    int64_t out_stride;
};

// Four values as the sum of `parts` partial sums, in order.
__device__ __forceinline__ float4 sum_parts(const float* y, int parts, int64_t stride)
{
    float4 v = *reinterpret_cast<const float4*>(y);
    for (int i = 1; i < parts; ++i)
    {
        const float4 o = *reinterpret_cast<const float4*>(y + i * stride);
        v.x += o.x; v.y += o.y; v.z += o.z; v.w += o.w;
    }
    return v;
}

__device__ __forceinline__ float route_weight(const void* w, int dtype, int64_t i)
{
    if (dtype == 0) return __ldg(reinterpret_cast<const float*>(w) + i);
    if (dtype == 1) return __half2float(reinterpret_cast<const __half*>(w)[i]);
    return __bfloat162float(reinterpret_cast<const __nv_bfloat16*>(w)[i]);
}

template <class To>
__global__ __launch_bounds__(256)
void combine_routes_kernel(const CombineArgs p)
{
    let_next_launch_start();
    wait_for_previous_launch();
    const int64_t t = blockIdx.y + (int64_t) blockIdx.z * 65535;
    if (t >= p.T) return;
    const int c = (blockIdx.x * 256 + threadIdx.x) * 4;
    if (c >= p.d) return;                                           // d % 4 == 0
    To* out = reinterpret_cast<To*>(p.out) + t * p.out_stride + c;
    float a[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    if (p.accumulate)
        #pragma unroll
        for (int i = 0; i < 4; ++i) a[i] = to_float(out[i]);
    // routes whose loads are in flight together; they do not wait for the ids: rows of unrouted slots exist, and what
    // they hold is not used
    constexpr int AHEAD = 8;
    for (int j0 = 0; j0 < p.topk; j0 += AHEAD)
    {
        float4 v[AHEAD];
        bool valid[AHEAD];
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j)
        {
            const int64_t s = t * p.topk + j0 + j;
            valid[j] = j0 + j < p.topk;
            if (valid[j]) v[j] = *reinterpret_cast<const float4*>(p.y + s * p.y_stride + c);
        }
        float w[AHEAD];
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j)
        {
            const int64_t s = t * p.topk + j0 + j;
            if (!valid[j]) continue;
            const int64_t e = p.ids_i64 ? __ldg(reinterpret_cast<const long long*>(p.ids) + s)
                                        : (int64_t) __ldg(reinterpret_cast<const int*>(p.ids) + s);
            valid[j] = e >= 0 && e < p.E;
            w[j] = route_weight(p.weights, p.wdtype, s);
        }
        #pragma unroll
        for (int j = 0; j < AHEAD; ++j)
        {
            if (!valid[j]) continue;
            const int64_t s = t * p.topk + j0 + j;
            for (int i = 1; i < p.parts; ++i)
            {
                const float4 o = *reinterpret_cast<const float4*>(p.y + s * p.y_stride + c + i * p.part_stride);
                v[j].x += o.x; v[j].y += o.y; v[j].z += o.z; v[j].w += o.w;
            }
            a[0] = fmaf(w[j], v[j].x, a[0]);
            a[1] = fmaf(w[j], v[j].y, a[1]);
            a[2] = fmaf(w[j], v[j].z, a[2]);
            a[3] = fmaf(w[j], v[j].w, a[3]);
        }
    }
    #pragma unroll
    for (int i = 0; i < 4; ++i) out[i] = from_float<To>(a[i]);
}

// ------------------------------------------------------------------------------------ products split along K
// out[r, n] = (accumulate ? out[r, n] : 0) + the parts' sum; N is the valid width, parts hold rows of part_ld values.
struct JoinArgs {
    const float* part;
    int parts;
    int64_t part_stride, part_ld;
    int64_t rows;
    int N, accumulate;
    void* out;
    int64_t out_stride;
};

template <class To>
__global__ __launch_bounds__(256)
void join_parts_kernel(const JoinArgs p)
{
    let_next_launch_start();
    wait_for_previous_launch();
    const int per_row = (p.N + 3) / 4;
    for (int64_t u = (int64_t) blockIdx.x * 256 + threadIdx.x; u < p.rows * per_row; u += (int64_t) gridDim.x * 256)
    {
        const int64_t r = u / per_row;
        const int n = (int) (u - r * per_row) * 4;
        const float4 v = sum_parts(p.part + r * p.part_ld + n, p.parts, p.part_stride);
        const float a[4] = {v.x, v.y, v.z, v.w};
        To* o = reinterpret_cast<To*>(p.out) + r * p.out_stride + n;
        #pragma unroll
        for (int i = 0; i < 4; ++i)
            if (n + i < p.N) o[i] = from_float<To>(p.accumulate ? to_float(o[i]) + a[i] : a[i]);
    }
}

// The gate and up halves of a row (columns 0..f-1 and f..2f-1 of the parts) to quantised activations: a warp per row and block of
// 128 columns, 4 a lane.
struct ActArgs {
    const float* part;
    int parts;
    int64_t part_stride, part_ld;
    int64_t rows;
    const int32_t* rows_dev;
    int f;
    float limit;
    uint8_t* h;
    int64_t h_stride;
    float* hs;
    int64_t hs_row, hs_blk;
};

__global__ __launch_bounds__(256)
void act_parts_kernel(const ActArgs p)
{
    let_next_launch_start();
    wait_for_previous_launch();
    const int lane = threadIdx.x & 31, blocks = p.f / kBlock;
    const int64_t rows = p.rows_dev ? min(p.rows, (int64_t) *p.rows_dev) : p.rows;
    for (int64_t u = (int64_t) blockIdx.x * 8 + (threadIdx.x >> 5); u < rows * blocks; u += (int64_t) gridDim.x * 8)
    {
        const int64_t r = u / blocks;
        const int b = (int) (u - r * blocks);
        const float* y = p.part + r * p.part_ld + b * kBlock + 4 * lane;
        const float4 g = sum_parts(y, p.parts, p.part_stride), w = sum_parts(y + p.f, p.parts, p.part_stride);
        const float a[4] = {clamped_swiglu(g.x, w.x, p.limit), clamped_swiglu(g.y, w.y, p.limit),
                            clamped_swiglu(g.z, w.z, p.limit), clamped_swiglu(g.w, w.w, p.limit)};
        uint32_t m = 0;
        #pragma unroll
        for (int i = 0; i < 4; ++i) m = max(m, __float_as_uint(a[i]) & 0x7fffffffu);
        const float s = block_scale(__uint_as_float(__reduce_max_sync(0xffffffffu, m)), false), inv = reciprocal(s);
        float q[4];
        #pragma unroll
        for (int i = 0; i < 4; ++i) q[i] = quotient(a[i], s, inv);
        reinterpret_cast<uint32_t*>(p.h + r * p.h_stride + b * kBlock)[lane] =
            to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
        if (lane == 0) p.hs[r * p.hs_row + b * p.hs_blk] = s;
    }
}

template <class T, int ALIGN>
int launch_quant(const QuantArgs& p, bool pow2, unsigned grid, bool after, cudaStream_t stream)
{
    auto go = [&](void (*kernel)(QuantArgs)) {
        if (after) return launch_after("fp8_quantize_rows", kernel, dim3(grid), Q_THREADS, 0, stream, p);
        kernel<<<grid, Q_THREADS, 0, stream>>>(p);
        return check_launch("fp8_quantize_rows");
    };
    const bool small = p.rows * p.n_blocks < (1LL << 31);           // (row, block) numbers fit 32 bits: cheap divisions
    if (pow2)
        return go(small ? quantize_rows_kernel<T, ALIGN, true, uint32_t> : quantize_rows_kernel<T, ALIGN, true, uint64_t>);
    return go(small ? quantize_rows_kernel<T, ALIGN, false, uint32_t> : quantize_rows_kernel<T, ALIGN, false, uint64_t>);
}

}  // namespace

int launch_fp8_quantize(const void* x, int dtype, int64_t rows, int K, int64_t x_stride, int pow2, void* q,
                        int64_t q_stride, float* scale, int64_t s_row, int64_t s_blk, const int64_t* slot, int topk,
                        const int32_t* rows_dev, bool after, cudaStream_t stream)
{
    QuantArgs p{};
    p.x = x; p.x_stride = x_stride; p.K = K; p.n_blocks = (K + kBlock - 1) / kBlock;
    p.q = static_cast<uint8_t*>(q); p.q_stride = q_stride; p.scale = scale; p.s_row = s_row; p.s_blk = s_blk;
    p.rows = rows; p.slot = slot; p.topk = topk; p.rows_dev = rows_dev;
    const int64_t size = dtype == 0 ? 4 : 2;
    const uintptr_t at = reinterpret_cast<uintptr_t>(x) | (uintptr_t) (x_stride * size);
    int align = K % 16 == 0 && q_stride % 16 == 0 && reinterpret_cast<uintptr_t>(q) % 16 == 0 ? 32 : 0;
    if (at % 32 != 0) align = align && at % 16 == 0 ? 16 : 0;
    const int64_t ctas = (rows * p.n_blocks + Q_THREADS / 8 - 1) / (Q_THREADS / 8);
    const int64_t most = (int64_t) device_sm_count() * 64;
    const unsigned grid = (unsigned) (ctas < most ? ctas : most);
    auto go = [&](auto v) {
        using T = decltype(v);
        if (align == 32) return launch_quant<T, 32>(p, pow2 != 0, grid, after, stream);
        if (align == 16) return launch_quant<T, 16>(p, pow2 != 0, grid, after, stream);
        return launch_quant<T, 0>(p, pow2 != 0, grid, after, stream);
    };
    if (dtype == 0) return go(float{});
    if (dtype == 1) return go(__half{});
    return go(__nv_bfloat16{});
}

int launch_fp8_gather(const void* q, const float* s, int64_t tokens, const int64_t* slot, int topk, int d,
                      const int32_t* rows_dev, void* q_out, float* s_out, int64_t rows, cudaStream_t stream)
{
    const GatherArgs p{static_cast<const uint8_t*>(q), s, tokens, slot, topk, d, rows_dev, static_cast<uint8_t*>(q_out),
                       s_out, rows};
    const int64_t ctas = (rows + 7) / 8, most = (int64_t) device_sm_count() * 16;
    return launch_after("fp8_gather", gather_rows_kernel, dim3((unsigned) (ctas < most ? ctas : most)), 256, 0, stream, p);
}

int launch_fp8_combine(const float* y, int64_t y_stride, int parts, int64_t part_stride, const void* ids, int ids_i64,
                       const void* weights, int wdtype, int64_t T, int topk, int E, int d, int accumulate, void* out,
                       int out_dtype, int64_t out_stride, cudaStream_t stream)
{
    const CombineArgs p{y, y_stride, parts, part_stride, ids, ids_i64, weights, wdtype, T, topk, E, d, accumulate, out,
                        out_stride};
    const dim3 grid((unsigned) ((d / 4 + 255) / 256), (unsigned) (T < 65535 ? T : 65535), (unsigned) ((T + 65534) / 65535));
    const char* what = "fp8_combine";
    if (out_dtype == 0) return launch_after(what, combine_routes_kernel<float>, grid, 256, 0, stream, p);
    if (out_dtype == 1) return launch_after(what, combine_routes_kernel<__half>, grid, 256, 0, stream, p);
    return launch_after(what, combine_routes_kernel<__nv_bfloat16>, grid, 256, 0, stream, p);
}

int launch_fp8_join(const float* part, int parts, int64_t part_stride, int64_t part_ld, int64_t rows, int N, int accumulate,
                    void* out, int out_dtype, int64_t out_stride, cudaStream_t stream)
{
    const JoinArgs p{part, parts, part_stride, part_ld, rows, N, accumulate, out, out_stride};
    const int64_t ctas = (rows * ((N + 3) / 4) + 255) / 256, most = (int64_t) device_sm_count() * 8;
    const dim3 grid((unsigned) (ctas < most ? ctas : most));
    const char* what = "fp8_join";
    if (out_dtype == 0) return launch_after(what, join_parts_kernel<float>, grid, 256, 0, stream, p);
    if (out_dtype == 1) return launch_after(what, join_parts_kernel<__half>, grid, 256, 0, stream, p);
    return launch_after(what, join_parts_kernel<__nv_bfloat16>, grid, 256, 0, stream, p);
}

int launch_fp8_act(const float* part, int parts, int64_t part_stride, int64_t part_ld, int64_t rows, const int32_t* rows_dev,
                   int f, float limit, void* h, int64_t h_stride, float* hs, int64_t hs_row, int64_t hs_blk,
                   cudaStream_t stream)
{
    const ActArgs p{part, parts, part_stride, part_ld, rows, rows_dev, f, limit, static_cast<uint8_t*>(h), h_stride, hs,
                    hs_row, hs_blk};
    const int64_t ctas = (rows * (f / kBlock) + 7) / 8, most = (int64_t) device_sm_count() * 8;
    return launch_after("fp8_act", act_parts_kernel, dim3((unsigned) (ctas < most ? ctas : most)), 256, 0, stream, p);
}

}  // namespace exl3b
