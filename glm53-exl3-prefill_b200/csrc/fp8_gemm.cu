// fp8_gemm.cu — products of quantised rows with e4m3 weights, one scale per row and 128 columns on one side
// and one per 128 x 128 block on the other (sm_100a, tcgen05 + TMA):
//
//     y[r, n] = sum over blocks b of sx[r, b] * sw[e, n / 128, b] * ( sum over k in b of qx[r, k] * qw[e, n, k] )
//
// for rows r of expert e (a plain layer is one expert).  Two epilogues:
//   store    y in fp32 / fp16 / bf16 at row r (optionally added to what is there) or at row slot[r];
//   swiglu   a = silu(min(g, L)) * clamp(u, -L, L) of the gate and up halves of y, quantised again:
//            e4m3 rows [rows, f] with one scale per row and 128 columns (the down product's input).
//
// The tensor core cannot apply fp32 scales per 128 columns of K, so each 128-deep block of K is one short
// accumulation in TMEM (four tcgen05.mma of K = 32, fp32), which epilogue warps take out, scale and add to
// fp32 sums in registers while the tensor core works on the next block in the other TMEM buffer.
//
// A tile is up to 128 rows (tokens) by 256 weight rows (two blocks of 128: neighbours, or the gate and up rows of
// the same columns for swiglu), in one of two orientations:
//   wide  (more than FG_THIN rows)  tokens are the MMA's M: TMEM lane = token, column = weight row.  The scale
//         is one register per thread, so the epilogue reads next to nothing from shared memory;
//   thin  weights are M: lane = weight row, column = token, N = the tile's rows rounded up to 16, so an
//         expert with few rows costs few columns.  Here every value needs its column's scale, which a warp reads from
//         shared memory (128 bytes a clock for the SM, operands of the MMA included): 8 clocks per column and
//         K block, 1024 for 128 columns, where the MMA takes 512.  Up to 64 columns it is the cheaper form.
//
//   warp 0        TMA producer: weight blocks [128 x 128 B] x 2 and token rows in boxes of 32, 128-byte swizzle;
//   warp 1        MMA issuer, TMEM owner;
//   warps 2, 3    scales: sx * sw of the coming K blocks into a shared-memory ring, loaded one group ahead;
//   warps 4..11   two warpgroups of epilogue: warpgroup g takes 64 columns of each block (wide), or every other
//                 chunk of 16 columns (thin).
// Persistent CTAs walk the tiles (expert, weight tile, token tile; token tiles fastest, so the CTAs running at
// one time share weight tiles through L2).  Every wait is bounded as in the trellis kernels.
#include <cuda.h>

#include "fp8_common.cuh"
#include "trellis_common.cuh"

namespace exl3b {

namespace {

using namespace fp8;

constexpr int FG_THREADS = 384;
constexpr int FG_BK = 128;                                  // K bytes per stage: one 128-byte swizzle atom
constexpr uint32_t FG_W_BYTES = 128 * FG_BK;                // one block of weight rows
constexpr int FG_XBOX = 32;                                 // token rows per TMA box
constexpr int NT = 128;                                     // token rows of a tile
constexpr int FG_THIN = 64;                                 // most rows of a thin tile
constexpr int FG_STAGES = 4;
constexpr uint32_t FG_STAGE_BYTES = 2 * FG_W_BYTES + NT * FG_BK;
constexpr int FG_SCALES = 8;                                // slots of the scale ring
constexpr uint64_t FG_DRAIN_NS = 200000000ull;

struct Fp8GemmArgs {
    int N, K, n_experts;
    int n_tiles_n, num_kb;
    int single_count;                // rows of the one expert when counts is null
    const int32_t* counts;           // [E] or null
    const int32_t* row0;             // [E] first row of each expert, or null
    const float* sx; int64_t sx_row, sx_blk;
    const float* sw; int64_t sw_expert, sw_n, sw_k;
    // store
    void* out; int64_t out_stride; int out_dtype; int accumulate;
    int out_vec;                     // rows are 16-byte aligned
    const int64_t* slot;             // output row of row r, or null
    // swiglu
    int f; float limit;
    uint8_t* h; int64_t h_stride; float* hs; int64_t hs_row, hs_blk;
    int32_t* status;
    uint64_t wait_ns;
};

__device__ __forceinline__ void umma_e4m3(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                          uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// Instruction descriptor, kind::f8f6f4: D fp32, A and B e4m3 (both K-major), shape M x N.
__device__ __forceinline__ uint32_t idesc_e4m3_f32(int M, int N)
{
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

__device__ __forceinline__ void tma_load_3d(void* smem_dst, const void* tmap, int32_t x, int32_t y, int32_t z,
                                            uint64_t* bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
        : "memory");
}

// 32 (16) consecutive columns of this warp's 32 TMEM lanes as register pairs, complete on return.
__device__ __forceinline__ void tmem_load(uint32_t taddr, uint64_t (&d)[16])
{
    asm volatile(
        "{\n\t.reg .b32 t<32>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
        "{t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10, t11, t12, t13, t14, t15, t16, t17, t18, t19, t20, t21, t22, t23, t24, t25, t26, t27, t28, t29, t30, t31}, [%16];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {t0, t1};\n\t"
        "mov.b64 %1, {t2, t3};\n\t"
        "mov.b64 %2, {t4, t5};\n\t"
        "mov.b64 %3, {t6, t7};\n\t"
        "mov.b64 %4, {t8, t9};\n\t"
        "mov.b64 %5, {t10, t11};\n\t"
        "mov.b64 %6, {t12, t13};\n\t"
        "mov.b64 %7, {t14, t15};\n\t"
        "mov.b64 %8, {t16, t17};\n\t"
        "mov.b64 %9, {t18, t19};\n\t"
        "mov.b64 %10, {t20, t21};\n\t"
        "mov.b64 %11, {t22, t23};\n\t"
        "mov.b64 %12, {t24, t25};\n\t"
        "mov.b64 %13, {t26, t27};\n\t"
        "mov.b64 %14, {t28, t29};\n\t"
        "mov.b64 %15, {t30, t31};\n\t"
        "}"
        : "=l"(d[0]), "=l"(d[1]), "=l"(d[2]), "=l"(d[3]), "=l"(d[4]), "=l"(d[5]), "=l"(d[6]), "=l"(d[7]), "=l"(d[8]), "=l"(d[9]), "=l"(d[10]), "=l"(d[11]), "=l"(d[12]), "=l"(d[13]), "=l"(d[14]), "=l"(d[15])
        : "r"(taddr));
}

__device__ __forceinline__ void tmem_load(uint32_t taddr, uint64_t (&d)[8])
{
    asm volatile(
        "{\n\t.reg .b32 t<16>;\n\t"
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{t0, t1, t2, t3, t4, t5, t6, t7, t8, t9, t10, t11, t12, t13, t14, t15}, [%8];\n\t"
        "tcgen05.wait::ld.sync.aligned;\n\t"
        "mov.b64 %0, {t0, t1};\n\t"
        "mov.b64 %1, {t2, t3};\n\t"
        "mov.b64 %2, {t4, t5};\n\t"
        "mov.b64 %3, {t6, t7};\n\t"
        "mov.b64 %4, {t8, t9};\n\t"
        "mov.b64 %5, {t10, t11};\n\t"
        "mov.b64 %6, {t12, t13};\n\t"
        "mov.b64 %7, {t14, t15};\n\t"
        "}"
        : "=l"(d[0]), "=l"(d[1]), "=l"(d[2]), "=l"(d[3]), "=l"(d[4]), "=l"(d[5]), "=l"(d[6]), "=l"(d[7])
        : "r"(taddr));
}

// Two fp32 values in a 64-bit register pair (column 2i in the low half).
__device__ __forceinline__ uint64_t pack2(uint32_t lo, uint32_t hi)
{
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "r"(lo), "r"(hi));
    return r;
}

__device__ __forceinline__ float half_of(uint64_t v, int i)
{
    uint32_t lo, hi;
    asm("mov.b64 {%0, %1}, %2;" : "=r"(lo), "=r"(hi) : "l"(v));
    return __uint_as_float(i ? hi : lo);
}

// a += d * s for two columns at once.
__device__ __forceinline__ void fma2(uint64_t& a, uint64_t d, uint64_t s)
{
    asm("fma.rn.f32x2 %0, %1, %2, %0;" : "+l"(a) : "l"(d), "l"(s));
}

struct Tile {
    bool thin;
    int e, nt, row0, rows, nh;       // nh: weight blocks with rows (1 at the end of an odd number of blocks)
};

template <bool SWIGLU>
__device__ __forceinline__ Tile tile_at(const Fp8GemmArgs& p, const int* pref, int t)
{
    Tile ti;
    ti.e = trellis::prefix_find(pref, p.n_experts, t / p.n_tiles_n);
    const int mts = pref[ti.e + 1] - pref[ti.e];
    const int local = t - pref[ti.e] * p.n_tiles_n;
    ti.nt = local / mts;
    const int mt = local - ti.nt * mts;
    const int count = p.counts ? __ldg(p.counts + ti.e) : p.single_count;
    ti.row0 = (p.row0 ? __ldg(p.row0 + ti.e) : 0) + mt * NT;
    ti.rows = min(NT, count - mt * NT);
    ti.thin = ti.rows <= FG_THIN;
    ti.nh = SWIGLU || ti.nt * 256 + 128 < p.N ? 2 : 1;
    return ti;
}

// Weight block (of 128 rows) that is half h of tile column nt.
template <bool SWIGLU>
__device__ __forceinline__ int weight_block(const Fp8GemmArgs& p, int nt, int h)
{
    return SWIGLU ? h * (p.f / kBlock) + nt : 2 * nt + h;
}

constexpr int FG_STEP = 8;                                  // tokens staged at a time by a warpgroup

// Eight consecutive outputs of one row.
template <class To>
__device__ __forceinline__ void store8(const Fp8GemmArgs& p, int64_t r, int n, const float* v)
{
    To* o = reinterpret_cast<To*>(p.out) + r * p.out_stride + n;
    float a[8];
    *reinterpret_cast<float4*>(a) = *reinterpret_cast<const float4*>(v);
    *reinterpret_cast<float4*>(a + 4) = *reinterpret_cast<const float4*>(v + 4);
    if (p.out_vec && !p.accumulate && n + 8 <= p.N)
    {
        __align__(16) To w[8];
        #pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = from_float<To>(a[i]);
        #pragma unroll
        for (int i = 0; i < (int) sizeof(w) / 16; ++i) reinterpret_cast<uint4*>(o)[i] = reinterpret_cast<const uint4*>(w)[i];
        return;
    }
    #pragma unroll
    for (int i = 0; i < 8; ++i)
        if (n + i < p.N) o[i] = from_float<To>(p.accumulate ? to_float(o[i]) + a[i] : a[i]);
}

// Thin tiles: the staged tokens [m0, m0 + FG_STEP) x 256 weight rows, by the 128 threads of a warpgroup.
template <bool SWIGLU>
__device__ __forceinline__ void write_step(const Fp8GemmArgs& p, const Tile& ti, const float* st, int m0, int tid)
{
    if constexpr (!SWIGLU)
    {
        #pragma unroll 1
        for (int u = tid; u < FG_STEP * 32; u += 128)
        {
            const int m = m0 + (u >> 5), c = (u & 31) * 8, n = ti.nt * 256 + c;
            if (m >= ti.rows || n >= p.N) continue;
            const int64_t r = p.slot ? __ldg(p.slot + ti.row0 + m) : (int64_t) ti.row0 + m;
            const float* v = st + (u >> 5) * 256 + c;
            if (p.out_dtype == 0) store8<float>(p, r, n, v);
            else if (p.out_dtype == 1) store8<__half>(p, r, n, v);
            else store8<__nv_bfloat16>(p, r, n, v);
        }
    }
    else
    {
        // 16 lanes per token, 8 columns each; the block's largest magnitude is four shuffles
        const int m = m0 + (tid >> 4), c = tid & 15;
        const float* v = st + (tid >> 4) * 256 + c * 4;
        float a[8];
        uint32_t mx = 0;
        #pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            const float4 g = *reinterpret_cast<const float4*>(v + 64 * i);
            const float4 u = *reinterpret_cast<const float4*>(v + 64 * i + 128);
            a[4 * i] = clamped_swiglu(g.x, u.x, p.limit);
            a[4 * i + 1] = clamped_swiglu(g.y, u.y, p.limit);
            a[4 * i + 2] = clamped_swiglu(g.z, u.z, p.limit);
            a[4 * i + 3] = clamped_swiglu(g.w, u.w, p.limit);
            #pragma unroll
            for (int j = 0; j < 4; ++j) mx = max(mx, __float_as_uint(a[4 * i + j]) & 0x7fffffffu);
        }
        #pragma unroll
        for (int o = 1; o < 16; o <<= 1) mx = max(mx, __shfl_xor_sync(0xffffffffu, mx, o));
        if (m >= ti.rows) return;
        const float s = block_scale(__uint_as_float(mx), false), inv = 1.0f / s;
        const int64_t r = ti.row0 + m;
        uint32_t* h = reinterpret_cast<uint32_t*>(p.h + r * p.h_stride + ti.nt * kBlock) + c;
        #pragma unroll
        for (int i = 0; i < 2; ++i)
        {
            float q[4];
            #pragma unroll
            for (int j = 0; j < 4; ++j) q[j] = quotient(a[4 * i + j], s, inv);
            h[16 * i] = to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
        }
        if (c == 0) p.hs[r * p.hs_row + ti.nt * p.hs_blk] = s;
    }
}

// Wide tiles, store: this thread's token, 64 columns of each of the two weight blocks.
template <class To>
__device__ __forceinline__ void store_wide(const Fp8GemmArgs& p, const Tile& ti, const uint64_t (&acc)[2][32], int g, int m)
{
    if (m >= ti.rows) return;
    const int64_t r = p.slot ? __ldg(p.slot + ti.row0 + m) : (int64_t) ti.row0 + m;
    To* row = reinterpret_cast<To*>(p.out) + r * p.out_stride;
    constexpr int PER = 32 / sizeof(To);                    // values of a 32-byte sector
    #pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        const int n0 = ti.nt * 256 + h * 128 + g * 64;
        if (p.out_vec && !p.accumulate && n0 + 64 <= p.N)
        {
            #pragma unroll
            for (int c = 0; c < 64; c += PER)
            {
                __align__(16) To w[PER];
                #pragma unroll
                for (int i = 0; i < PER; ++i) w[i] = from_float<To>(half_of(acc[h][(c + i) >> 1], i & 1));
                const uint4* v = reinterpret_cast<const uint4*>(w);
                uint4* o = reinterpret_cast<uint4*>(row + n0 + c);
                o[0] = v[0];
                o[1] = v[1];
            }
        }
        else
        {
            #pragma unroll
            for (int c = 0; c < 64; ++c)
                if (n0 + c < p.N)
                {
                    float v = half_of(acc[h][c >> 1], c & 1);
                    if (p.accumulate) v += to_float(row[n0 + c]);
                    row[n0 + c] = from_float<To>(v);
                }
        }
    }
}

template <bool SWIGLU>
__global__ __launch_bounds__(FG_THREADS, 1)
void fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     const Fp8GemmArgs p)
{
    constexpr uint32_t TMEM_COLS = 512;                     // two buffers of 256 columns
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[FG_STAGES], bar_empty[FG_STAGES];
    __shared__ uint64_t bar_sfull[FG_SCALES], bar_sempty[FG_SCALES];
    __shared__ uint64_t bar_tfull[2], bar_tempty[2], bar_done;
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort, s_fail;
    __shared__ int s_pref[kMaxExperts + 1];
    __shared__ __align__(16) float s_scale[FG_SCALES][2][NT];
    __shared__ __align__(16) float s_stage[2][FG_STEP][256];
    __shared__ uint32_t s_amax[2][NT];

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    if (warp == 0)
    {
        // tiles of rows per expert, as an exclusive prefix
        const int per = (p.n_experts + 31) / 32;
        auto tiles = [&](int e) {
            return e < p.n_experts ? ((p.counts ? __ldg(p.counts + e) : p.single_count) + NT - 1) / NT : 0;
        };
        int sum = 0;
        for (int i = 0; i < per; ++i) sum += tiles(lane * per + i);
        int inc = sum;
        #pragma unroll
        for (int o = 1; o < 32; o <<= 1)
        {
            const int y = __shfl_up_sync(0xffffffffu, inc, o);
            if (lane >= o) inc += y;
        }
        int run = inc - sum;
        for (int i = 0; i < per; ++i)
            if (lane * per + i < p.n_experts)
            {
                s_pref[lane * per + i] = run;
                run += tiles(lane * per + i);
            }
        if (lane == 31) s_pref[p.n_experts] = inc;
    }
    if (warp == 1)
    {
        if (lane == 0)
        {
            for (int s = 0; s < FG_STAGES; ++s)
            {
                mbar_init(&bar_full[s], 1);
                mbar_init(&bar_empty[s], 1);
            }
            for (int s = 0; s < FG_SCALES; ++s)
            {
                mbar_init(&bar_sfull[s], 2);
                mbar_init(&bar_sempty[s], 8);
            }
            for (int b = 0; b < 2; ++b)
            {
                mbar_init(&bar_tfull[b], 1);
                mbar_init(&bar_tempty[b], 8);
            }
            mbar_init(&bar_done, 1);
            s_abort = 0;
            s_fail = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc(&s_tmem_base, TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem_base;
    volatile int* abort_flag = &s_abort;
    const int total = s_pref[p.n_experts] * p.n_tiles_n;
    const int nkb = p.num_kb;

    if (warp < 4)
    {
        setmaxnreg_dec<88>();
        if (warp == 0)
        {
            // ============================================================ TMA producer
            if (lane == 0)
            {
                int issued = 0;
                bool ok = true;
                for (int t = blockIdx.x; ok && t < total; t += gridDim.x)
                {
                    const Tile ti = tile_at<SWIGLU>(p, s_pref, t);
                    const int boxes = (ti.rows + FG_XBOX - 1) / FG_XBOX;
                    const uint32_t bytes = ti.nh * FG_W_BYTES + boxes * (FG_XBOX * FG_BK);
                    for (int kb = 0; kb < nkb; ++kb, ++issued)
                    {
                        const int s = issued % FG_STAGES;
                        const uint32_t ph = (issued / FG_STAGES) & 1u;
                        if (issued >= FG_STAGES && !mbar_wait(&bar_empty[s], ph ^ 1u, abort_flag, p.status, p.wait_ns))
                        {
                            ok = false;
                            break;
                        }
                        uint8_t* w = smem + s * FG_STAGE_BYTES;
                        mbar_arrive_expect_tx(&bar_full[s], bytes);
                        for (int h = 0; h < ti.nh; ++h)
                            tma_load_3d(w + h * FG_W_BYTES, &tmap_w, kb * FG_BK, weight_block<SWIGLU>(p, ti.nt, h) * kBlock,
                                        ti.e, &bar_full[s]);
                        for (int b = 0; b < boxes; ++b)
                            tma_load_2d(w + 2 * FG_W_BYTES + b * (FG_XBOX * FG_BK), &tmap_x, kb * FG_BK,
                                        ti.row0 + b * FG_XBOX, &bar_full[s]);
                    }
                }
                // copies in flight land before the CTA's shared memory goes away
                for (int i = issued > FG_STAGES ? issued - FG_STAGES : 0; i < issued; ++i)
                    mbar_drain(&bar_full[i % FG_STAGES], (i / FG_STAGES) & 1u, FG_DRAIN_NS);
            }
        }
        else if (warp == 1)
        {
            // ============================================================ MMA issuer
            if (lane == 0)
            {
                int it = 0;
                bool ok = true;
                for (int t = blockIdx.x; ok && t < total; t += gridDim.x)
                {
                    const Tile ti = tile_at<SWIGLU>(p, s_pref, t);
                    const uint32_t idesc = idesc_e4m3_f32(128, ti.thin ? (ti.rows + 15) & ~15 : ti.nh * 128);
                    for (int kb = 0; kb < nkb; ++kb, ++it)
                    {
                        const int s = it % FG_STAGES, b = it & 1;
                        if ((it >= 2 && !mbar_wait(&bar_tempty[b], ((it >> 1) & 1u) ^ 1u, abort_flag, p.status, p.wait_ns)) ||
                            !mbar_wait(&bar_full[s], (it / FG_STAGES) & 1u, abort_flag, p.status, p.wait_ns))
                        {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t w = smem_u32(smem + s * FG_STAGE_BYTES);
                        const uint64_t x_desc = smem_desc_sw128(w + 2 * FG_W_BYTES), w_desc = smem_desc_sw128(w);
                        const uint32_t d = tmem_base + b * 256;
                        if (ti.thin)
                        {
                            for (int h = 0; h < ti.nh; ++h)
                                #pragma unroll
                                for (int kk = 0; kk < FG_BK / 32; ++kk)
                                    umma_e4m3(d + h * 128, w_desc + h * (FG_W_BYTES >> 4) + 2 * kk, x_desc + 2 * kk, idesc, kk != 0);
                        }
                        else
                        {
                            #pragma unroll
                            for (int kk = 0; kk < FG_BK / 32; ++kk)
                                umma_e4m3(d, x_desc + 2 * kk, w_desc + 2 * kk, idesc, kk != 0);
                        }
                        umma_commit(&bar_empty[s]);
                        umma_commit(&bar_tfull[b]);
                    }
                }
                umma_commit(&bar_done);
                mbar_drain(&bar_done, 0, FG_DRAIN_NS);
            }
        }
        else
        {
            // ============================================================ scales
            constexpr int PER = NT >= 64 ? NT / 64 : 1;     // columns per lane
            constexpr int AHEAD = 4;                        // K blocks loaded together
            const int j0 = (warp - 2) * 32 + lane;
            int it = 0;
            bool ok = true;
            for (int t = blockIdx.x; ok && t < total; t += gridDim.x)
            {
                const Tile ti = tile_at<SWIGLU>(p, s_pref, t);
                const float* sw0 = p.sw + ti.e * p.sw_expert + weight_block<SWIGLU>(p, ti.nt, 0) * p.sw_n;
                const float* sw1 = ti.nh > 1 ? p.sw + ti.e * p.sw_expert + weight_block<SWIGLU>(p, ti.nt, 1) * p.sw_n : sw0;
                float x[PER][AHEAD], w0[AHEAD], w1[AHEAD];
                auto load = [&](int kb0) {
                    #pragma unroll
                    for (int a = 0; a < AHEAD; ++a)
                    {
                        const bool in = kb0 + a < nkb;
                        w0[a] = in ? __ldg(sw0 + (kb0 + a) * p.sw_k) : 0.0f;
                        w1[a] = in ? __ldg(sw1 + (kb0 + a) * p.sw_k) : 0.0f;
                        #pragma unroll
                        for (int i = 0; i < PER; ++i)
                        {
                            const int m = j0 + 64 * i;
                            x[i][a] = in && m < ti.rows ? __ldg(p.sx + (ti.row0 + m) * p.sx_row + (kb0 + a) * p.sx_blk) : 0.0f;
                        }
                    }
                };
                load(0);
                for (int kb0 = 0; ok && kb0 < nkb; kb0 += AHEAD)
                {
                    float o0[PER][AHEAD], o1[PER][AHEAD];
                    #pragma unroll
                    for (int a = 0; a < AHEAD; ++a)
                        #pragma unroll
                        for (int i = 0; i < PER; ++i)
                        {
                            o0[i][a] = x[i][a] * w0[a];
                            o1[i][a] = x[i][a] * w1[a];
                        }
                    if (kb0 + AHEAD < nkb) load(kb0 + AHEAD);
                    #pragma unroll
                    for (int a = 0; a < AHEAD; ++a)
                    {
                        if (kb0 + a >= nkb) break;
                        const int q = it % FG_SCALES;
                        if (it >= FG_SCALES &&
                            !__all_sync(0xffffffffu, mbar_wait(&bar_sempty[q], ((it / FG_SCALES) & 1u) ^ 1u, abort_flag,
                                                               p.status, p.wait_ns)))
                        {
                            ok = false;
                            break;
                        }
                        #pragma unroll
                        for (int i = 0; i < PER; ++i)
                            if (j0 + 64 * i < NT)
                            {
                                s_scale[q][0][j0 + 64 * i] = o0[i][a];
                                s_scale[q][1][j0 + 64 * i] = o1[i][a];
                            }
                        __syncwarp();
                        if (lane == 0) mbar_arrive(&bar_sfull[q]);
                        ++it;
                    }
                }
            }
        }
    }
    else
    {
        // ================================================================ epilogue
        setmaxnreg_inc<208>();
        const int g = (warp - 4) >> 2;                      // warpgroup
        const int quarter = warp & 3;
        const int lane_in = quarter * 32 + lane;            // TMEM lane: token (wide) or weight row (thin)
        int it = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x)
        {
            const Tile ti = tile_at<SWIGLU>(p, s_pref, t);
            uint64_t acc[2][32];                            // wide: 64 columns of each block; thin: 2 chunks of 16
            #pragma unroll
            for (int h = 0; h < 2; ++h)
                #pragma unroll
                for (int i = 0; i < 32; ++i) acc[h][i] = 0;
            bool ok = true;
            #pragma unroll 1
            for (int kb = 0; kb < nkb; ++kb, ++it)
            {
                const int b = it & 1, q = it % FG_SCALES;
                if (!mbar_try_wait(&bar_sfull[q], (it / FG_SCALES) & 1u) || !mbar_try_wait(&bar_tfull[b], (it >> 1) & 1u))
                    ok = mbar_wait(&bar_sfull[q], (it / FG_SCALES) & 1u, abort_flag, p.status, p.wait_ns) &&
                         mbar_wait(&bar_tfull[b], (it >> 1) & 1u, abort_flag, p.status, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + b * 256;
                if (!ti.thin)
                {
                    #pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        const uint32_t f = __float_as_uint(s_scale[q][h][lane_in]);
                        const uint64_t ff = pack2(f, f);
                        #pragma unroll
                        for (int c = 0; c < 2; ++c)
                        {
                            uint64_t d[16];
                            tmem_load(taddr + h * 128 + g * 64 + c * 32, d);
                            #pragma unroll
                            for (int i = 0; i < 16; ++i) fma2(acc[h][c * 16 + i], d[i], ff);
                        }
                    }
                }
                else
                {
                    #pragma unroll
                    for (int ci = 0; ci < 2; ++ci)
                        if ((2 * ci + g) * 16 < ti.rows)
                        {
                            const float* sc = &s_scale[q][0][(2 * ci + g) * 16];
                            #pragma unroll
                            for (int h = 0; h < 2; ++h)
                            {
                                uint64_t d[8];
                                tmem_load(taddr + h * 128 + (2 * ci + g) * 16, d);
                                #pragma unroll
                                for (int i = 0; i < 4; ++i)
                                {
                                    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(sc + h * NT + 4 * i);
                                    fma2(acc[h][ci * 8 + 2 * i], d[2 * i], f.x);
                                    fma2(acc[h][ci * 8 + 2 * i + 1], d[2 * i + 1], f.y);
                                }
                            }
                        }
                }
                tc_fence_before();
                __syncwarp();
                if (lane == 0)
                {
                    mbar_arrive(&bar_tempty[b]);
                    mbar_arrive(&bar_sempty[q]);
                }
            }
            // A warp that gave up says so before the epilogue's barrier, and every warp reads it between this
            // barrier and the next: one decision for all eight.
            if (!ok && lane == 0) s_fail = 1;
            named_bar_sync(3, 256);
            const bool fail = *(volatile int*) &s_fail != 0;
            if (fail)
            {
                named_bar_sync(3, 256);
                break;
            }
            if (ti.thin)
            {
                float* st = &s_stage[g][0][0];
                #pragma unroll
                for (int ci = 0; ci < 2; ++ci)
                    #pragma unroll
                    for (int j0 = 0; j0 < 16; j0 += FG_STEP)
                    {
                        const int m0 = (2 * ci + g) * 16 + j0;
                        if (m0 < ti.rows)
                        {
                            #pragma unroll
                            for (int j = 0; j < FG_STEP; ++j)
                                #pragma unroll
                                for (int h = 0; h < 2; ++h)
                                    st[j * 256 + h * 128 + lane_in] = half_of(acc[h][ci * 8 + ((j0 + j) >> 1)], j & 1);
                            named_bar_sync(1 + g, 128);
                            write_step<SWIGLU>(p, ti, st, m0, threadIdx.x & 127);
                            named_bar_sync(1 + g, 128);
                        }
                    }
                named_bar_sync(3, 256);
            }
            else if constexpr (!SWIGLU)
            {
                if (p.out_dtype == 0) store_wide<float>(p, ti, acc, g, lane_in);
                else if (p.out_dtype == 1) store_wide<__half>(p, ti, acc, g, lane_in);
                else store_wide<__nv_bfloat16>(p, ti, acc, g, lane_in);
                named_bar_sync(3, 256);
            }
            else
            {
                // this thread's token: 64 of the block's 128 columns; the largest magnitude of the other 64 comes from
                // the other warpgroup
                float act[64];
                uint32_t mx = 0;
                #pragma unroll
                for (int i = 0; i < 64; ++i)
                {
                    act[i] = clamped_swiglu(half_of(acc[0][i >> 1], i & 1), half_of(acc[1][i >> 1], i & 1), p.limit);
                    mx = max(mx, __float_as_uint(act[i]) & 0x7fffffffu);
                }
                s_amax[g][lane_in] = mx;
                named_bar_sync(3, 256);
                mx = max(mx, s_amax[g ^ 1][lane_in]);
                if (lane_in < ti.rows)
                {
                    const float s = block_scale(__uint_as_float(mx), false), inv = 1.0f / s;
                    const int64_t r = ti.row0 + lane_in;
                    uint4* h = reinterpret_cast<uint4*>(p.h + r * p.h_stride + ti.nt * kBlock + g * 64);
                    #pragma unroll
                    for (int c = 0; c < 4; ++c)
                    {
                        uint32_t w[4];
                        #pragma unroll
                        for (int j = 0; j < 4; ++j)
                        {
                            float q[4];
                            #pragma unroll
                            for (int i = 0; i < 4; ++i) q[i] = quotient(act[16 * c + 4 * j + i], s, inv);
                            w[j] = to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
                        }
                        h[c] = make_uint4(w[0], w[1], w[2], w[3]);
                    }
                    if (g == 0) p.hs[r * p.hs_row + ti.nt * p.hs_blk] = s;
                }
            }
        }
    }

    // ---- teardown
    tc_fence_before();
    __syncthreads();
    if (warp == 1)
    {
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

int make_map(CUtensorMap* tmap, const void* base, int rank, const cuuint64_t* dims, const cuuint64_t* strides,
             uint32_t box_rows)
{
    auto encode = trellis::get_encode_fn();
    if (!encode) return set_error("fp8_gemm: cuTensorMapEncodeTiled unavailable");
    const cuuint32_t box[3] = {FG_BK, box_rows, 1};
    const cuuint32_t estr[3] = {1, 1, 1};
    const CUresult cr = encode(tmap, CU_TENSOR_MAP_DATA_TYPE_UINT8, rank, const_cast<void*>(base), dims, strides, box,
                               estr, CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
                               CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (cr != CUDA_SUCCESS) return set_error("fp8_gemm: cuTensorMapEncodeTiled failed (%d)", (int) cr);
    return 0;
}

std::atomic<bool> g_fp8_attr_set[kMaxDevices] = {};

constexpr uint32_t kDynBytes = FG_STAGES * FG_STAGE_BYTES + 1024;

}  // namespace

int launch_fp8_gemm(const Fp8GemmProblem& q, cudaStream_t stream)
{
    Fp8GemmArgs p{};
    p.N = q.N; p.K = q.K; p.n_experts = q.n_experts;
    p.n_tiles_n = q.swiglu ? q.N / 2 / kBlock : (q.N + 255) / 256;
    p.num_kb = (q.K + FG_BK - 1) / FG_BK;
    p.single_count = (int) q.rows;
    p.counts = q.counts; p.row0 = q.row0;
    p.sx = q.sx; p.sx_row = q.sx_row; p.sx_blk = q.sx_blk;
    p.sw = q.sw; p.sw_expert = q.sw_expert; p.sw_n = q.sw_n; p.sw_k = 1;
    p.out = q.out; p.out_stride = q.out_stride; p.out_dtype = q.out_dtype; p.accumulate = q.accumulate;
    p.slot = q.slot;
    p.out_vec = reinterpret_cast<uintptr_t>(q.out) % 16 == 0 && q.out_stride * (q.out_dtype == 0 ? 4 : 2) % 16 == 0;
    p.f = q.N / 2; p.limit = q.limit;
    p.h = static_cast<uint8_t*>(q.h); p.h_stride = q.h_stride; p.hs = q.hs; p.hs_row = q.hs_row; p.hs_blk = q.hs_blk;
    p.status = q.status;
    p.wait_ns = wait_limit_ns();
    CUtensorMap tw, tx;
    const cuuint64_t wd[3] = {(cuuint64_t) q.K, (cuuint64_t) q.N, (cuuint64_t) q.n_experts};
    const cuuint64_t ws[2] = {(cuuint64_t) q.w_stride, (cuuint64_t) q.w_expert};
    int rc = make_map(&tw, q.w, 3, wd, ws, 128);
    if (rc) return rc;
    const cuuint64_t xd[2] = {(cuuint64_t) q.K, (cuuint64_t) q.rows};
    const cuuint64_t xs[1] = {(cuuint64_t) q.x_stride};
    rc = make_map(&tx, q.x, 2, xd, xs, FG_XBOX);
    if (rc) return rc;
    rc = once_per_device(g_fp8_attr_set, "fp8_gemm", [](int) {
        cudaError_t err = cudaSuccess;
        auto set = [&](const void* fn, uint32_t bytes) {
            if (err == cudaSuccess) err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) bytes);
        };
        set((const void*) fp8_gemm_kernel<false>, kDynBytes);
        set((const void*) fp8_gemm_kernel<true>, kDynBytes);
        return err == cudaSuccess ? 0 : set_cuda_error("fp8_gemm: cudaFuncSetAttribute", err);
    });
    if (rc) return rc;
    // tiles are counted on the device; this bound only keeps the grid from being larger than the work
    const int64_t sms = device_sm_count();
    const int64_t tiles = (q.rows / NT + (q.rows < q.n_experts ? q.rows : q.n_experts)) * p.n_tiles_n;
    const unsigned grid = (unsigned) (tiles < sms ? tiles : sms);
    if (q.swiglu) fp8_gemm_kernel<true><<<grid, FG_THREADS, kDynBytes, stream>>>(tw, tx, p);
    else fp8_gemm_kernel<false><<<grid, FG_THREADS, kDynBytes, stream>>>(tw, tx, p);
    return check_launch("fp8_gemm");
}

}  // namespace exl3b
