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
// Weights are the MMA's 128-row operand (M) and tokens its columns (N = the tile's rows rounded up to 16, so an expert
// with few rows costs few columns): TMEM lane = weight row, column = token.  A tile is two blocks of
// 128 weight rows (gate and up rows of the same columns for swiglu) by up to NT tokens.
//
//   warp 0        TMA producer: weight blocks [128 x 128 B] x 2 and token rows in boxes of 32, 128-byte swizzle;
//   warp 1        MMA issuer, TMEM owner;
//   warps 2, 3    scales: sx * sw of the coming K blocks into a shared-memory ring, loaded one group ahead;
//   warps 4..11   two warpgroups of epilogue; warpgroup g takes the 16-column chunks c with c % 2 == g.
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
constexpr int FG_SCALES = 8;                                // slots of the scale ring
constexpr uint64_t FG_DRAIN_NS = 200000000ull;
constexpr int FG_MAX_STAGES = 6;

struct Fp8GemmArgs {
    int N, K, n_experts;
    int n_tiles_n, num_kb;
    int single_count;                // rows of the one expert when counts is null
    const int32_t* counts;           // [E] or null
    const int32_t* row0;             // [E] first row of each expert, or null
    const float* sx; int64_t sx_row, sx_blk;
    const float* sw; int64_t sw_expert, sw_n, sw_k;
    int stages;
    // store
    void* out; int64_t out_stride; int out_dtype; int accumulate;
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

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16])
{
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
        "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
        : "r"(taddr));
}

// a += d * s for two columns at once.
__device__ __forceinline__ void fma2(float2& a, uint32_t d0, uint32_t d1, float s0, float s1)
{
    asm("{\n\t.reg .b64 a, d, s;\n\t"
        "mov.b64 a, {%0, %1};\n\tmov.b64 d, {%2, %3};\n\tmov.b64 s, {%4, %5};\n\t"
        "fma.rn.f32x2 a, d, s, a;\n\t"
        "mov.b64 {%0, %1}, a;\n\t}"
        : "+f"(a.x), "+f"(a.y) : "r"(d0), "r"(d1), "f"(s0), "f"(s1));
}

struct Tile {
    int e, nt, row0, rows, nh;       // nh: weight blocks with rows (1 at the end of an odd number of blocks)
};

template <bool SWIGLU>
__device__ __forceinline__ Tile tile_at(const Fp8GemmArgs& p, const int* pref, int NT, int t)
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
    ti.nh = SWIGLU || ti.nt * 256 + 128 < p.N ? 2 : 1;
    return ti;
}

// Weight block (of 128 rows) that is half h of tile column nt.
template <bool SWIGLU>
__device__ __forceinline__ int weight_block(const Fp8GemmArgs& p, int nt, int h)
{
    return SWIGLU ? h * (p.f / kBlock) + nt : 2 * nt + h;
}

template <class To, int NC>
__device__ __forceinline__ void store_tile(const Fp8GemmArgs& p, const Tile& ti, float2 (&acc)[2][NC][8], int g, int n_in)
{
    To* out = reinterpret_cast<To*>(p.out);
    #pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        const int n = ti.nt * 256 + h * 128 + n_in;
        if (n >= p.N) continue;
        #pragma unroll
        for (int ci = 0; ci < NC; ++ci)
            #pragma unroll
            for (int i = 0; i < 16; ++i)
            {
                const int m = (2 * ci + g) * 16 + i;
                if (m < ti.rows)
                {
                    const int64_t r = p.slot ? __ldg(p.slot + ti.row0 + m) : (int64_t) ti.row0 + m;
                    To* o = out + r * p.out_stride + n;
                    float v = i & 1 ? acc[h][ci][i >> 1].y : acc[h][ci][i >> 1].x;
                    if (p.accumulate) v += to_float(*o);
                    *o = from_float<To>(v);
                }
            }
    }
}

template <int NT, bool SWIGLU, int MIN_CTAS>
__global__ __launch_bounds__(FG_THREADS, MIN_CTAS)
void fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     const Fp8GemmArgs p)
{
    constexpr int NC = NT / 32;                             // 16-column chunks per epilogue warpgroup
    constexpr uint32_t TMEM_COLS = 4 * NT;                  // two buffers of two weight blocks
    constexpr uint32_t X_BYTES = NT * FG_BK;
    constexpr uint32_t STAGE_BYTES = 2 * FG_W_BYTES + X_BYTES;
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[FG_MAX_STAGES], bar_empty[FG_MAX_STAGES];
    __shared__ uint64_t bar_sfull[FG_SCALES], bar_sempty[FG_SCALES];
    __shared__ uint64_t bar_tfull[2], bar_tempty[2], bar_done;
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort, s_fail[2];
    __shared__ int s_pref[kMaxExperts + 1];
    __shared__ __align__(16) float s_scale[FG_SCALES][2][NT];
    __shared__ __align__(16) float s_amax[2][NT / 2][4];

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
            for (int s = 0; s < p.stages; ++s)
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
                s_fail[b] = 0;
            }
            mbar_init(&bar_done, 1);
            s_abort = 0;
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
        if constexpr (MIN_CTAS == 1 && NT == 128) setmaxnreg_dec<64>();
        if (warp == 0)
        {
            // ============================================================ TMA producer
            if (lane == 0)
            {
                int issued = 0;
                bool ok = true;
                for (int t = blockIdx.x; ok && t < total; t += gridDim.x)
                {
                    const Tile ti = tile_at<SWIGLU>(p, s_pref, NT, t);
                    const int boxes = (ti.rows + FG_XBOX - 1) / FG_XBOX;
                    const uint32_t bytes = ti.nh * FG_W_BYTES + boxes * (FG_XBOX * FG_BK);
                    for (int kb = 0; kb < nkb; ++kb, ++issued)
                    {
                        const int s = issued % p.stages;
                        const uint32_t ph = (issued / p.stages) & 1u;
                        if (issued >= p.stages && !mbar_wait(&bar_empty[s], ph ^ 1u, abort_flag, p.status, p.wait_ns))
                        {
                            ok = false;
                            break;
                        }
                        uint8_t* w = smem + s * STAGE_BYTES;
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
                for (int i = issued > p.stages ? issued - p.stages : 0; i < issued; ++i)
                    mbar_drain(&bar_full[i % p.stages], (i / p.stages) & 1u, FG_DRAIN_NS);
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
                    const Tile ti = tile_at<SWIGLU>(p, s_pref, NT, t);
                    const uint32_t idesc = idesc_e4m3_f32(128, (ti.rows + 15) & ~15);
                    for (int kb = 0; kb < nkb; ++kb, ++it)
                    {
                        const int s = it % p.stages, b = it & 1;
                        if ((it >= 2 && !mbar_wait(&bar_tempty[b], ((it >> 1) & 1u) ^ 1u, abort_flag, p.status, p.wait_ns)) ||
                            !mbar_wait(&bar_full[s], (it / p.stages) & 1u, abort_flag, p.status, p.wait_ns))
                        {
                            ok = false;
                            break;
                        }
                        tc_fence_after();
                        const uint32_t w = smem_u32(smem + s * STAGE_BYTES);
                        const uint64_t x_desc = smem_desc_sw128(w + 2 * FG_W_BYTES);
                        for (int h = 0; h < ti.nh; ++h)
                        {
                            const uint64_t w_desc = smem_desc_sw128(w + h * FG_W_BYTES);
                            #pragma unroll
                            for (int kk = 0; kk < FG_BK / 32; ++kk)
                                umma_e4m3(tmem_base + b * 2 * NT + h * NT, w_desc + 2 * kk, x_desc + 2 * kk, idesc, kk != 0);
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
                const Tile ti = tile_at<SWIGLU>(p, s_pref, NT, t);
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
        if constexpr (MIN_CTAS == 1 && NT == 128) setmaxnreg_inc<216>();
        const int g = (warp - 4) >> 2;                      // warpgroup
        const int quarter = warp & 3;
        const int n_in = quarter * 32 + lane;               // TMEM lane: weight row of the block
        int it = 0;
        for (int t = blockIdx.x; t < total; t += gridDim.x)
        {
            const Tile ti = tile_at<SWIGLU>(p, s_pref, NT, t);
            float2 acc[2][NC][8];
            #pragma unroll
            for (int h = 0; h < 2; ++h)
                #pragma unroll
                for (int ci = 0; ci < NC; ++ci)
                    #pragma unroll
                    for (int i = 0; i < 8; ++i) acc[h][ci][i] = make_float2(0.0f, 0.0f);
            bool ok = true;
            for (int kb = 0; kb < nkb; ++kb, ++it)
            {
                const int b = it & 1, q = it % FG_SCALES;
                ok = mbar_wait(&bar_sfull[q], (it / FG_SCALES) & 1u, abort_flag, p.status, p.wait_ns) &&
                     mbar_wait(&bar_tfull[b], (it >> 1) & 1u, abort_flag, p.status, p.wait_ns);
                ok = __all_sync(0xffffffffu, ok);
                if (!ok) break;
                tc_fence_after();
                const uint32_t taddr = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + b * 2 * NT;
                #pragma unroll
                for (int ci = 0; ci < NC; ++ci)
                {
                    const int c0 = (2 * ci + g) * 16;
                    if (c0 < ti.rows)
                    {
                        uint32_t d0[16], d1[16];
                        tmem_ld16(taddr + c0, d0);
                        tmem_ld16(taddr + NT + c0, d1);
                        tmem_wait_ld();
                        #pragma unroll
                        for (int i = 0; i < 16; ++i) asm volatile("" : "+r"(d0[i]), "+r"(d1[i]));
                        #pragma unroll
                        for (int i = 0; i < 4; ++i)
                        {
                            const float4 s0 = *reinterpret_cast<const float4*>(&s_scale[q][0][c0 + 4 * i]);
                            const float4 s1 = *reinterpret_cast<const float4*>(&s_scale[q][1][c0 + 4 * i]);
                            fma2(acc[0][ci][2 * i], d0[4 * i], d0[4 * i + 1], s0.x, s0.y);
                            fma2(acc[0][ci][2 * i + 1], d0[4 * i + 2], d0[4 * i + 3], s0.z, s0.w);
                            fma2(acc[1][ci][2 * i], d1[4 * i], d1[4 * i + 1], s1.x, s1.y);
                            fma2(acc[1][ci][2 * i + 1], d1[4 * i + 2], d1[4 * i + 3], s1.z, s1.w);
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
            if constexpr (!SWIGLU)
            {
                if (!ok) break;
                if (p.out_dtype == 0) store_tile<float, NC>(p, ti, acc, g, n_in);
                else if (p.out_dtype == 1) store_tile<__half, NC>(p, ti, acc, g, n_in);
                else store_tile<__nv_bfloat16, NC>(p, ti, acc, g, n_in);
            }
            else
            {
                // the block's largest magnitude per token: 32 weight rows by a warp reduction, four warps through
                // shared memory.  A warp that gave up still takes part in the two barriers.
                uint32_t mx[(NT / 2 + 31) / 32];
                #pragma unroll
                for (int ci = 0; ci < NC; ++ci)
                    #pragma unroll
                    for (int i = 0; i < 16; ++i)
                    {
                        float& gv = i & 1 ? acc[0][ci][i >> 1].y : acc[0][ci][i >> 1].x;
                        const float uv = i & 1 ? acc[1][ci][i >> 1].y : acc[1][ci][i >> 1].x;
                        gv = clamped_swiglu(gv, uv, p.limit);
                        const uint32_t m = __reduce_max_sync(0xffffffffu, __float_as_uint(gv) & 0x7fffffffu);
                        const int c = ci * 16 + i;
                        if (lane == (c & 31)) mx[c >> 5] = m;
                    }
                #pragma unroll
                for (int i = 0; i < (NT / 2 + 31) / 32; ++i)
                    if (lane + 32 * i < NT / 2) s_amax[g][lane + 32 * i][quarter] = __uint_as_float(mx[i]);
                if (!ok && lane == 0) s_fail[g] = 1;
                named_bar_sync(1 + g, 128);
                const bool fail = *(volatile int*) &s_fail[g] != 0;
                if (!fail)
                {
                    #pragma unroll
                    for (int ci = 0; ci < NC; ++ci)
                        #pragma unroll
                        for (int i = 0; i < 16; ++i)
                        {
                            const int c = ci * 16 + i, m = (2 * ci + g) * 16 + i;
                            if (m < ti.rows)
                            {
                                const uint4 a = *reinterpret_cast<const uint4*>(s_amax[g][c]);
                                const float s = block_scale(__uint_as_float(max(max(a.x, a.y), max(a.z, a.w))), false);
                                const float v = i & 1 ? acc[0][ci][i >> 1].y : acc[0][ci][i >> 1].x;
                                const int64_t r = ti.row0 + m;
                                p.h[r * p.h_stride + ti.nt * kBlock + n_in] = (uint8_t) to_e4m3x2(quotient(v, s, 1.0f / s), 0.0f);
                                if (n_in == 0) p.hs[r * p.hs_row + ti.nt * p.hs_blk] = s;
                            }
                        }
                }
                named_bar_sync(1 + g, 128);
                if (fail) break;
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

constexpr uint32_t dyn_bytes(int NT, int stages) { return stages * (2 * FG_W_BYTES + NT * FG_BK) + 1024; }
constexpr int kStages128 = 4, kStages32 = 2;

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
        set((const void*) fp8_gemm_kernel<128, false, 1>, dyn_bytes(128, kStages128));
        set((const void*) fp8_gemm_kernel<128, true, 1>, dyn_bytes(128, kStages128));
        set((const void*) fp8_gemm_kernel<32, false, 2>, dyn_bytes(32, kStages32));
        set((const void*) fp8_gemm_kernel<32, true, 2>, dyn_bytes(32, kStages32));
        return err == cudaSuccess ? 0 : set_cuda_error("fp8_gemm: cudaFuncSetAttribute", err);
    });
    if (rc) return rc;
    const int sms = device_sm_count();
    const int64_t most_rows_per_expert = q.counts ? (q.rows + q.n_experts - 1) / q.n_experts : q.rows;
    const bool wide = most_rows_per_expert > 32;
    const int NT = wide ? 128 : 32;
    p.stages = wide ? kStages128 : kStages32;
    // tiles are counted on the device; this bound only keeps the grid from being larger than the work
    const int64_t tiles = (q.rows / NT + (q.rows < q.n_experts ? q.rows : q.n_experts)) * (int64_t) p.n_tiles_n;
    const int64_t slots = (int64_t) sms * (wide ? 1 : 2);
    const unsigned grid = (unsigned) (tiles < slots ? tiles : slots);
    if (wide)
    {
        if (q.swiglu) fp8_gemm_kernel<128, true, 1><<<grid, FG_THREADS, dyn_bytes(128, p.stages), stream>>>(tw, tx, p);
        else fp8_gemm_kernel<128, false, 1><<<grid, FG_THREADS, dyn_bytes(128, p.stages), stream>>>(tw, tx, p);
    }
    else
    {
        if (q.swiglu) fp8_gemm_kernel<32, true, 2><<<grid, FG_THREADS, dyn_bytes(32, p.stages), stream>>>(tw, tx, p);
        else fp8_gemm_kernel<32, false, 2><<<grid, FG_THREADS, dyn_bytes(32, p.stages), stream>>>(tw, tx, p);
    }
    return check_launch("fp8_gemm");
}

}  // namespace exl3b
