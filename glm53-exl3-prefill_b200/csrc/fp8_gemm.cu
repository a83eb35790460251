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
// Two CTAs (a cluster) work on one tile with cta_group::2 MMAs, M = 256 over the pair: a single SM's operands
// (A and B of 128 x 256 x 32: 12 KB per 128 clocks at the full rate, beside 48 KB of new data per K block) come out of
// shared memory at two thirds of the tensor core's rate; the pair holds each operand once between two SMs.
// A tile is a run of rows (tokens) of one expert by 256 or 512 weight rows, in one of two orientations:
//   wide  (129..256 rows)  tokens are M: CTA r holds tokens 128 r .. 128 r + 127 and weight block r of two (neighbours,
//         or the gate and up rows of the same columns for swiglu); TMEM lane = token, column = weight row of
//         both blocks.  The scale is one register per thread.
//   thin  (up to 128 rows)  weights are M: CTA r holds two weight blocks of four (for swiglu gate and up of its own
//         128 columns) and half of the tokens, N = the tile's rows rounded up to 16; lane = weight row, column =
//         token.  An expert with few rows costs few columns.  Every value needs its column's scale here, which a warp
//         reads from shared memory (128 bytes a clock for the SM): 8 clocks per column and K block.
//
// A K block is two halves, each with its own pair of TMEM buffers, MMAs and barriers: half j is rows 64 j .. 64 j + 63 of
// both weight blocks (wide) or tokens 64 j .. (thin), and is worked on by warpgroups 2 j and 2 j + 1.  What bounds
// the loop is the way round one TMEM buffer (MMA, commit, taking the sums out, arrival, next MMA: about 2000 clocks),
// and the two halves go round out of step.  A 256 x 256 x 128 block takes the pair about 1050 clocks, of which the MMAs
// need 512, and the end of a tile about 5000, in which the tensor core waits (the sums are half of the register file, so there
// is no second set): 8192 x 12288 x 4096 in 463 us, 53 % of twice the measured bf16 rate, alone; 540..555 us, 45 %, call after
// call, where the power cap lowers the clock.  Eight epilogue warps with 64 columns
// each (spills: 562 us), all sixteen on each half in turn (553 us: more barriers a block) and spinning waits (511 us) were slower.
//
//   warp 0        TMA producer of this CTA's operands: weight blocks [128 x 128 B], token rows in boxes of 32;
//   warp 1        MMA issuer (in CTA 0, for both), TMEM owner;
//   warps 2, 3    scales of the coming K blocks into a shared-memory ring (cp.async, up to eight blocks ahead);
//   warps 4..19   four warpgroups of epilogue: warpgroup g takes 32 columns of each block (wide) or 32 tokens (thin).
// The clusters walk the tiles (expert, weight tile, token tile; token tiles fastest, so the clusters running at
// one time share weight tiles through L2).  With fewer tiles than clusters, each tile's K is split over several of them:
// fp32 partial sums to a workspace, joined in order by the kernel that follows (fp8_rows.cu); a K block takes a cluster
// about half a microsecond however few rows there are.  Every wait is bounded as in the trellis kernels.
#include <cuda.h>

#include "fp8_common.cuh"
#include "trellis_common.cuh"

namespace exl3b {

namespace {

using namespace fp8;

constexpr int FG_EPI_WARPS = 16;
constexpr int FG_EPI_THREADS = FG_EPI_WARPS * 32;
constexpr int FG_THREADS = 128 + FG_EPI_THREADS;
constexpr int FG_BK = 128;                                  // K bytes per stage: one 128-byte swizzle atom
constexpr uint32_t FG_W_BYTES = 128 * FG_BK;                // one block of weight rows
constexpr int FG_XBOX = 32;                                 // token rows per TMA box
constexpr int NT = 128;                                     // tokens of a CTA in a wide tile, of the pair in a thin one
constexpr int FG_STAGES = 5;
constexpr uint32_t FG_STAGE_BYTES = 2 * FG_W_BYTES + 64 * FG_BK;    // thin: two weight blocks, 64 tokens
constexpr int FG_SCALES = 8;                                // slots of the scale ring
constexpr uint64_t FG_DRAIN_NS = 200000000ull;

struct Fp8GemmArgs {
    int N, K, n_experts;
    int n_wide, n_thin, num_kb;      // weight tiles of a wide and of a thin row tile; K blocks
    int n_blocks;                    // weight blocks of 128 rows
    int splits;                      // clusters that share a tile's K; > 1: fp32 partial sums to out + split * split_stride
    int64_t split_stride;
    int single_count;                // rows of the one expert when counts is null
    const int32_t* counts;           // [E] or null
    const int32_t* row0;             // [E] first row of each expert, or null
    const float* sx; int64_t sx_row, sx_blk;
    const float* sw; int64_t sw_expert, sw_n;
    // store
    void* out; int64_t out_stride; int out_dtype; int accumulate;
    int out_vec;                     // rows are 32-byte aligned
    const int64_t* slot;             // output row of row r, or null
    // swiglu
    int f; float limit;
    uint8_t* h; int64_t h_stride; float* hs; int64_t hs_row, hs_blk;
    int32_t* status;
    uint64_t wait_ns;
};

// D (both CTAs' TMEM) (+)= A . B^T over the pair: M = 256, each CTA holding 128 rows of A and N / 2 rows of B.
__device__ __forceinline__ void umma_e4m3_pair(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc,
                                               uint32_t accumulate)
{
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "setp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}"
        :: "r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}

// Arrive (once) on `bar` in the CTAs of `mask` when every MMA issued so far by this thread has completed.
__device__ __forceinline__ void umma_commit_pair(uint64_t* bar, uint16_t mask = 3)
{
    asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;"
                 :: "r"(smem_u32(bar)), "h"(mask) : "memory");
}

__device__ __forceinline__ uint32_t cluster_rank()
{
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}

__device__ __forceinline__ void cluster_sync()
{
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
}

// The address of `p` in CTA 0 of the cluster.
__device__ __forceinline__ uint32_t in_cta0(const void* p)
{
    uint32_t r;
    asm("mapa.shared::cluster.u32 %0, %1, 0;" : "=r"(r) : "r"(smem_u32(p)));
    return r;
}

__device__ __forceinline__ void mbar_arrive_cluster(uint32_t bar)
{
    asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" :: "r"(bar) : "memory");
}

// One lane of a converged warp.  Roles of a single thread run as a whole warp with the instruction itself behind this:
// with the loop inside an `if (lane == 0)` the compiler cannot keep descriptors and addresses in uniform
// registers, and the MMA thread took 1300 clocks per K block.
__device__ __forceinline__ bool elect_one()
{
    uint32_t r;
    asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(r));
    return r != 0;
}

// Instruction descriptor, kind::f8f6f4: D fp32, A and B e4m3 (both K-major), shape M x N.
__device__ __forceinline__ uint32_t idesc_e4m3_f32(int M, int N)
{
    return (1u << 4) | (static_cast<uint32_t>(N >> 3) << 17) | (static_cast<uint32_t>(M >> 4) << 24);
}

// Tiled loads into this CTA's shared memory that complete on a barrier (`bar`) of CTA 0.
__device__ __forceinline__ void tma_pair_3d(void* smem_dst, const void* tmap, int32_t x, int32_t y, int32_t z, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3, %4}], [%5];"
        :: "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(bar) : "memory");
}

__device__ __forceinline__ void tma_pair_2d(void* smem_dst, const void* tmap, int32_t x, int32_t y, uint32_t bar)
{
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes "
        "[%0], [%1, {%2, %3}], [%4];"
        :: "r"(smem_u32(smem_dst)), "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(bar) : "memory");
}

__device__ __forceinline__ void tmem_alloc_pair(uint32_t* smem_dst, uint32_t ncols)
{
    asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;"
                 :: "r"(smem_u32(smem_dst)), "r"(ncols) : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}

__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols)
{
    asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" :: "r"(taddr), "r"(ncols) : "memory");
}

__device__ __forceinline__ void cp_async4(void* smem_dst, const void* gmem_src)
{
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4;" :: "r"(smem_u32(smem_dst)), "l"(gmem_src) : "memory");
}

// Arrive (once per thread) on `bar` when this thread's cp.async copies so far have landed.
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar)
{
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" :: "r"(smem_u32(bar)) : "memory");
}

__device__ __forceinline__ void cp_async_wait_all()
{
    asm volatile("cp.async.wait_all;" ::: "memory");
}

// Non-blocking test of one phase each of two barriers (shared-memory addresses).
__device__ __forceinline__ bool mbar_test2(uint32_t bar_a, uint32_t parity_a, uint32_t bar_b, uint32_t parity_b)
{
    uint32_t done;
    asm volatile(
        "{\n\t.reg .pred pa, pb;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 pa, [%1], %2;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 pb, [%3], %4;\n\t"
        "and.pred pa, pa, pb;\n\t"
        "selp.u32 %0, 1, 0, pa;\n\t}"
        : "=r"(done) : "r"(bar_a), "r"(parity_a), "r"(bar_b), "r"(parity_b) : "memory");
    return done != 0;
}

// 16 consecutive columns of this warp's 32 TMEM lanes as register pairs, complete on return.
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

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b)
{
    uint64_t r;
    asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
    return r;
}

// Which of three phases are complete (bits 0..2; the same answer for the whole warp), without blocking.
__device__ __forceinline__ uint32_t mbar_test3(uint64_t* a, uint32_t parity_a, uint64_t* b, uint64_t* c, uint32_t parity_bc)
{
    uint32_t r;
    asm volatile(
        "{\n\t.reg .pred pa, pb, pc;\n\t.reg .b32 x, y;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 pa, [%1], %2;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 pb, [%3], %5;\n\t"
        "mbarrier.test_wait.parity.shared::cta.b64 pc, [%4], %5;\n\t"
        "selp.u32 %0, 1, 0, pa;\n\t"
        "selp.u32 x, 2, 0, pb;\n\t"
        "selp.u32 y, 4, 0, pc;\n\t"
        "or.b32 %0, %0, x;\n\tor.b32 %0, %0, y;\n\t}"
        : "=&r"(r) : "r"(smem_u32(a)), "r"(parity_a), "r"(smem_u32(b)), "r"(smem_u32(c)), "r"(parity_bc) : "memory");
    return __reduce_and_sync(0xffffffffu, r);
}

// mbar_wait by a whole warp, with one answer for it.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* status,
                                          uint64_t limit_ns)
{
    if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    return __all_sync(0xffffffffu, mbar_wait(bar, parity, abort_flag, status, limit_ns));
}

// Position in a ring of N barriers: slot and the parity of the current pass.
template <int N>
struct Ring {
    int slot = 0;
    uint32_t parity = 0;
    __device__ __forceinline__ void next()
    {
        if (++slot == N)
        {
            slot = 0;
            parity ^= 1u;
        }
    }
};

struct Tile {
    bool thin;
    int e, nt;
    int row0, rows;                  // rows of the tile (of both CTAs)
    int ncols;                       // thin: rows rounded up to 16
    int kb0, kb1;                    // its K blocks
    int64_t out_offset;              // of this part of K's sums
};

// 256-row tiles of an expert with `count` rows, and whether its last rows (up to 128) are a thin tile.
__device__ __forceinline__ int wide_tiles(int count) { return count / 256 + (count % 256 > 128 ? 1 : 0); }
__device__ __forceinline__ int thin_tiles(int count) { const int r = count % 256; return r > 0 && r <= 128 ? 1 : 0; }

__device__ __forceinline__ int row_count(const Fp8GemmArgs& p, int e)
{
    return p.counts ? __ldg(p.counts + e) : p.single_count;
}

__device__ __forceinline__ int expert_tiles(const Fp8GemmArgs& p, int e)
{
    const int count = row_count(p, e);
    return wide_tiles(count) * p.n_wide + thin_tiles(count) * p.n_thin;
}

// Work unit t: a tile, or a part of its K.
__device__ __forceinline__ Tile tile_at(const Fp8GemmArgs& p, const int* pref, int t)
{
    Tile ti;
    ti.kb0 = 0;
    ti.kb1 = p.num_kb;
    ti.out_offset = 0;
    if (p.splits > 1)                                       // (divisions only where they are needed)
    {
        const int tile = t / p.splits, split = t - tile * p.splits;
        ti.kb0 = split * p.num_kb / p.splits;
        ti.kb1 = (split + 1) * p.num_kb / p.splits;
        ti.out_offset = split * p.split_stride;
        t = tile;
    }
    ti.e = p.n_experts > 1 ? trellis::prefix_find(pref, p.n_experts, t) : 0;
    const int count = row_count(p, ti.e), wide = wide_tiles(count);
    const int local = p.n_experts > 1 ? t - pref[ti.e] : t;
    ti.thin = local >= wide * p.n_wide;
    ti.nt = ti.thin ? local - wide * p.n_wide : wide > 1 ? local / wide : local;
    const int first = ti.thin ? count / 256 * 256 : (local - ti.nt * wide) * 256;
    ti.row0 = (p.row0 ? __ldg(p.row0 + ti.e) : 0) + first;
    ti.rows = min(256, count - first);
    ti.ncols = (ti.rows + 15) & ~15;
    return ti;
}

// Weight block (of 128 rows) h (0, 1) of CTA r: wide tiles have one per CTA (h = r, whatever is asked for the epilogue),
// thin ones two.  May be past the last block: loads there give zeros.
template <bool SWIGLU>
__device__ __forceinline__ int weight_block(const Fp8GemmArgs& p, const Tile& ti, int r, int h)
{
    if (!ti.thin) return SWIGLU ? h * (p.f / kBlock) + ti.nt : 2 * ti.nt + h;
    return SWIGLU ? h * (p.f / kBlock) + 2 * ti.nt + r : 4 * ti.nt + 2 * r + h;
}

constexpr int FG_STEP = 4;                                  // tokens staged at a time by a warpgroup

// Eight consecutive outputs of one row.
template <class To>
__device__ __forceinline__ void store8(const Fp8GemmArgs& p, const Tile& ti, int64_t r, int n, const float* v)
{
    To* o = reinterpret_cast<To*>(p.out) + ti.out_offset + r * p.out_stride + n;
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

// Thin tiles: the staged tokens [m0, m0 + FG_STEP) x 256 weight rows of CTA r, by the 128 threads of a warpgroup.
template <bool SWIGLU>
__device__ __forceinline__ void write_step(const Fp8GemmArgs& p, const Tile& ti, int r0, const float* st, int m0, int tid)
{
    if constexpr (!SWIGLU)
    {
        const int m = m0 + (tid >> 5), c = (tid & 31) * 8, n = (2 * ti.nt + r0) * 256 + c;
        if (m >= ti.rows || n >= p.N) return;
        const int64_t r = p.slot ? __ldg(p.slot + ti.row0 + m) : (int64_t) ti.row0 + m;
        const float* v = st + (tid >> 5) * 256 + c;
        if (p.out_dtype == 0) store8<float>(p, ti, r, n, v);
        else if (p.out_dtype == 1) store8<__half>(p, ti, r, n, v);
        else store8<__nv_bfloat16>(p, ti, r, n, v);
    }
    else
    {
        // a warp per token, 4 columns a lane
        const int m = m0 + (tid >> 5), c = tid & 31;
        const float4 g = *reinterpret_cast<const float4*>(st + (tid >> 5) * 256 + c * 4);
        const float4 u = *reinterpret_cast<const float4*>(st + (tid >> 5) * 256 + 128 + c * 4);
        const float a[4] = {clamped_swiglu(g.x, u.x, p.limit), clamped_swiglu(g.y, u.y, p.limit),
                            clamped_swiglu(g.z, u.z, p.limit), clamped_swiglu(g.w, u.w, p.limit)};
        uint32_t mx = 0;
        #pragma unroll
        for (int j = 0; j < 4; ++j) mx = max(mx, __float_as_uint(a[j]) & 0x7fffffffu);
        mx = __reduce_max_sync(0xffffffffu, mx);
        const int fb = 2 * ti.nt + r0;
        if (m >= ti.rows || fb * kBlock >= p.f) return;
        const float s = block_scale(__uint_as_float(mx), false), inv = reciprocal(s);
        const int64_t r = ti.row0 + m;
        float q[4];
        #pragma unroll
        for (int j = 0; j < 4; ++j) q[j] = quotient(a[j], s, inv);
        reinterpret_cast<uint32_t*>(p.h + r * p.h_stride + fb * kBlock)[c] =
            to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
        if (c == 0) p.hs[r * p.hs_row + fb * p.hs_blk] = s;
    }
}

// One whole 32-byte sector.
__device__ __forceinline__ void store32(void* dst, const uint32_t* w)
{
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};"
                 :: "l"(dst), "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3]), "r"(w[4]), "r"(w[5]), "r"(w[6]), "r"(w[7])
                 : "memory");
}

// Wide tiles, store: this thread's token, 32 columns of each of the two weight blocks.
template <class To>
__device__ __forceinline__ void store_wide(const Fp8GemmArgs& p, const Tile& ti, const uint64_t (&acc)[2][16], int g, int m)
{
    if (m >= ti.rows) return;
    const int64_t r = p.slot ? __ldg(p.slot + ti.row0 + m) : (int64_t) ti.row0 + m;
    To* row = reinterpret_cast<To*>(p.out) + ti.out_offset + r * p.out_stride;
    constexpr int PER = 32 / sizeof(To);                    // values of a 32-byte sector
    #pragma unroll
    for (int h = 0; h < 2; ++h)
    {
        const int n0 = ti.nt * 256 + h * 128 + g * 32;
        if (p.out_vec && !p.accumulate && n0 + 32 <= p.N)
        {
            #pragma unroll
            for (int c = 0; c < 32; c += PER)
            {
                __align__(32) To w[PER];
                #pragma unroll
                for (int i = 0; i < PER; ++i) w[i] = from_float<To>(half_of(acc[h][(c + i) >> 1], i & 1));
                store32(row + n0 + c, reinterpret_cast<const uint32_t*>(w));
            }
        }
        else
        {
            #pragma unroll
            for (int c = 0; c < 32; ++c)
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
__global__ __cluster_dims__(2, 1, 1) __launch_bounds__(FG_THREADS, 1)
void fp8_gemm_kernel(const __grid_constant__ CUtensorMap tmap_w, const __grid_constant__ CUtensorMap tmap_x,
                     const Fp8GemmArgs p)
{
    constexpr uint32_t TMEM_COLS = 512;                     // two buffers of 256 columns
    extern __shared__ uint8_t smem_raw[];
    __shared__ uint64_t bar_full[FG_STAGES];                // CTA 0: both CTAs' operands of a stage have landed
    __shared__ uint64_t bar_half[FG_STAGES];                // the MMAs of its first half are done
    __shared__ uint64_t bar_done[FG_STAGES];                // all its MMAs are done: the stage is free
    __shared__ uint64_t bar_sfull[FG_SCALES], bar_sempty[FG_SCALES];
    __shared__ uint64_t bar_tempty[4];                      // CTA 0: both CTAs have taken the sums of (half, buffer) out
    __shared__ __align__(16) float s_sx[FG_SCALES][NT];
    __shared__ float s_sw[FG_SCALES][2];
    __shared__ uint32_t s_tmem_base;
    __shared__ int s_abort, s_fail;
    __shared__ int s_pref[kMaxExperts + 1];
    __shared__ __align__(16) float s_stage[4][FG_STEP][256];

    let_next_launch_start();
    const int rank = (int) cluster_rank();
    const int cluster = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;
    const int warp = __shfl_sync(0xffffffffu, threadIdx.x >> 5, 0), lane = threadIdx.x & 31;
    uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));

    if (warp == 0)
    {
        wait_for_previous_launch();                         // (the counts are an earlier launch's)
        // tiles per expert, as an exclusive prefix
        const int per = (p.n_experts + 31) / 32;
        auto tiles = [&](int e) { return e < p.n_experts ? expert_tiles(p, e) : 0; };
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
                mbar_init(&bar_half[s], 1);
                mbar_init(&bar_done[s], 1);
            }
            for (int s = 0; s < FG_SCALES; ++s)
            {
                mbar_init(&bar_sfull[s], 64);
                mbar_init(&bar_sempty[s], FG_EPI_WARPS);
            }
            for (int b = 0; b < 4; ++b) mbar_init(&bar_tempty[b], FG_EPI_WARPS);      // half of them, in two CTAs
            s_abort = 0;
            s_fail = 0;
            fence_mbar_init();
        }
        __syncwarp();
        tmem_alloc_pair(&s_tmem_base, TMEM_COLS);
    }
    tc_fence_before();
    __syncthreads();
    cluster_sync();                                         // both CTAs' barriers and TMEM exist
    wait_for_previous_launch();
    tc_fence_after();
    const uint32_t tmem_base = s_tmem_base;
    volatile int* abort_flag = &s_abort;
    const int total = s_pref[p.n_experts] * p.splits;       // work units: (tile, part of K), parts fastest

    if (warp < 4)
    {
        setmaxnreg_dec<56>();
        if (warp == 0)
        {
            // ============================================================ TMA producer
            Ring<FG_STAGES> st;
            int issued = 0;
            // with a limit of zero it gives up at the first stage that is not free, and the other roles find the flag (a
            // try_wait by itself suspends for longer than any of these waits takes)
            const int room = p.wait_ns > 0 ? -1 : FG_STAGES;
            bool ok = true;
            for (int t = cluster; ok && t < total; t += n_clusters)
            {
                const Tile ti = tile_at(p, s_pref, t);
                // rows of this CTA's first and last box, boxes, and the pair's bytes: wide, one weight block and up to
                // 128 tokens a CTA; thin, two weight blocks and half of the columns of each half
                const int nc1 = max(ti.ncols - 64, 0), nc0 = ti.ncols - nc1;
                const int boxes0 = ti.thin ? (nc1 ? 2 : 1) : 4;
                const int boxes1 = ti.thin ? boxes0 : (ti.rows - 128 + FG_XBOX - 1) / FG_XBOX;
                const uint32_t bytes = (ti.thin ? 4 : 2) * FG_W_BYTES + (boxes0 + boxes1) * (FG_XBOX * FG_BK);
                const int boxes = rank ? boxes1 : boxes0;
                const int row = ti.row0 + rank * (ti.thin ? nc0 / 2 : 128);
                const int row1 = ti.thin ? ti.row0 + 64 + rank * (nc1 / 2) : row + FG_XBOX;
                const int w_row0 = weight_block<SWIGLU>(p, ti, rank, ti.thin ? 0 : rank) * kBlock;
                const int w_row1 = weight_block<SWIGLU>(p, ti, rank, 1) * kBlock;
                const uint32_t x_off = ti.thin ? 2 * FG_W_BYTES : FG_W_BYTES;
                for (int kb = ti.kb0; kb < ti.kb1; ++kb, ++issued, st.next())
                {
                    // (the first pass does not wait: a fresh barrier counts as past the phase of parity 1)
                    ok = issued != room && warp_wait(&bar_done[st.slot], st.parity ^ 1u, abort_flag, p.status, p.wait_ns);
                    if (!ok) break;
                    if (elect_one())
                    {
                        uint8_t* w = smem + st.slot * FG_STAGE_BYTES;
                        const uint32_t full = in_cta0(&bar_full[st.slot]);
                        if (rank == 0) mbar_arrive_expect_tx(&bar_full[st.slot], bytes);
                        tma_pair_3d(w, &tmap_w, kb * FG_BK, w_row0, ti.e, full);
                        if (ti.thin) tma_pair_3d(w + FG_W_BYTES, &tmap_w, kb * FG_BK, w_row1, ti.e, full);
                        tma_pair_2d(w + x_off, &tmap_x, kb * FG_BK, row, full);
                        for (int b = 1; b < boxes; ++b)
                            tma_pair_2d(w + x_off + b * (FG_XBOX * FG_BK), &tmap_x, kb * FG_BK, row1 + (b - 1) * FG_XBOX, full);
                    }
                    __syncwarp();
                }
            }
            if (issued == room && !ok)
            {
                *abort_flag = 1;
                record_error(p.status, kErrWaitTimeout);
            }
            // a stage whose MMAs are done has landed; after an abort this gives the copies in flight their time
            for (int i = issued > FG_STAGES ? issued - FG_STAGES : 0; i < issued; ++i)
                mbar_drain(&bar_done[i % FG_STAGES], (i / FG_STAGES) & 1u, FG_DRAIN_NS);
        }
        else if (warp == 1)
        {
            // ============================================================ MMA issuer
            if (rank == 0)
            {
                Ring<FG_STAGES> st;
                Ring<2> buf;
                const bool leader = elect_one();
                bool ok = true;
                for (int t = cluster; ok && t < total; t += n_clusters)
                {
                    const Tile ti = tile_at(p, s_pref, t);
                    const int nc1 = max(ti.ncols - 64, 0), nc0 = ti.ncols - nc1;
                    for (int kb = ti.kb0; kb < ti.kb1; ++kb, st.next(), buf.next())
                    {
                        // one round trip to shared memory for the three barriers of a K block: this warp's own
                        // instructions are what the loop waits for once the sums keep up
                        const uint32_t ready = mbar_test3(&bar_full[st.slot], st.parity, &bar_tempty[buf.slot],
                                                          &bar_tempty[2 + buf.slot], buf.parity ^ 1u);
                        if (!(ready & 1u))
                            ok = warp_wait(&bar_full[st.slot], st.parity, abort_flag, p.status, p.wait_ns);
                        const uint64_t w_desc = smem_desc_sw128(smem_u32(smem) + st.slot * FG_STAGE_BYTES);
                        const uint32_t d0 = tmem_base + buf.slot * 128;
                        #pragma unroll
                        for (int j = 0; j < 2; ++j)
                        {
                            if (!(ready & (2u << j)))
                                ok = ok && warp_wait(&bar_tempty[2 * j + buf.slot], buf.parity ^ 1u, abort_flag, p.status,
                                                     p.wait_ns);
                            if (!ok) break;
                            tc_fence_after();
                            if (leader)
                            {
                                const uint32_t d = d0 + 256 * j;
                                if (ti.thin)
                                {
                                    const int nc = j ? nc1 : nc0;
                                    const uint32_t idesc = idesc_e4m3_f32(256, nc);
                                    const uint64_t x_desc = w_desc + (2 * FG_W_BYTES + j * (FG_XBOX * FG_BK) >> 4);
                                    if (nc)
                                        #pragma unroll
                                        for (int h = 0; h < 2; ++h)
                                            #pragma unroll
                                            for (int kk = 0; kk < FG_BK / 32; ++kk)
                                                umma_e4m3_pair(d + h * 64, w_desc + h * (FG_W_BYTES >> 4) + 2 * kk,
                                                               x_desc + 2 * kk, idesc, kk != 0);
                                }
                                else
                                {
                                    const uint32_t idesc = idesc_e4m3_f32(256, 128);
                                    const uint64_t x_desc = w_desc + (FG_W_BYTES >> 4);
                                    #pragma unroll
                                    for (int kk = 0; kk < FG_BK / 32; ++kk)
                                        umma_e4m3_pair(d, x_desc + 2 * kk, w_desc + j * (64 * FG_BK >> 4) + 2 * kk, idesc, kk != 0);
                                }
                                umma_commit_pair(j ? &bar_done[st.slot] : &bar_half[st.slot]);
                            }
                            __syncwarp();
                        }
                        if (!ok) break;
                    }
                }
                // the MMAs of the last stages are done before the CTAs leave: the producer's drain waits for them
            }
        }
        else
        {
            // ============================================================ scales
            const int j = (warp - 2) * 32 + lane;           // tokens j and j + 64; weight block j for j < 2
            Ring<FG_SCALES> sr;
            bool ok = true;
            for (int t = cluster; ok && t < total; t += n_clusters)
            {
                const Tile ti = tile_at(p, s_pref, t);
                const int rows = ti.thin ? ti.rows : min(128, ti.rows - 128 * rank);
                const float* sx = p.sx + (int64_t) (ti.row0 + (ti.thin ? 0 : 128 * rank) + j) * p.sx_row + ti.kb0 * p.sx_blk;
                // a block past the last one has sums of zero: any scale will do
                const float* sw = p.sw + ti.e * p.sw_expert + min(weight_block<SWIGLU>(p, ti, rank, j & 1), p.n_blocks - 1) * p.sw_n +
                                  ti.kb0;
                for (int kb = ti.kb0; kb < ti.kb1; ++kb, sr.next())
                {
                    const int q = sr.slot;
                    ok = warp_wait(&bar_sempty[q], sr.parity ^ 1u, abort_flag, p.status, p.wait_ns);
                    if (!ok) break;
                    if (j < rows) cp_async4(&s_sx[q][j], sx);
                    if (j + 64 < rows) cp_async4(&s_sx[q][j + 64], sx + 64 * p.sx_row);
                    if (j < 2) cp_async4(&s_sw[q][j], sw);
                    cp_async_arrive(&bar_sfull[q]);
                    sx += p.sx_blk;
                    sw += 1;
                }
            }
            cp_async_wait_all();
        }
    }
    else
    {
        // ================================================================ epilogue
        setmaxnreg_inc<104>();
        const int g = (warp - 4) >> 2;                      // warpgroup
        const int quarter = warp & 3;
        const int lane_in = quarter * 32 + lane;            // TMEM lane: token (wide) or weight row (thin)
        // registers are short here (64 of sums, 16 on their way): positions from one counter, 32-bit addresses
        Ring<FG_STAGES> sg;
        uint32_t it = 0;
        const uint32_t tempty = in_cta0(&bar_tempty[2 * (g >> 1)]);
        const uint32_t sums = smem_u32(g >> 1 ? bar_done : bar_half);
        const uint32_t tmem = tmem_base + (static_cast<uint32_t>(quarter * 32) << 16) + (g >> 1) * 256 + (g & 1) * 32;
        for (int t = cluster; t < total; t += n_clusters)
        {
            Tile ti = tile_at(p, s_pref, t);
            int blocks = ti.kb1 - ti.kb0;
            uint64_t acc[2][16];                            // 32 columns (wide) or tokens (thin) of each block
            #pragma unroll
            for (int h = 0; h < 2; ++h)
                #pragma unroll
                for (int i = 0; i < 16; ++i) acc[h][i] = 0;
            const bool work = !ti.thin || g * 32 < ti.rows;
            bool ok = true;
            #pragma unroll 1
            for (; blocks > 0; --blocks)
            {
                const uint32_t q = it % FG_SCALES, q_parity = (it / FG_SCALES) & 1u;
                if (!__all_sync(0xffffffffu, mbar_test2(smem_u32(bar_sfull) + q * 8, q_parity, sums + sg.slot * 8, sg.parity)))
                {
                    ok = warp_wait(&bar_sfull[q], q_parity, abort_flag, p.status, p.wait_ns) &&
                         warp_wait(&(g >> 1 ? bar_done : bar_half)[sg.slot], sg.parity, abort_flag, p.status, p.wait_ns);
                    if (!ok) break;
                }
                tc_fence_after();
                const uint32_t taddr = tmem + (it & 1u) * 128;
                auto release = [&] {                        // the buffer is free: its sums are in registers
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) mbar_arrive_cluster(tempty + (it & 1u) * 8);
                };
                if (!ti.thin)
                {
                    const float x = s_sx[q][lane_in];
                    #pragma unroll
                    for (int h = 0; h < 2; ++h)
                    {
                        const uint32_t f = __float_as_uint(x * s_sw[q][h]);
                        const uint64_t ff = pack2(f, f);
                        #pragma unroll
                        for (int c = 0; c < 2; ++c)
                        {
                            uint64_t d[8];
                            tmem_load(taddr + h * 64 + c * 16, d);
                            if (h == 1 && c == 1) release();
                            #pragma unroll
                            for (int i = 0; i < 8; ++i) fma2(acc[h][c * 8 + i], d[i], ff);
                        }
                    }
                }
                else if (work)
                {
                    const float* sc = &s_sx[q][g * 32];
                    const uint32_t w0 = __float_as_uint(s_sw[q][0]), w1 = __float_as_uint(s_sw[q][1]);
                    const uint64_t ww[2] = {pack2(w0, w0), pack2(w1, w1)};
                    #pragma unroll
                    for (int c = 0; c < 2; ++c)
                        if (g * 32 + c * 16 < ti.rows)
                        {
                            #pragma unroll
                            for (int h = 0; h < 2; ++h)
                            {
                                uint64_t d[8];
                                tmem_load(taddr + h * 64 + c * 16, d);
                                if (h == 1 && (c == 1 || g * 32 + 16 >= ti.rows)) release();
                                #pragma unroll
                                for (int i = 0; i < 4; ++i)
                                {
                                    const ulonglong2 f = *reinterpret_cast<const ulonglong2*>(sc + c * 16 + 4 * i);
                                    fma2(acc[h][c * 8 + 2 * i], d[2 * i], mul2(f.x, ww[h]));
                                    fma2(acc[h][c * 8 + 2 * i + 1], d[2 * i + 1], mul2(f.y, ww[h]));
                                }
                            }
                        }
                }
                else release();
                __syncwarp();
                if (lane == 0) mbar_arrive(&bar_sempty[q]);
                ++it;
                sg.next();
            }
            // A warp that gave up says so before the epilogue's barrier, and every warp reads it between this
            // barrier and the next: one decision for all of them.
            if (!ok && lane == 0) s_fail = 1;
            named_bar_sync(5, FG_EPI_THREADS);
            const bool fail = *(volatile int*) &s_fail != 0;
            if (fail)
            {
                named_bar_sync(5, FG_EPI_THREADS);
                break;
            }
            if (ti.thin)
            {
                float* st = &s_stage[g][0][0];
                #pragma unroll
                for (int j0 = 0; j0 < 32; j0 += FG_STEP)
                {
                    const int m0 = g * 32 + j0;
                    if (m0 < ti.rows)
                    {
                        #pragma unroll
                        for (int j = 0; j < FG_STEP; ++j)
                            #pragma unroll
                            for (int h = 0; h < 2; ++h)
                                st[j * 256 + h * 128 + lane_in] = half_of(acc[h][(j0 + j) >> 1], j & 1);
                        named_bar_sync(1 + g, 128);
                        write_step<SWIGLU>(p, ti, rank, st, m0, threadIdx.x & 127);
                        named_bar_sync(1 + g, 128);
                    }
                }
                named_bar_sync(5, FG_EPI_THREADS);
            }
            else if constexpr (!SWIGLU)
            {
                ti.row0 += 128 * rank;                      // this CTA's tokens
                ti.rows -= 128 * rank;
                if (p.out_dtype == 0) store_wide<float>(p, ti, acc, g, lane_in);
                else if (p.out_dtype == 1) store_wide<__half>(p, ti, acc, g, lane_in);
                else store_wide<__nv_bfloat16>(p, ti, acc, g, lane_in);
                named_bar_sync(5, FG_EPI_THREADS);
            }
            else
            {
                // this thread's token: 32 of the block's 128 columns; the largest magnitude of the others comes from
                // the other warpgroups
                float act[32];
                uint32_t mx = 0;
                #pragma unroll
                for (int i = 0; i < 32; ++i)
                {
                    act[i] = clamped_swiglu(half_of(acc[0][i >> 1], i & 1), half_of(acc[1][i >> 1], i & 1), p.limit);
                    mx = max(mx, __float_as_uint(act[i]) & 0x7fffffffu);
                }
                uint32_t (*s_amax)[NT] = reinterpret_cast<uint32_t (*)[NT]>(&s_stage[0][0][0]);     // thin tiles' memory
                s_amax[g][lane_in] = mx;
                named_bar_sync(5, FG_EPI_THREADS);
                mx = max(max(s_amax[0][lane_in], s_amax[1][lane_in]), max(s_amax[2][lane_in], s_amax[3][lane_in]));
                if (128 * rank + lane_in < ti.rows)
                {
                    const float s = block_scale(__uint_as_float(mx), false), inv = reciprocal(s);
                    const int64_t r = ti.row0 + 128 * rank + lane_in;
                    uint32_t w[8];
                    #pragma unroll
                    for (int j = 0; j < 8; ++j)
                    {
                        float q[4];
                        #pragma unroll
                        for (int i = 0; i < 4; ++i) q[i] = quotient(act[4 * j + i], s, inv);
                        w[j] = to_e4m3x2(q[0], q[1]) | to_e4m3x2(q[2], q[3]) << 16;
                    }
                    store32(p.h + r * p.h_stride + ti.nt * kBlock + g * 32, w);     // (rows of h are 128-byte aligned)
                    if (g == 0) p.hs[r * p.hs_row + ti.nt * p.hs_blk] = s;
                }
            }
        }
    }

    // ---- teardown: neither CTA leaves while the other may still use its shared memory or its TMEM
    tc_fence_before();
    __syncthreads();
    cluster_sync();
    if (warp == 1)
    {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
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
std::atomic<int> g_fp8_clusters[kMaxDevices] = {};

int max_clusters()
{
    int dev = 0;
    if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= kMaxDevices) return device_sm_count() / 2;
    const int n = g_fp8_clusters[dev].load(std::memory_order_relaxed);
    return n > 0 ? n : device_sm_count() / 2;
}

constexpr uint32_t kDynBytes = FG_STAGES * FG_STAGE_BYTES + 1024;

}  // namespace

int launch_fp8_gemm(const Fp8GemmProblem& q, cudaStream_t stream)
{
    Fp8GemmArgs p{};
    p.N = q.N; p.K = q.K; p.n_experts = q.n_experts;
    p.n_blocks = (q.N + kBlock - 1) / kBlock;
    const int units = q.swiglu ? q.N / 2 / kBlock : (p.n_blocks + 1) / 2;   // pairs of blocks that belong together
    p.n_wide = units;
    p.n_thin = (units + 1) / 2;
    p.num_kb = (q.K + FG_BK - 1) / FG_BK;
    p.single_count = (int) q.rows;
    p.counts = q.counts; p.row0 = q.row0;
    p.sx = q.sx; p.sx_row = q.sx_row; p.sx_blk = q.sx_blk;
    p.sw = q.sw; p.sw_expert = q.sw_expert; p.sw_n = q.sw_n;
    p.out = q.out; p.out_stride = q.out_stride; p.out_dtype = q.out_dtype; p.accumulate = q.accumulate;
    p.slot = q.slot;
    p.out_vec = reinterpret_cast<uintptr_t>(q.out) % 32 == 0 && q.out_stride * (q.out_dtype == 0 ? 4 : 2) % 32 == 0;
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
    rc = once_per_device(g_fp8_attr_set, "fp8_gemm", [](int dev) {
        cudaError_t err = cudaSuccess;
        auto set = [&](const void* fn, uint32_t bytes) {
            if (err == cudaSuccess) err = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, (int) bytes);
        };
        set((const void*) fp8_gemm_kernel<false>, kDynBytes);
        set((const void*) fp8_gemm_kernel<true>, kDynBytes);
        if (err != cudaSuccess) return set_cuda_error("fp8_gemm: cudaFuncSetAttribute", err);
        // clusters that run at one time (SMs without a partner in their GPC stay out)
        cudaLaunchConfig_t cfg{};
        cfg.gridDim = dim3(2 * 1024);
        cfg.blockDim = dim3(FG_THREADS);
        cfg.dynamicSmemBytes = kDynBytes;
        int n = 0;
        err = cudaOccupancyMaxActiveClusters(&n, fp8_gemm_kernel<true>, &cfg);
        if (err != cudaSuccess || n < 1) return set_cuda_error("fp8_gemm: cudaOccupancyMaxActiveClusters", err);
        g_fp8_clusters[dev] = n;
        return 0;
    });
    if (rc) return rc;
    p.splits = q.splits > 1 ? q.splits : 1;
    p.split_stride = q.split_stride;
    // tiles are counted on the device; this bound only keeps the grid from being larger than the work
    const int64_t tiles = (q.rows / 256 + (q.rows < q.n_experts ? q.rows : q.n_experts)) * p.n_wide * p.splits;
    const int64_t most = max_clusters();
    const dim3 grid(2u * (unsigned) (tiles < most ? tiles : most));
    return q.swiglu ? launch_after("fp8_gemm", fp8_gemm_kernel<true>, grid, FG_THREADS, kDynBytes, stream, tw, tx, p)
                    : launch_after("fp8_gemm", fp8_gemm_kernel<false>, grid, FG_THREADS, kDynBytes, stream, tw, tx, p);
}

int fp8_gemm_splits(int64_t rows, int n_experts, int N, int K)
{
    // the clusters that run at one time (74 on a B200 whose SMs all have a partner, fewer where some do not; a constant, since a
    // workspace's size does not depend on the device), the tiles there will be (an expert's last rows taken for a thin tile),
    // and at least four K blocks a part: 777 x 576 x 4096 takes 22 us in six parts and 31 in one, 32 x 4096 x 4096 17 us in
    // eight and 28 in one
    constexpr int64_t clusters = 72;
    const int64_t units = (N + 255) / 256, kb = (K + FG_BK - 1) / FG_BK;
    const int64_t experts = rows < n_experts ? rows : n_experts;
    const int64_t tiles = rows / 256 * units + experts * ((units + 1) / 2);
    int64_t s = clusters / (tiles > 0 ? tiles : 1);
    if (s > kb / 4) s = kb / 4;
    if (s > 8) s = 8;
    return s < 2 ? 1 : (int) s;
}

}  // namespace exl3b
