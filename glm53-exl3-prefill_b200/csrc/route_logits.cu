// route_logits.cu — routing to experts from a layer's router logits.
//
// For one token with logits l[E] (fp32, fp16 or bf16) and an optional bias b[E]:
//     s    = sigmoid(l)  or  softmax(l) over the token's experts
//     c    = s + b                                   (the selection score; b balances the experts' load)
//     G(g) = sum of the group_top largest c of group g (n_group equal groups of consecutive experts)
//     ids  = the topk experts by c among the topk_group groups with the largest G, best first
//     w    = s[ids] / (sum s[ids] + 1e-20) (the division only if norm) * scale
// Ties go to the lower expert (group) number.  Logits that are NaN or -inf are masked: never chosen, and
// outside the softmax; a bias of NaN or -inf only keeps its expert from being chosen, and
// +inf counts as the largest float.  A token with fewer than topk
// experts left gets id -1 and weight 0 in its last slots.
// The sigmoid router of GLM-5.3-Flash (docs/research/02-glm-5.3-flash-architecture.md:33) is the case
// of one group; router.cu fuses that case with the router's product for callers that hold hidden states.
//
// One warp per token: lane i holds experts i, i + 32, ... as keys (unsigned integers in the order of the floats) and
// knows its two best; each of the topk rounds is two warp-wide integer reductions (the largest key, then the lowest
// expert that holds it), after which the owner moves up its second best and only looks at its keys again when that is
// gone too.  The bytes of the logits (33 MB for 32768 tokens of 256 experts, 5 us) bound it in principle; the instructions and
// the waits of one warp on its own loads and shuffles do in fact, about 870 instructions a token without groups and 1125 with:
// 8192 tokens of 288 experts take 14.4 us (1.6 by bytes), 32768 of 256 in 8 groups 54 us.
//
// The choice is the one that 64-bit scores make.  Without a bias both score functions grow with the
// logit, so experts are ranked by the logits themselves.  With a bias, scores in 32 bits rank them, and where two scores
// that a decision separates are closer than that arithmetic can tell (kTol), the candidates, one a lane, are
// ranked again by their scores in 64 bits; where two groups nearly tie, the groups are.  Biased scores that are equal in
// 64 bits are ties (sigmoids of logits above 37 all are 1 there).
#include <cstdint>
#include <type_traits>
#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include "common.cuh"
#include "exl3_internal.h"

namespace exl3b {

namespace {

constexpr int RL_THREADS = 128;
constexpr int RL_WARPS = RL_THREADS / 32;
constexpr unsigned kFull = 0xffffffffu;
constexpr int kNoExpert = 0x7fffffff;
// Two selection scores closer than kTol * (1 + |c|) are not told apart in 32 bits.  A score's error: ex2.approx and
// rcp.approx (2^-22 each, relative), the rounding of the exponent's argument (under 2^-24 * |l| s (1 - s) <= 2^-26), for softmax
// the sum's (2^-20, relative): under 1.3e-6 of a value that is at most 1; and the rounding of s + b, 2^-24 of it.  Twice
// that (two scores) is under 3e-6.
constexpr float kTol = 4e-6f;

struct RouteLogitsArgs {
    const void* logits;
    int64_t T, row_stride;
    const float* bias;
    int E, topk, n_group, topk_group, group_top, per_group, lanes_per_group, norm;
    float scale;
    int64_t* ids;
    float* weights;
};

template <class Tl> __device__ __forceinline__ float load_logit(const Tl* p);
template <> __device__ __forceinline__ float load_logit(const float* p) { return *p; }
template <> __device__ __forceinline__ float load_logit(const __half* p) { return __half2float(*p); }
template <> __device__ __forceinline__ float load_logit(const __nv_bfloat16* p) { return __bfloat162float(*p); }

// Unsigned integers in the order of the floats (+0 and -0 equal); 0 is below every float that is not NaN.
__device__ __forceinline__ uint32_t order_key(float v)
{
    const uint32_t u = __float_as_uint(v + 0.0f);
    return (u & 0x80000000u) ? ~u : u | 0x80000000u;
}

__device__ __forceinline__ float key_value(uint32_t k)
{
    return __uint_as_float((k & 0x80000000u) ? k & 0x7fffffffu : ~k);
}

__device__ __forceinline__ double warp_sum(double v)
{
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

__device__ __forceinline__ float warp_sum(float v)
{
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(kFull, v, o);
    return v;
}

__device__ __forceinline__ float warp_max(float v)
{
    for (int o = 16; o > 0; o >>= 1) v = fmaxf(v, __shfl_xor_sync(kFull, v, o));
    return v;
}

// exp(l - m) of the softmax; the largest logit gives 1 even where it is +inf.
__device__ __forceinline__ float soft_exp(float l, float m) { return l == m ? 1.0f : expf(l - m); }

// Scores for ranking: fast, to kTol (results below 2^-126 are zero, which is far below it).
__device__ __forceinline__ float fast_exp2(float x)
{
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
constexpr float kLog2e = 1.44269504f;
__device__ __forceinline__ float fast_exp(float l, float m) { return l == m ? 1.0f : fast_exp2((l - m) * kLog2e); }
__device__ __forceinline__ float fast_sigmoid(float l)
{
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(1.0f + fast_exp2(l * -kLog2e)));
    return r;
}

// A bias of +inf as the largest float, so that sums with masked experts stay out of NaN.
__device__ __forceinline__ float bounded(float b) { return b > 3.402823466e38f ? 3.402823466e38f : b; }

// The selection score of expert e in 64 bits (inv: the softmax's 1 / sum, in 64 bits).
template <bool SOFTMAX>
__device__ __forceinline__ double exact_score(const RouteLogitsArgs& p, float l, int e, float m, double inv)
{
    const double s = SOFTMAX ? (l == m ? 1.0 : exp((double) l - (double) m)) * inv : 1.0 / (1.0 + exp(-(double) l));
    return p.bias ? s + (double) bounded(p.bias[e]) : s;
}

// 1 / sum of the softmax in 64 bits.
template <class Tl>
__device__ __forceinline__ double exact_inverse_sum(const RouteLogitsArgs& p, const Tl* row, float m, int lane)
{
    double z = 0.0;
    for (int e = lane; e < p.E; e += 32)
    {
        const float l = load_logit(row + e);
        if (l > -INFINITY) z += l == m ? 1.0 : exp((double) l - (double) m);
    }
    return 1.0 / warp_sum(z);
}

// The candidates, one per lane (expert mine, -1 past n of them and where fewer experts than slots are left; every other
// expert's score is clearly below the last chosen one), ranked by their scores in 64 bits: lane j < topk returns the
// expert of slot j.  A lane without an expert counts as -inf, which no expert's score is, so empty slots come last.
template <bool SOFTMAX, class Tl>
__device__ __noinline__ int rank_in_64_bits(const RouteLogitsArgs& p, const Tl* row, float m, int lane, int mine, int n)
{
    const double inv = SOFTMAX ? exact_inverse_sum(p, row, m, lane) : 1.0;
    const double c = mine >= 0 ? exact_score<SOFTMAX>(p, load_logit(row + mine), mine, m, inv) : -(double) INFINITY;
    int rank = 0;
    for (int j = 0; j < n; ++j)
    {
        const double o = __shfl_sync(kFull, c, j);
        const int oe = __shfl_sync(kFull, mine, j);
        rank += o > c || (o == c && oe < mine);
    }
    int out = -1;
    for (int j = 0; j < n; ++j)
    {
        const int r = __shfl_sync(kFull, rank, j), e = __shfl_sync(kFull, mine, j);
        if (r == lane) out = e;
    }
    return out;
}

template <class F> __device__ __forceinline__ F lowest();
template <> __device__ __forceinline__ float lowest() { return -INFINITY; }
template <> __device__ __forceinline__ double lowest() { return -(double) INFINITY; }

// The token's whole selection in 64 bits, by one warp: lane j < topk returns the expert of slot j (-1: none).  A path for
// more than 32 candidates that nearly tie, written for its size: scores are computed again wherever needed.
template <bool SOFTMAX, class Tl>
__device__ __noinline__ int select_in_64_bits(const RouteLogitsArgs& p, const Tl* row, float m, int lane, unsigned kept)
{
    const double inv = SOFTMAX ? exact_inverse_sum(p, row, m, lane) : 1.0;
    auto score = [&](int e, bool& ok) {
        const float l = load_logit(row + e);
        const double c = exact_score<SOFTMAX>(p, l, e, m, inv);
        ok = l > -INFINITY && c > lowest<double>();
        return c;
    };
    // the best expert in [lo, hi) that comes after (pv, pe) in the order: larger score first, then lower number
    auto next = [&](int lo, int hi, unsigned groups, double pv, int pe, double& bv) {
        int be = kNoExpert;
        bv = -INFINITY;
        for (int e = lo + lane; e < hi; e += 32)
        {
            bool ok;
            const double c = score(e, ok);
            if (!ok || !(groups >> (p.n_group > 1 ? e / p.per_group : 0) & 1u)) continue;
            const bool after = pe < 0 || c < pv || (c == pv && e > pe);
            if (after && (be == kNoExpert || c > bv)) { bv = c; be = e; }
        }
        for (int o = 16; o > 0; o >>= 1)
        {
            const double ov = __shfl_xor_sync(kFull, bv, o);
            const int oe = __shfl_xor_sync(kFull, be, o);
            if (oe != kNoExpert && (be == kNoExpert || ov > bv || (ov == bv && oe < be))) { bv = ov; be = oe; }
        }
        return be;
    };
    int mine = -1, pe = -1;
    double pv = 0.0;
    for (int j = 0; j < p.topk; ++j)
    {
        double v;
        pe = next(0, p.E, kept, pv, pe, v);
        if (pe == kNoExpert) break;
        pv = v;
        if (lane == j) mine = pe;
    }
    return mine;
}

// The groups kept (a bit each) by their scores, from the token's selection scores sc[E] in shared memory.  A group's score is
// taken as half of its definition's (a mean where two are summed): the order is the same and no sum overflows.  `tie`:
// whether a kept group's score may really be below a dropped one's, each score being off by up to kTol / 2 times (1 +
// the mean of its addends' magnitudes): two of opposite sign may cancel in the sum, their roundings do not.
// lanes_per_group lanes scan a group and merge their two best.
template <class F>
__device__ __forceinline__ unsigned kept_groups(const RouteLogitsArgs& p, const F* sc, int lane, bool& tie)
{
    const int lpg = p.lanes_per_group, g = lane / lpg, sub = lane - g * lpg;
    F b1 = lowest<F>(), b2 = lowest<F>();
    if (g < p.n_group)
        for (int i = sub; i < p.per_group; i += lpg)
        {
            const F c = sc[g * p.per_group + i];
            b2 = max(b2, min(b1, c));
            b1 = max(b1, c);
        }
    for (int o = lpg >> 1; o > 0; o >>= 1)
    {
        const F o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
        b2 = max(min(b1, o1), max(b2, o2));
        b1 = max(b1, o1);
    }
    if (p.group_top == 1) b2 = b1;
    const F half1 = F(0.5) * b1, half2 = F(0.5) * b2;
    const F gs = __shfl_sync(kFull, half1 + half2, (lane * lpg) & 31);      // lane g: group g
    int rank = 0;
    for (int o = 0; o < p.n_group; ++o)
    {
        const F x = __shfl_sync(kFull, gs, o);
        rank += x > gs || (x == gs && o < lane);
    }
    const bool is_group = lane < p.n_group, is_kept = is_group && rank < p.topk_group;
    if constexpr (std::is_same_v<F, float>)
    {
        // a group without the experts for its score is at -inf, above or below which nothing is in doubt
        const float mag = __shfl_sync(kFull, fabsf(half1) + fabsf(half2), (lane * lpg) & 31);
        const float err = gs > -INFINITY ? 0.5f * kTol * (1.0f + mag) : 0.0f;
        const uint32_t low = __reduce_min_sync(kFull, is_kept ? order_key(gs - err) : kFull);
        const uint32_t next = __reduce_max_sync(kFull, is_group && !is_kept ? order_key(gs + err) : 0u);
        tie = next >= low && low > order_key(-INFINITY);
    }
    return __ballot_sync(kFull, is_kept);
}

// The same from scores in 64 bits, which replace sc.
template <bool SOFTMAX, class Tl>
__device__ __noinline__ unsigned kept_groups_in_64_bits(const RouteLogitsArgs& p, const Tl* row, float m, int lane, double* sc)
{
    const double inv = SOFTMAX ? exact_inverse_sum(p, row, m, lane) : 1.0;
    __syncwarp();
    for (int e = lane; e < p.E; e += 32)
    {
        const float l = load_logit(row + e);
        const double c = exact_score<SOFTMAX>(p, l, e, m, inv);
        sc[e] = l > -INFINITY && c > lowest<double>() ? c : lowest<double>();
    }
    __syncwarp();
    bool tie;
    return kept_groups<double>(p, sc, lane, tie);
}

// CTAs that an SM holds at a time (64, 80 or 128 registers a thread).
constexpr int rl_resident(int MPL) { return MPL <= 9 ? 8 : MPL <= 16 ? 6 : 4; }

// Registers: MPL = the experts a lane holds, at least ceil(E / 32).
template <int MPL, bool SOFTMAX, class Tl>
__global__ __launch_bounds__(RL_THREADS, rl_resident(MPL))
void route_logits_kernel(const __grid_constant__ RouteLogitsArgs p)
{
    extern __shared__ double s_rows[];                      // [RL_WARPS][E]: selection scores (group selection only)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool grouped = p.topk_group < p.n_group;
    const bool by_score = p.bias != nullptr;                // keys: the selection score with a bias, else the logit
    float bias[MPL];
    uint32_t group[MPL];                                    // the group's bit
    #pragma unroll
    for (int i = 0; i < MPL; ++i)
    {
        const int e = lane + 32 * i;
        bias[i] = by_score && e < p.E ? bounded(__ldg(p.bias + e)) : 0.0f;
        group[i] = e < p.E ? 1u << (e / p.per_group) : 0u;
    }
    for (int64_t t = (int64_t) blockIdx.x * RL_WARPS + warp; t < p.T; t += (int64_t) gridDim.x * RL_WARPS)
    {
        const Tl* row = reinterpret_cast<const Tl*>(p.logits) + t * p.row_stride;
        float v[MPL];                                       // the logits; NaN: masked or past the end
        #pragma unroll
        for (int i = 0; i < MPL; ++i)
        {
            const int e = lane + 32 * i;
            const float l = e < p.E ? load_logit(row + e) : NAN;
            v[i] = l > -INFINITY ? l : NAN;
        }
        float m = 0.0f, inv = 1.0f;
        if (SOFTMAX)
        {
            m = -INFINITY;
            #pragma unroll
            for (int i = 0; i < MPL; ++i) m = fmaxf(m, v[i]);               // fmaxf passes over NaN
            m = warp_max(m);
            float z = 0.0f;
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
                if (v[i] == v[i]) z += fast_exp(v[i], m);
            inv = 1.0f / warp_sum(z);
        }
        uint32_t key[MPL];
        #pragma unroll
        for (int i = 0; i < MPL; ++i)
        {
            float c = v[i];
            if (by_score) c = (SOFTMAX ? fast_exp(c, m) * inv : fast_sigmoid(c)) + bias[i];
            key[i] = c > -INFINITY ? order_key(c) : 0u;                     // masked by its logit (NaN here) or its bias
        }
        unsigned kept = ~0u;
        if (grouped)
        {
            float* sc = reinterpret_cast<float*>(s_rows + warp * p.E);
            const bool sums = p.group_top > 1;
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
            {
                const int e = lane + 32 * i;
                if (e >= p.E) continue;
                float c = key[i] ? key_value(key[i]) : -INFINITY;
                if (!by_score && sums && key[i]) c = SOFTMAX ? fast_exp(c, m) * inv : fast_sigmoid(c);
                sc[e] = c;
            }
            __syncwarp();
            bool tie;
            kept = kept_groups<float>(p, sc, lane, tie);
            if ((by_score || sums) && tie)
                kept = kept_groups_in_64_bits<SOFTMAX, Tl>(p, row, m, lane, s_rows + warp * p.E);
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
                if (!(kept & group[i])) key[i] = 0u;
            __syncwarp();                                                    // the row is rewritten for the next token
        }
        int my_id = -1;
        {
            // the lane's two best; keys are compared in rising expert order, so equal keys leave the lower expert first
            uint32_t k1 = 0u, k2 = 0u;
            int i1 = kNoExpert, i2 = kNoExpert;
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
            {
                const bool first = key[i] > k1, second = key[i] > k2;
                k2 = first ? k1 : second ? key[i] : k2;
                i2 = first ? i1 : second ? lane + 32 * i : i2;
                k1 = first ? key[i] : k1;
                i1 = first ? lane + 32 * i : i1;
            }
            uint32_t my_key = 0u;                           // lane n: the n-th best
            auto take = [&](int n) {
                const uint32_t best = __reduce_max_sync(kFull, k1);
                const int id = __reduce_min_sync(kFull, k1 == best ? i1 : kNoExpert);
                if (lane == n)
                {
                    my_key = best;
                    my_id = best ? id : -1;
                }
                if (i1 == id && best)
                {
                    if (k2 == 0u)                           // both known ones are gone: the best that comes after
                    {
                        #pragma unroll
                        for (int i = 0; i < MPL; ++i)
                        {
                            const int e = lane + 32 * i;
                            const bool after = key[i] < best || (key[i] == best && e > id);
                            if (after && key[i] > k2) { k2 = key[i]; i2 = e; }
                        }
                    }
                    k1 = k2;
                    i1 = i2;
                    k2 = 0u;
                    i2 = kNoExpert;
                }
            };
            const int k = p.topk;
            for (int n = 0; n < k; ++n) take(n);
            if (by_score)
            {
                // near-ties among the chosen, and of the last of them with what is left
                const uint32_t left = __reduce_max_sync(kFull, k1);
                const uint32_t below = __shfl_down_sync(kFull, my_key, 1);
                const uint32_t next = lane == k - 1 ? left : below;
                const float c = key_value(my_key), tol = kTol * (1.0f + fabsf(c));
                const bool tie = lane < k && next && c - key_value(next) <= tol;
                if (__any_sync(kFull, tie))
                {
                    const uint32_t last = __shfl_sync(kFull, my_key, k - 1);
                    const float bar = key_value(last) - kTol * (1.0f + fabsf(key_value(last)));
                    int n = k;                              // candidates: topk, and what may belong before the last of them
                    bool more = true;
                    for (;; ++n)
                    {
                        const uint32_t best = __reduce_max_sync(kFull, k1);
                        more = best && last && key_value(best) >= bar;
                        if (!more || n == 32) break;
                        take(n);
                    }
                    my_id = more ? select_in_64_bits<SOFTMAX, Tl>(p, row, m, lane, kept)
                                 : rank_in_64_bits<SOFTMAX, Tl>(p, row, m, lane, my_id, n);
                }
            }
            if (lane >= p.topk) my_id = -1;
        }
        float s = 0.0f;
        if (my_id >= 0)
        {
            const float l = load_logit(row + my_id);
            s = SOFTMAX ? soft_exp(l, m) * inv : 1.0f / (1.0f + expf(-l));
        }
        const float sum = warp_sum(s);
        if (lane < p.topk)
        {
            p.ids[t * p.topk + lane] = my_id;
            p.weights[t * p.topk + lane] = (p.norm ? s / (sum + 1e-20f) : s) * p.scale;
        }
    }
}

template <int MPL, bool SOFTMAX>
void launch_typed(const RouteLogitsArgs& p, int dtype, size_t smem, cudaStream_t stream)
{
    // as many CTAs as run at one time, each warp with the same number of tokens (give or take one) and its biases
    // in registers
    const int64_t want = (p.T + RL_WARPS - 1) / RL_WARPS, most = (int64_t) device_sm_count() * rl_resident(MPL);
    const int64_t rounds = (want + most - 1) / most;
    const unsigned grid = (unsigned) ((want + rounds - 1) / rounds);
    if (dtype == 0) route_logits_kernel<MPL, SOFTMAX, float><<<grid, RL_THREADS, smem, stream>>>(p);
    else if (dtype == 1) route_logits_kernel<MPL, SOFTMAX, __half><<<grid, RL_THREADS, smem, stream>>>(p);
    else route_logits_kernel<MPL, SOFTMAX, __nv_bfloat16><<<grid, RL_THREADS, smem, stream>>>(p);
}

}  // namespace

int launch_route_logits(const void* logits, int dtype, int64_t T, int E, int64_t row_stride, const float* bias,
                        int softmax, int n_group, int topk_group, int group_top, int topk, int norm, float scale,
                        int64_t* ids, float* weights, cudaStream_t stream)
{
    RouteLogitsArgs p{};
    p.logits = logits; p.T = T; p.row_stride = row_stride; p.bias = bias; p.E = E; p.topk = topk;
    p.n_group = n_group; p.topk_group = topk_group; p.group_top = group_top; p.per_group = E / n_group;
    p.lanes_per_group = 1;
    while (2 * p.lanes_per_group * n_group <= 32) p.lanes_per_group *= 2;
    p.norm = norm; p.scale = scale; p.ids = ids; p.weights = weights;
    const size_t smem = topk_group < n_group ? sizeof(double) * RL_WARPS * (size_t) E : 0;
    // the smallest instantiation that holds ceil(E / 32) experts a lane
    auto go = [&](auto sm) {
        constexpr bool SM = decltype(sm)::value;
        if (E <= 64) launch_typed<2, SM>(p, dtype, smem, stream);
        else if (E <= 128) launch_typed<4, SM>(p, dtype, smem, stream);
        else if (E <= 256) launch_typed<8, SM>(p, dtype, smem, stream);
        else if (E <= 288) launch_typed<9, SM>(p, dtype, smem, stream);
        else if (E <= 512) launch_typed<16, SM>(p, dtype, smem, stream);
        else launch_typed<32, SM>(p, dtype, smem, stream);
    };
    if (softmax) go(std::true_type{});
    else go(std::false_type{});
    return check_launch("route_logits");
}

}  // namespace exl3b
