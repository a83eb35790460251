// route_logits.cu — routing to experts from a layer's router logits.
//
// For one token with logits l[E] (fp32, fp16 or bf16) and an optional bias b[E]:
//     s    = sigmoid(l)  or  softmax(l) over the token's experts
//     c    = s + b                                   (the selection score; b balances the experts' load)
//     G(g) = sum of the group_top largest c of group g (n_group equal groups of consecutive experts)
//     ids  = the topk experts by c among the topk_group groups with the largest G, best first
//     w    = s[ids] / (sum s[ids] + 1e-20) (the division only if norm) * scale
// Ties go to the lower expert (group) number.  Logits that are NaN or -inf are masked: never chosen, and
// outside the softmax; a token with fewer than topk experts left gets id -1 and weight 0 in its last slots.
// The sigmoid router of GLM-5.3-Flash (docs/research/02-glm-5.3-flash-architecture.md:33) is the case
// of one group; router.cu fuses that case with the router's product for callers that hold hidden states.
//
// One warp per token: lane i holds experts i, i + 32, ... as keys (unsigned integers in the order of the
// floats), and each of the topk rounds is two warp-wide integer reductions (the largest key, then the lowest
// expert that holds it) and a rescan by the lane that owned it.
//
// The choice is the one that exact arithmetic makes.  Without a bias both score functions grow with the
// logit, so experts are ranked by the logits themselves.  With a bias, or for sums of a group's best, the 32-bit
// scores rank them, and wherever two scores that a decision separates are closer than 32-bit arithmetic
// can tell (kTol), that token is decided again in 64 bits.
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
// Two selection scores closer than kTol * (1 + |c|) are not told apart in 32 bits.  A score's error: expf, a
// sum and a division, under 2^-20 of a value that is at most 1, and the rounding of s + b, 2^-24 of it.
// A sum of two doubles that; 8e-6 covers both.
constexpr float kTol = 8e-6f;

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

// The token's whole selection in 64 bits, by one warp: lane j < topk returns the expert of slot j (-1: none).
// A rare path (a near-tie decides, kTol), written for its size: scores are computed again wherever needed.
template <bool SOFTMAX, class Tl>
__device__ __noinline__ int select_in_64_bits(const RouteLogitsArgs& p, const Tl* row, float m, int lane)
{
    double inv = 1.0;
    if (SOFTMAX)
    {
        double z = 0.0;
        for (int e = lane; e < p.E; e += 32)
        {
            const float l = load_logit(row + e);
            if (l > -INFINITY) z += l == m ? 1.0 : exp((double) l - (double) m);
        }
        inv = 1.0 / warp_sum(z);
    }
    bool by_logit = false;                                  // the ranking without a bias
    auto score = [&](int e, bool& ok) {
        const float l = load_logit(row + e);
        ok = l > -INFINITY;
        if (by_logit) return (double) l;
        const double s = SOFTMAX ? (l == m ? 1.0 : exp((double) l - (double) m)) * inv : 1.0 / (1.0 + exp(-(double) l));
        return p.bias ? s + (double) p.bias[e] : s;
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
    unsigned kept = ~0u;
    if (p.topk_group < p.n_group)
    {
        double gs = -INFINITY;                              // lane g: the score of group g
        for (int g = 0; g < p.n_group; ++g)
        {
            double sum = 0.0, pv = 0.0;
            int pe = -1;
            for (int j = 0; j < p.group_top; ++j)
            {
                double v;
                pe = next(g * p.per_group, (g + 1) * p.per_group, ~0u, pv, pe, v);
                if (pe == kNoExpert) { sum = -INFINITY; break; }
                pv = v;
                sum += v;
            }
            if (lane == g) gs = sum;
        }
        int rank = 0;
        for (int g = 0; g < p.n_group; ++g)
        {
            const double o = __shfl_sync(kFull, gs, g);
            rank += o > gs || (o == gs && g < lane);
        }
        kept = __ballot_sync(kFull, lane < p.n_group && rank < p.topk_group);
    }
    by_logit = p.bias == nullptr;
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

// Registers: MPL = the experts a lane holds, at least ceil(E / 32).
template <int MPL, bool SOFTMAX, class Tl>
__global__ __launch_bounds__(RL_THREADS)
void route_logits_kernel(const RouteLogitsArgs p)
{
    extern __shared__ float s_rows[];                       // [RL_WARPS][E]: selection scores (group selection only)
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const bool grouped = p.topk_group < p.n_group;
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
                if (v[i] == v[i]) z += soft_exp(v[i], m);
            inv = 1.0f / warp_sum(z);
        }
        // keys: by the selection score with a bias, by the logit without one
        const bool by_score = p.bias != nullptr;
        uint32_t key[MPL];
        #pragma unroll
        for (int i = 0; i < MPL; ++i)
        {
            float c = v[i];
            if (by_score && c == c)
            {
                const float s = SOFTMAX ? soft_exp(c, m) * inv : 1.0f / (1.0f + expf(-c));
                c = s + __ldg(p.bias + lane + 32 * i);
            }
            key[i] = c == c ? order_key(c) : 0u;
        }
        bool near = false;
        if (grouped)
        {
            // lanes_per_group lanes scan a group's scores from shared memory and merge their two best
            float* sc = s_rows + warp * p.E;
            const bool sums = p.group_top > 1;
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
            {
                const int e = lane + 32 * i;
                if (e >= p.E) continue;
                float c = key[i] ? key_value(key[i]) : -INFINITY;
                if (!by_score && sums && key[i]) c = SOFTMAX ? soft_exp(c, m) * inv : 1.0f / (1.0f + expf(-c));
                sc[e] = c;
            }
            __syncwarp();
            const int lpg = p.lanes_per_group, g = lane / lpg, sub = lane - g * lpg;
            float b1 = -INFINITY, b2 = -INFINITY;
            if (g < p.n_group)
                for (int i = sub; i < p.per_group; i += lpg)
                {
                    const float c = sc[g * p.per_group + i];
                    b2 = fmaxf(b2, fminf(b1, c));
                    b1 = fmaxf(b1, c);
                }
            for (int o = lpg >> 1; o > 0; o >>= 1)
            {
                const float o1 = __shfl_xor_sync(kFull, b1, o), o2 = __shfl_xor_sync(kFull, b2, o);
                b2 = fmaxf(fminf(b1, o1), fmaxf(b2, o2));
                b1 = fmaxf(b1, o1);
            }
            const float mine = g < p.n_group ? (sums ? b1 + b2 : b1) : -INFINITY;
            const float gs = __shfl_sync(kFull, mine, (lane * lpg) & 31);   // lane g: group g
            int rank = 0;
            for (int o = 0; o < p.n_group; ++o)
            {
                const float x = __shfl_sync(kFull, gs, o);
                rank += x > gs || (x == gs && o < lane);
            }
            const bool in = lane < p.n_group && rank < p.topk_group;
            const unsigned kept = __ballot_sync(kFull, in);
            if (by_score || sums)
            {
                const float low = -warp_max(in ? -gs : -INFINITY);          // the last kept and the best dropped
                const float high = warp_max(lane < p.n_group && !in ? gs : -INFINITY);
                near = low - high <= 2.0f * kTol * (1.0f + fabsf(low)) && high > -INFINITY;
            }
            #pragma unroll
            for (int i = 0; i < MPL; ++i)
                if (!((kept >> min((lane + 32 * i) / p.per_group, 31)) & 1u)) key[i] = 0u;
            __syncwarp();                                                    // the row is rewritten for the next token
        }
        // the lane's best: keys are compared in rising expert order, so equal keys leave the lowest expert
        uint32_t lk = 0u;
        int le = kNoExpert;
        #pragma unroll
        for (int i = 0; i < MPL; ++i)
            if (key[i] > lk) { lk = key[i]; le = lane + 32 * i; }
        int my_id = -1;
        float last = INFINITY;
        const int rounds = by_score && !near ? p.topk + 1 : p.topk;          // one more: the best that is not chosen
        for (int j = 0; j < rounds; ++j)
        {
            const uint32_t best = __reduce_max_sync(kFull, lk);
            if (best == 0u) break;
            const int id = __reduce_min_sync(kFull, lk == best ? le : kNoExpert);
            if (by_score)
            {
                const float c = key_value(best);
                near |= j > 0 && last - c <= kTol * (1.0f + fabsf(c));
                last = c;
            }
            if (lane == j && j < p.topk) my_id = id;
            if (le == id)
            {
                lk = 0u;
                le = kNoExpert;
                #pragma unroll
                for (int i = 0; i < MPL; ++i)
                {
                    if (lane + 32 * i == id) key[i] = 0u;
                    if (key[i] > lk) { lk = key[i]; le = lane + 32 * i; }
                }
            }
        }
        if (near) my_id = select_in_64_bits<SOFTMAX, Tl>(p, row, m, lane);
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
void launch_typed(const RouteLogitsArgs& p, int dtype, unsigned grid, size_t smem, cudaStream_t stream)
{
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
    const int64_t want = (T + RL_WARPS - 1) / RL_WARPS;
    const unsigned grid = (unsigned) (want < (1 << 20) ? want : (1 << 20));
    const size_t smem = topk_group < n_group ? sizeof(float) * RL_WARPS * (size_t) E : 0;
    // the smallest instantiation that holds ceil(E / 32) experts a lane
    auto go = [&](auto sm) {
        constexpr bool SM = decltype(sm)::value;
        if (E <= 64) launch_typed<2, SM>(p, dtype, grid, smem, stream);
        else if (E <= 128) launch_typed<4, SM>(p, dtype, grid, smem, stream);
        else if (E <= 288) launch_typed<9, SM>(p, dtype, grid, smem, stream);
        else if (E <= 512) launch_typed<16, SM>(p, dtype, grid, smem, stream);
        else launch_typed<32, SM>(p, dtype, grid, smem, stream);
    };
    if (softmax) go(std::true_type{});
    else go(std::false_type{});
    return check_launch("route_logits");
}

}  // namespace exl3b
