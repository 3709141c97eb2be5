// MoE routing on the device: top-k selection and the stable sort of (token, expert) pairs by expert.
//
// Replaces the chain of torch calls at the head of cinnamon's MoE.forward (src/layers.py:122-148):
// sigmoid, + expert_bias, topk, gather, normalise, sort by expert, token_indices, bincount.  Two or three launches:
//
//   route_topk_kernel     one warp per token: sigmoid scores, the k largest of score + bias (ties: the lower
//                         expert id), gates = score / (sum of the k scores + 1e-9); every CTA also leaves a histogram
//                         of the experts its tokens selected in the workspace
//   route_scan_kernel     the running sum of those histograms over the CTAs (the histograms become offsets) -> counts.  With 32 CTAs or fewer the scatter kernel does this itself.
//   route_scatter_kernel  the same CTAs again: an exclusive scan of the counts gives every expert's first row, and every
//                         pair gets the next free row of its expert, pairs taken in (token, slot) order, so the order is
//                         that of a stable sort and the same on every run; writes token_indices / sorted_scores /
//                         sorted_experts, the experts' row ranges, and per token its k rows in ascending order with their
//                         gates (what the combine pass reads)
//
// The workspace (one int per CTA and expert, and one more per expert) is the only memory beyond inputs and outputs.
#include "common.cuh"
#include <mutex>

namespace cinn {

constexpr int ROUTE_MAX_TOKENS_PER_CTA = 128;
constexpr int ROUTE_FEW_CTAS = 32;             // up to here the scatter kernel sums the histograms itself
constexpr int64_t ROUTE_STATIC_MAX_INTS = 1 << 19;                     // 2 MiB: the built-in scratch (moe_route_static)

// Tokens per CTA, a power of two: as few as one per warp while that is at most five CTAs per SM, more for more tokens.  Selecting
// the top k is a serial chain of shuffles per token, so what counts is how many warps there are, until the histograms of every
// CTA cost more than the chains save; five per SM is where the measured lines cross (us at 8 / 16 / 32 / 64 / 128 tokens per CTA:
// 2048 tokens x 256 experts 27 / 29 / 41 / 66 / 116, 8192 x 64 37 / 31 / 31 / 39 / 64, 16384 x 256 82 / 67 / 64 / 78 / 121,
// 32768 x 256 150 / 117 / 104 / 107 / 137, 131072 x 256 539 / 414 / 346 / 322 / 330).  (Any multiple of 8 instead: 24 and 72 tokens
// are up to 11 % slower than 32 and 128 with 8 pairs a token, which the scatter takes 256 at a time.)  Fewer CTAs where their
// histograms would not fit the built-in scratch, so that it serves what it serves at 128 tokens per CTA.
static inline int route_tokens_per_cta(int64_t T, int E) {
    int64_t per = 8;
    while (per < ROUTE_MAX_TOKENS_PER_CTA &&
           (T > per * 5 * sm_count() || ((T + per - 1) / per + 1) * E > ROUTE_STATIC_MAX_INTS)) per *= 2;
    return (int)per;
}

template <typename L> __device__ __forceinline__ float logit(L v);
template <> __device__ __forceinline__ float logit<float>(float v) { return v; }
template <> __device__ __forceinline__ float logit<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float logit<__half>(__half v) { return __half2float(v); }

template <typename L> __device__ __forceinline__ L from_float(float v);
template <> __device__ __forceinline__ float from_float<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half from_float<__half>(float v) { return __float2half_rn(v); }

constexpr int ROUTE_MAX_EXPERTS = 1024;
constexpr int ROUTE_MAX_TOPK = 32;

template <int VPL, typename L>      // expert values per lane, E <= 32 * VPL
__global__ void __launch_bounds__(256)
route_topk_kernel(const L* __restrict__ logits, const float* __restrict__ bias, int T, int E, int top_k, int tokens_per_cta,
                  int* __restrict__ top_experts, float* __restrict__ top_gates, int* __restrict__ hist) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_hist[ROUTE_MAX_EXPERTS];
    for (int e = threadIdx.x; e < E; e += 256) s_hist[e] = 0;
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t_begin = blockIdx.x * tokens_per_cta;
    const int t_end = min(t_begin + tokens_per_cta, T);
    float b[VPL];
#pragma unroll
    for (int i = 0; i < VPL; ++i) b[i] = (lane + 32 * i < E) ? bias[lane + 32 * i] : 0.0f;
    for (int t = t_begin + warp; t < t_end; t += 8) {
        float s[VPL], sel[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            const int e = lane + 32 * i;
            if (e < E) {
                const float x = logit<L>(logits[(int64_t)t * E + e]);
                s[i] = __fdiv_rn(1.0f, 1.0f + expf(-x));                  // torch.sigmoid in fp32
                sel[i] = s[i] + b[i];
                if (sel[i] != sel[i]) sel[i] = -INFINITY;                  // a NaN is never selected
            } else {
                s[i] = 0.0f;
                sel[i] = -INFINITY;
            }
        }
        float my_score = 0.0f;
        int my_expert = 0;
        for (int r = 0; r < top_k; ++r) {
            float best = -INFINITY;
            int best_e = 0x7fffffff;
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (sel[i] > best) { best = sel[i]; best_e = lane + 32 * i; }
            if (best == -INFINITY) best_e = 0x7fffffff;
#pragma unroll
            for (int o = 16; o > 0; o >>= 1) {
                const float ov = __shfl_xor_sync(0xffffffffu, best, o);
                const int oe = __shfl_xor_sync(0xffffffffu, best_e, o);
                if (ov > best || (ov == best && oe < best_e)) { best = ov; best_e = oe; }
            }
            // fewer than k selectable experts (E < k, or NaNs): fall back to the lowest unused ids
            if (best_e == 0x7fffffff) best_e = r < E ? r : 0;
            float sc = 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (lane + 32 * i == best_e) { sc = s[i]; sel[i] = -INFINITY; }
            sc = __shfl_sync(0xffffffffu, sc, best_e & 31);
            if (lane == r) { my_score = sc; my_expert = best_e; }
        }
        float sum = lane < top_k ? my_score : 0.0f;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane < top_k) {
            top_experts[(int64_t)t * top_k + lane] = my_expert;
            top_gates[(int64_t)t * top_k + lane] = __fdiv_rn(my_score, sum + 1e-9f);
            atomicAdd(&s_hist[my_expert], 1);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 256) hist[(int64_t)blockIdx.x * E + e] = s_hist[e];
}

// ---------------------------------------------------------------------------
// The router's other forms: softmax scores, groups of experts, gates as they are or scaled (moe_route_form)
//
//   s = sigmoid(logit) or softmax(logits);  chosen by s + bias: first the groups (of equally many neighbours) with the largest sums of
//   their two best, then the k best experts in them, ties to the lower id;  gate = scale * s / (sum of the k s + 1e-9), or scale * s
//
// Which expert is the last to be chosen can hang on the last bit of a score, so the choice is the one that 64-bit arithmetic makes.
// Hardly any token needs it: a warp chooses with quick scores and looks at the gaps between those it chose and to the next ones; where one
// is too small to be sure of (and not a tie of the same logit and bias), those that can be meant are ranked in 64 bits, a lane
// each.  Where it is a group that is in doubt, a softmax with a bias, or a NaN, the whole token is (route_exact).  Gates come
// from the chosen experts' logits in fp32.
// ---------------------------------------------------------------------------
struct RouteForm {
    int n_groups, top_groups, renormalise;
    float scale;
};

constexpr int ROUTE_MAX_GROUPS = 32;

__device__ __forceinline__ uint32_t ordered(float v) {
    const uint32_t b = __float_as_uint(v);
    return b ^ ((uint32_t)((int)b >> 31) | 0x80000000u);
}
__device__ __forceinline__ float unordered(uint32_t k) { return __uint_as_float(k & 0x80000000u ? k & 0x7fffffffu : ~k); }
__device__ __forceinline__ float warp_sum(float v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ double warp_sum(double v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}

// The groups of rank < top_groups among the warp's lanes' scores (lane g: group g), as a mask; equal scores: the lower group first
template <typename F>
__device__ __forceinline__ unsigned best_groups(F score, int n_groups, int top_groups, int lane) {
    int rank = 0;
    for (int g = 0; g < n_groups; ++g) {
        const F o = __shfl_sync(0xffffffffu, score, g);
        rank += o > score || (o == score && g < lane);
    }
    return __ballot_sync(0xffffffffu, lane < n_groups && rank < top_groups);
}

__device__ __forceinline__ uint64_t ordered(double v) {
    const uint64_t b = (uint64_t)__double_as_longlong(v);
    return b >> 63 ? ~b : b | 0x8000000000000000ull;
}
__device__ __forceinline__ double unordered(uint64_t k) { return __longlong_as_double((long long)(k >> 63 ? k & 0x7fffffffffffffffull : ~k)); }
__device__ __forceinline__ uint64_t reduce_max(uint64_t k) {
    const uint32_t hi = __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32));
    return (uint64_t)hi << 32 | __reduce_max_sync(0xffffffffu, (uint32_t)(k >> 32) == hi ? (uint32_t)k : 0u);
}

// One token in 64 bits, all of it; returns lane r's expert (r < top_k).
template <int VPL, typename L, bool SOFTMAX>
__device__ __noinline__ int route_exact(const L* __restrict__ row, const float* __restrict__ bias, int E, int top_k, int n_groups, int top_groups) {
    const int lane = threadIdx.x & 31, e0 = lane * VPL;
    uint64_t key[VPL];                                       // score + bias, ordered; 0: not to be chosen
    {
        float x[VPL];
        double sel[VPL], m = 0.0, sum = 1.0;
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = e0 + i < E ? logit<L>(row[e0 + i]) : -INFINITY;
        if constexpr (SOFTMAX) {
            float top = x[0];
#pragma unroll
            for (int i = 1; i < VPL; ++i) top = fmaxf(top, x[i]);
            m = (double)warp_max(top);
            sum = 0.0;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            sel[i] = exp(SOFTMAX ? (double)x[i] - m : -(double)x[i]);
            if (SOFTMAX && e0 + i < E) sum += sel[i];
        }
        if constexpr (SOFTMAX) sum = warp_sum(sum);
#pragma unroll
        for (int i = 0; i < VPL; ++i) {
            sel[i] = SOFTMAX ? sel[i] / sum : 1.0 / (1.0 + sel[i]);
            if (bias && e0 + i < E) sel[i] += (double)bias[e0 + i];
            key[i] = e0 + i < E ? ordered(sel[i] == sel[i] ? sel[i] : (double)-INFINITY) : 0ull;        // a NaN comes last
        }
    }
    if (n_groups > 1) {
        const int per = E / n_groups;
        double mine = -INFINITY;
        for (int g = 0; g < n_groups; ++g) {
            uint64_t a = 0, c = 0;                           // the group's two best
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                const uint64_t k = e0 + i >= g * per && e0 + i < (g + 1) * per ? key[i] : 0ull;
                c = max(c, min(a, k));
                a = max(a, k);
            }
            const uint64_t top = reduce_max(a);
            const int owner = __ffs(__ballot_sync(0xffffffffu, a == top)) - 1;
            const uint64_t next = reduce_max(lane == owner ? c : a);
            if (lane == g) mine = per > 1 ? unordered(top) + unordered(next) : unordered(top);
        }
        if (mine != mine) mine = -INFINITY;                  // (infinities of both signs)
        const unsigned groups = best_groups(mine, n_groups, top_groups, lane);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (e0 + i < E && !(groups >> ((unsigned)(e0 + i) / (unsigned)per) & 1)) key[i] = 0ull;
    }
    int my_expert = 0;
    for (int r = 0; r < top_k; ++r) {
        uint64_t best = 0;
        int at = 0;
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (key[i] > best) { best = key[i]; at = i; }
        const uint64_t top = reduce_max(best);
        const int w = __ffs(__ballot_sync(0xffffffffu, best == top)) - 1, e = w * VPL + __shfl_sync(0xffffffffu, at, w);
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (lane == w && i == at) key[i] = 0ull;
        if (lane == r) my_expert = e;
    }
    return my_expert;
}

// The same for a list that is known to hold the best: lane r < n has an expert, its logit and bias; afterwards lane r has the expert of
// rank r.  Scores of a softmax without a bias are compared before their common quotient.
template <bool SOFTMAX>
__device__ __noinline__ int rank_exact(int expert, float x, float bias, float m, int n) {
    const int lane = threadIdx.x & 31;
    const double e = exp(SOFTMAX ? (double)x - (double)m : -(double)x), mine = SOFTMAX ? e : 1.0 / (1.0 + e) + (double)bias;
    int rank = 0;
    for (int j = 0; j < n; ++j) {
        const double o = __shfl_sync(0xffffffffu, mine, j);
        const int oe = __shfl_sync(0xffffffffu, expert, j);
        rank += o > mine || (o == mine && oe < expert);
    }
    int out = 0;
    for (int j = 0; j < n; ++j) {
        const int r = __shfl_sync(0xffffffffu, rank, j), oe = __shfl_sync(0xffffffffu, expert, j);
        if (r == lane) out = oe;
    }
    return out;
}

__device__ __forceinline__ float exp2_approx(float x) {          // relative error 2^-22
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
__device__ __forceinline__ float rcp_approx(float x) {           // relative error 2^-23
    float r;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}

// a lane's VPL neighbouring logits; vec: rows of whole, aligned pieces
template <int VPL, typename L>
__device__ __forceinline__ void load_logits(const L* __restrict__ row, int e0, int E, bool vec, float (&x)[VPL]) {
    constexpr int BYTES = VPL * (int)sizeof(L) < 16 ? VPL * (int)sizeof(L) : 16, PER = BYTES / (int)sizeof(L);
    struct alignas(BYTES) Piece { L v[PER]; };
    if (vec) {
#pragma unroll
        for (int i = 0; i < VPL; i += PER) {
            if (e0 < E) {
                const Piece q = *reinterpret_cast<const Piece*>(row + e0 + i);
#pragma unroll
                for (int j = 0; j < PER; ++j) x[i + j] = logit<L>(q.v[j]);
            } else {
#pragma unroll
                for (int j = 0; j < PER; ++j) x[i + j] = -INFINITY;
            }
        }
    } else {
#pragma unroll
        for (int i = 0; i < VPL; ++i) x[i] = e0 + i < E ? logit<L>(row[e0 + i]) : -INFINITY;
    }
}

constexpr int ROUTE_KEPT = 8;                                // keys that a lane keeps, at most

__device__ __forceinline__ void order_keys(uint32_t& a, uint32_t& b) { const uint32_t hi = max(a, b); b = min(a, b); a = hi; }

// The largest KEEP of VPL keys, in falling order: pieces of KEEP sorted (odd-even merges), and merged by their larger halves (bitonic)
template <int VPL, int KEEP>
__device__ __forceinline__ void largest_keys(const uint32_t (&k)[VPL], uint32_t (&out)[KEEP]) {
#pragma unroll
    for (int at = 0; at < VPL; at += KEEP) {
        uint32_t q[KEEP];
#pragma unroll
        for (int i = 0; i < KEEP; ++i) q[i] = k[at + i];
#pragma unroll
        for (int p = 1; p < KEEP; p *= 2)
#pragma unroll
            for (int w = p; w >= 1; w /= 2)
#pragma unroll
                for (int j = w % p; j + w < KEEP; j += 2 * w)
#pragma unroll
                    for (int i = 0; i < w; ++i)
                        if (j + i + w < KEEP && (j + i) / (2 * p) == (j + i + w) / (2 * p)) order_keys(q[j + i], q[j + i + w]);
        if (at == 0) {
#pragma unroll
            for (int i = 0; i < KEEP; ++i) out[i] = q[i];
        } else {
#pragma unroll
            for (int i = 0; i < KEEP; ++i) out[i] = max(out[i], q[KEEP - 1 - i]);
#pragma unroll
            for (int w = KEEP / 2; w >= 1; w /= 2)
#pragma unroll
                for (int i = 0; i < KEEP; ++i)
                    if ((i & w) == 0) order_keys(out[i], out[i + w]);
        }
    }
}

// What it is made of are integer instructions at half the rate of the floating-point ones: selections, comparisons, minima.  So a lane's VPL
// neighbouring experts are keys that need little of them: score + bias, made positive by a common offset, is a float whose bits are in order
// as they are, and its last bits are the expert's number in the lane (the lower one larger).  A lane keeps its eight largest, sorted; should
// one run out of them, the token is chosen in 64 bits.  A round is one reduction, a vote and a shift of the winner's keys.  8 of 256 experts,
// 32768 tokens, 46 us, 760 instructions a token, 16 of them a round.  (All keys of a lane unsorted, with a look through the winner's: 1280
// and 83 us; 1024 experts, all 32 keys of a lane sorted: 281 us in all, like this 110.)  What bounds it now is latency: of 63 thousand active cycles at that size a
// scheduler issues in 42 thousand and the integer pipe works in 31 thousand; 30 of 40 warps are resident, and a warp waits for a token's logits with
// none of the next one's on their way.  32 of more experts than 32 always go through route_exact, since the list has no place for the one behind
// the last (4096 tokens to 32 of 64 32 us, to 31 of them 26).
//
// Errors of the quick scores.  Sigmoid: the exponent's rounding is |x| 2^-24 of e^-x, its part in the score s (1 - s) |x| 2^-24 < 2^-26, and
// ex2, the sum and rcp add less than 2^-22: two scores are sure to be in order when they are 2^-20 apart, and HIDDEN of the key: what
// its last bits hide, and the sum with the bias.  Softmax: p |x - max| 2^-24 is below 2^-25 of the largest p, ex2, the sum and the
// quotient are 2^-21 of p: 2^-19 of the largest p.  A group's sum of two: twice as much.
template <int VPL, typename L, bool SOFTMAX>                 // E <= 32 * VPL
__global__ void __launch_bounds__(256, VPL <= 8 ? 5 : 2)
route_form_kernel(const L* __restrict__ logits, const float* __restrict__ bias, int T, int E, int top_k, const RouteForm form, int tokens_per_cta, int vec,
                  int* __restrict__ top_experts, float* __restrict__ top_gates, int* __restrict__ hist) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_hist[ROUTE_MAX_EXPERTS];
    __shared__ uint2 s_list[8][32];                                            // per warp: the chosen keys and their lanes
    for (int e = threadIdx.x; e < E; e += 256) s_hist[e] = 0;
    __syncthreads();
    constexpr int KEEP = VPL < ROUTE_KEPT ? VPL : ROUTE_KEPT;
    constexpr uint32_t INDEX = VPL - 1;
    constexpr float HIDDEN = (float)(2 * VPL + 4) * 0x1p-23f;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e0 = lane * VPL;
    const uint32_t below = (1u << lane) - 1u;
    const int t_end = min((int)(blockIdx.x + 1) * tokens_per_cta, T);
    const int per = E / form.n_groups, lanes_per = per / VPL;                  // a group's experts; its lanes, where they are whole
    const bool whole = per % VPL == 0 && (lanes_per & (lanes_per - 1)) == 0;
    const unsigned my_group = whole ? (unsigned)lane / (unsigned)lanes_per & 31u : 0u;
    float b[VPL], lowest = 0.0f;
    bool bans = false;                                                         // biases that keep experts out
#pragma unroll
    for (int i = 0; i < VPL; ++i) {
        b[i] = bias && e0 + i < E ? bias[e0 + i] : 0.0f;
        if (b[i] <= -1e30f) { b[i] = -1e30f; bans = true; }
        else lowest = fminf(lowest, b[i]);
    }
    bans = __any_sync(0xffffffffu, bans);
    lowest = -warp_max(-lowest);
#pragma unroll
    for (int i = 0; i < VPL; ++i) b[i] -= lowest;
    for (int t = blockIdx.x * tokens_per_cta + warp; t < t_end; t += 8) {
        const L* row = logits + (int64_t)t * E;
        float m = 0.0f, sum = 1.0f, near;
        uint32_t key[VPL];                                                     // 0: not to be chosen
        float odd = 0.0f;                                                      // a NaN where a score is a NaN or infinite
        {
            float x[VPL];
            load_logits<VPL, L>(row, e0, E, vec, x);
            if constexpr (SOFTMAX) {
                m = x[0];
#pragma unroll
                for (int i = 1; i < VPL; ++i) m = fmaxf(m, x[i]);
                m = warp_max(m);
                float part = 0.0f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) {
                    x[i] = exp2_approx((x[i] - m) * 1.4426950408889634f);
                    part += x[i];
                }
                sum = warp_sum(part);
                const float inv = rcp_approx(sum);
                near = inv * 0x1p-19f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) x[i] = fmaf(x[i], inv, b[i]);
            } else {
                near = 0x1p-20f;
#pragma unroll
                for (int i = 0; i < VPL; ++i) x[i] = rcp_approx(1.0f + exp2_approx(x[i] * -1.4426950408889634f)) + b[i];
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) odd = fmaf(x[i], 0.0f, odd);
            if (bans) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) x[i] = fmaxf(x[i], 0.0f);
            }
#pragma unroll
            for (int i = 0; i < VPL; ++i) key[i] = (__float_as_uint(x[i]) & ~INDEX) | (INDEX - i);
            if (e0 + VPL > E) {
#pragma unroll
                for (int i = 0; i < VPL; ++i) key[i] = e0 + i < E ? key[i] : 0u;
            }
        }
        // (a group's sum with a banned expert in it is not what these keys add up to)
        bool unsure = __any_sync(0xffffffffu, odd != odd) || (bans && form.n_groups > 1);
        uint32_t best[KEEP];
        if (whole) largest_keys<VPL, KEEP>(key, best);
        if (form.n_groups > 1 && !unsure) {
            float mine = -1.0f;                                                // lane g: group g's score
            if (whole) {
                uint32_t a = best[0] & ~INDEX, c = KEEP > 1 ? best[KEEP > 1] & ~INDEX : 0u;    // the lane's two best, then the group's
                for (int o = 1; o < lanes_per; o <<= 1) {
                    const uint32_t oa = __shfl_xor_sync(0xffffffffu, a, o), oc = __shfl_xor_sync(0xffffffffu, c, o);
                    c = max(min(a, oa), max(c, oc));
                    a = max(a, oa);
                }
                const float score = __uint_as_float(a) + __uint_as_float(c);
                const float of_group = __shfl_sync(0xffffffffu, score, (lane * lanes_per) & 31);
                if (lane < form.n_groups) mine = of_group;
            } else {
                for (int g = 0; g < form.n_groups; ++g) {
                    uint32_t a = 0, c = 0;
#pragma unroll
                    for (int i = 0; i < VPL; ++i) {
                        const uint32_t k = e0 + i >= g * per && e0 + i < (g + 1) * per ? key[i] & ~INDEX : 0u;
                        c = max(c, min(a, k));
                        a = max(a, k);
                    }
                    const uint32_t top = __reduce_max_sync(0xffffffffu, a);
                    const int owner = __ffs(__ballot_sync(0xffffffffu, a == top)) - 1;
                    const uint32_t next = __reduce_max_sync(0xffffffffu, lane == owner ? c : a);
                    if (lane == g) mine = __uint_as_float(top) + __uint_as_float(next);
                }
            }
            const unsigned groups = best_groups(mine, form.n_groups, form.top_groups, lane);
            const bool in = groups >> lane & 1;
            // (positive floats are in order as integers)
            const float worst = __uint_as_float(__reduce_min_sync(0xffffffffu, in ? __float_as_uint(mine) : 0x7f800000u));
            const float next = __uint_as_float(__reduce_max_sync(0xffffffffu, in || lane >= form.n_groups ? 0u : __float_as_uint(mine)));
            if (form.top_groups < form.n_groups && !(worst - next > 2.0f * near + (worst + next) * HIDDEN)) unsure = true;
            if (whole) {
                const bool open = groups >> my_group & 1;
#pragma unroll
                for (int i = 0; i < KEEP; ++i) best[i] = open ? best[i] : 0u;
            } else {
#pragma unroll
                for (int i = 0; i < VPL; ++i)
                    if (e0 + i < E && !(groups >> ((unsigned)(e0 + i) / (unsigned)per) & 1)) key[i] = 0u;
            }
        }
        if (!whole) largest_keys<VPL, KEEP>(key, best);
        int my_expert = 0;
        float my_logit = 0.0f;
        if (!unsure) {
            const bool more = VPL > KEEP && best[KEEP - 1] != 0u;              // (there may be keys that were not kept)
            // the n-th of the list is the best key left (and off it goes); returns it without its last bits, 0: there is none
            auto take = [&](int n) {
                const uint32_t head = best[0] & ~INDEX, top = __reduce_max_sync(0xffffffffu, head);
                const bool equal = head == top;
                const unsigned all = __ballot_sync(0xffffffffu, equal);
                if (equal && !(all & below)) {                                 // of equal keys the lowest lane's: the lower expert
                    s_list[warp][n] = make_uint2(best[0], lane);
#pragma unroll
                    for (int i = 0; i + 1 < KEEP; ++i) best[i] = best[i + 1];
                    best[KEEP - 1] = 0u;
                }
                return top;
            };
            uint32_t top = 0;
            for (int r = 0; r < top_k; ++r) {
                top = take(r);
                if (top == 0u) unsure = true;
            }
            // ... and those behind the last one that are as good as it, as far as these scores can tell
            const float v_last = __uint_as_float(top), wide = near + v_last * HIDDEN;
            int n = top_k;
            for (; n < 32; ++n) {
                const uint32_t next = take(n);
                if (v_last - __uint_as_float(next) > wide) break;
                if (next == 0u) { unsure = unsure || n < E; break; }           // (where all are taken, one of them may have been no key)
            }
            if (n == 32 && top_k < E) unsure = true;                           // (more of them than lanes)
            if (__any_sync(0xffffffffu, more && best[0] == 0u)) unsure = true;
            __syncwarp();
            float v = 0.0f, my_bias = 0.0f;
            if (lane < n) {
                const uint2 chosen = s_list[warp][lane];
                my_expert = min((int)chosen.y * VPL + (int)(INDEX - (chosen.x & INDEX)), E - 1);
                v = __uint_as_float(chosen.x & ~INDEX);
                my_logit = logit<L>(row[my_expert]);
                my_bias = bias ? bias[my_expert] : 0.0f;
            }
            // sure of the order: every gap is wide, or the two are equal in logit and bias (the lower expert came first)
            const float v_next = __shfl_down_sync(0xffffffffu, v, 1);
            const float l_next = __shfl_down_sync(0xffffffffu, my_logit, 1), b_next = __shfl_down_sync(0xffffffffu, my_bias, 1);
            const bool same = my_logit == l_next && my_bias == b_next, gap = v - v_next > near + v * HIDDEN;
            if (!unsure && !__all_sync(0xffffffffu, lane >= n - 1 || gap || same)) {
                if (SOFTMAX && bias) {
                    unsure = true;
                } else {
                    my_expert = rank_exact<SOFTMAX>(my_expert, my_logit, my_bias, m, n);
                    if (lane < top_k) my_logit = logit<L>(row[my_expert]);
                }
            }
            __syncwarp();
        }
        if (unsure) {
            my_expert = route_exact<VPL, L, SOFTMAX>(row, bias, E, top_k, form.n_groups, form.top_groups);
            if (lane < top_k) my_logit = logit<L>(row[my_expert]);
        }
        float score = 0.0f;
        if (lane < top_k) score = SOFTMAX ? __fdiv_rn(expf(my_logit - m), sum) : __fdiv_rn(1.0f, 1.0f + expf(-my_logit));
        const float total = warp_sum(score) + 1e-9f;
        if (lane < top_k) {
            top_experts[(int64_t)t * top_k + lane] = my_expert;
            top_gates[(int64_t)t * top_k + lane] = (form.renormalise ? __fdiv_rn(score, total) : score) * form.scale;
            atomicAdd(&s_hist[my_expert], 1);
        }
    }
    __syncthreads();
    for (int e = threadIdx.x; e < E; e += 256) hist[(int64_t)blockIdx.x * E + e] = s_hist[e];
}

// d logits of the gates, from their gradients by slot (d_top), in the order of pair_pos (d_pair) and by sorted pair (d_sorted); null: none.  One warp per
// token; d score of a chosen expert is scale * d gate, or with renormalised gates scale * (d gate - sum_j d gate_j s_j / S) / S, S = sum of
// the chosen s + 1e-9; then s (1 - s) d, or for a softmax s_e (d_e - sum_j d_j s_j).  Two of these differences cancel, wholly so for a single
// chosen expert, whose gate is 1 - 1e-9 / S whatever its score; they are taken as what is left: (sum_j s_j (d gate - d gate_j) + 1e-9 d gate) / S^2,
// and 1e-9 sum_j d gate_j s_j / S^2.  Bound by reading and writing the logits.
template <int VPL, typename L, bool SOFTMAX>
__global__ void __launch_bounds__(256)
route_form_backward_kernel(const L* __restrict__ logits, const int* __restrict__ top_experts, const int64_t* __restrict__ sorted_experts,
                           const int64_t* __restrict__ pair_pos, const float* __restrict__ d_top, const float* __restrict__ d_pair,
                           const float* __restrict__ d_sorted, const RouteForm form,
                           L* __restrict__ d_logits, int64_t T, int E, int top_k) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, e0 = lane * VPL;
    for (int64_t t = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); t < T; t += (int64_t)gridDim.x * 8) {
        const L* row = logits + t * E;
        float x[VPL], m = 0.0f, inv = 1.0f;
        if constexpr (SOFTMAX) {
            m = -INFINITY;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                x[i] = e0 + i < E ? logit<L>(row[e0 + i]) : -INFINITY;
                m = fmaxf(m, x[i]);
            }
            m = warp_max(m);
            float part = 0.0f;
#pragma unroll
            for (int i = 0; i < VPL; ++i) {
                x[i] = e0 + i < E ? expf(x[i] - m) : 0.0f;
                part += x[i];
            }
            inv = __fdiv_rn(1.0f, warp_sum(part));
        }
        int mine = -1;
        float s = 0.0f, g = 0.0f;
        if (lane < top_k) {
            mine = top_experts[t * top_k + lane];
            if ((unsigned)mine < (unsigned)E) {
                const float v = logit<L>(row[mine]);
                s = SOFTMAX ? expf(v - m) * inv : __fdiv_rn(1.0f, 1.0f + expf(-v));
                if (d_top) g = d_top[t * top_k + lane];
            } else {
                mine = -1;                                                     // (not what the forward wrote: no part in anything)
            }
        }
        if (d_pair || d_sorted) {                                              // lane j: the token's j-th pair, its expert and its gradient
            int e = -2;
            float h = 0.0f;
            if (lane < top_k) {
                const int64_t at = pair_pos[t * top_k + lane];
                if (at >= 0 && at < T * top_k) {
                    const int64_t chosen = sorted_experts[at];
                    if (chosen >= 0 && chosen < E) e = (int)chosen;
                    if (d_pair) h = d_pair[t * top_k + lane];
                    if (d_sorted) h += d_sorted[at];
                }
            }
            for (int j = 0; j < top_k; ++j) {
                const int ej = __shfl_sync(0xffffffffu, e, j);
                const float hj = __shfl_sync(0xffffffffu, h, j);
                if (ej == mine) g += hj;
            }
        }
        g *= form.scale;
        float common = 0.0f;
        if (form.renormalise) {
            const float total = warp_sum(s) + 1e-9f;
            if (SOFTMAX) common = 1e-9f * warp_sum(g * s) / total / total;
            float d = 1e-9f * g;
            for (int j = 0; j < top_k; ++j) d = fmaf(__shfl_sync(0xffffffffu, s, j), g - __shfl_sync(0xffffffffu, g, j), d);
            g = lane < top_k ? d / total / total : 0.0f;
        } else if (SOFTMAX) {
            common = warp_sum(g * s);
        }
        float d = s * (1.0f - s) * g;
        float out[VPL];
#pragma unroll
        for (int i = 0; i < VPL; ++i) out[i] = SOFTMAX ? -(x[i] * inv) * common : 0.0f;
        if constexpr (SOFTMAX) d = s * (g - common);
        for (int j = 0; j < top_k; ++j) {
            const int e = __shfl_sync(0xffffffffu, mine, j) - e0;
            const float v = __shfl_sync(0xffffffffu, d, j);
#pragma unroll
            for (int i = 0; i < VPL; ++i)
                if (e == i) out[i] = v;
        }
#pragma unroll
        for (int i = 0; i < VPL; ++i)
            if (e0 + i < E) d_logits[t * E + e0 + i] = from_float<L>(out[i]);
    }
}

__global__ void __launch_bounds__(256)
route_scan_kernel(int* __restrict__ hist, int n_ctas, int E, int* __restrict__ totals) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, e = blockIdx.x * 8 + (threadIdx.x >> 5);
    if (e >= E) return;
    int carry = 0;
    for (int b0 = 0; b0 < n_ctas; b0 += 128) {               // four histograms per lane in flight
        int v[4];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int b = b0 + u * 32 + lane;
            v[u] = b < n_ctas ? hist[(int64_t)b * E + e] : 0;
        }
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int b = b0 + u * 32 + lane;
            int incl = v[u];
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int x = __shfl_up_sync(0xffffffffu, incl, o);
                if (lane >= o) incl += x;
            }
            if (b < n_ctas) hist[(int64_t)b * E + e] = carry + incl - v[u];
            carry += __shfl_sync(0xffffffffu, incl, 31);
        }
    }
    if (lane == 0) totals[e] = carry;
}

// The same where there is much of it: a CTA takes 32 experts, a lane each, and a warp a 32nd of the histograms: their sums, where each warp begins,
// then the running sums.  A warp for each expert reads 32 lines with every load: routing 32768 tokens to 256 experts 97 us so, 85 like this;
// to 16 experts 23 and 30, 8192 tokens to 64 21 and 23 (a CTA or two do all of it).  From 2^16 counts on.
__global__ void __launch_bounds__(1024)
route_scan_wide_kernel(int* __restrict__ hist, int n_ctas, int E, int* __restrict__ totals) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_sum[32][33];
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, e = blockIdx.x * 32 + lane;
    const int first = (int)((int64_t)n_ctas * warp / 32), last = (int)((int64_t)n_ctas * (warp + 1) / 32);
    int sum = 0;
    if (e < E) {
#pragma unroll 8
        for (int b = first; b < last; ++b) sum += hist[(int64_t)b * E + e];
    }
    s_sum[warp][lane] = sum;
    __syncthreads();
    int carry = 0, all = 0;
#pragma unroll
    for (int w = 0; w < 32; ++w) {
        const int v = s_sum[w][lane];
        carry += w < warp ? v : 0;
        all += v;
    }
    if (e >= E) return;
    for (int b0 = first; b0 < last; b0 += 8) {               // eight histograms in flight
        int v[8];
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] = b0 + u < last ? hist[(int64_t)(b0 + u) * E + e] : 0;
#pragma unroll
        for (int u = 0; u < 8; ++u) {
            if (b0 + u < last) hist[(int64_t)(b0 + u) * E + e] = carry;
            carry += v[u];
        }
    }
    if (warp == 0) totals[e] = all;
}

// totals: per-expert counts from route_scan_kernel, with `hist` turned into offsets; null: hist still holds counts
__global__ void __launch_bounds__(256)
route_scatter_kernel(const int* __restrict__ top_experts, const float* __restrict__ top_gates, const int* __restrict__ hist,
                     const int* __restrict__ totals, int T, int E, int top_k, int tokens_per_cta, int64_t* __restrict__ token_indices,
                     float* __restrict__ sorted_scores, int64_t* __restrict__ sorted_experts, int64_t* __restrict__ counts,
                     int64_t* __restrict__ starts, int64_t* __restrict__ ends, int64_t* __restrict__ pair_pos,
                     float* __restrict__ pair_gate) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_next[ROUTE_MAX_EXPERTS];                                  // next free row of every expert
    __shared__ unsigned long long s_warps[ROUTE_MAX_EXPERTS];                  // of 256 pairs: how many of each warp are the expert's, a byte each
    __shared__ int s_warp[8];
    __shared__ int s_pos[ROUTE_MAX_TOKENS_PER_CTA * ROUTE_MAX_TOPK];
    for (int e = threadIdx.x; e < E; e += 256) s_warps[e] = 0ull;
    {
        // thread i: experts 4 i .. 4 i + 3; their counts, the rows of earlier CTAs, and a scan of the counts
        int cnt[4], mine[4], sum = 0;
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = threadIdx.x * 4 + u;
            cnt[u] = 0; mine[u] = 0;
            if (e < E) {
                if (totals) {
                    cnt[u] = totals[e];
                    mine[u] = hist[(int64_t)blockIdx.x * E + e];
                } else {
                    for (int b = 0; b < (int)gridDim.x; ++b) {
                        const int v = hist[(int64_t)b * E + e];
                        if (b < (int)blockIdx.x) mine[u] += v;
                        cnt[u] += v;
                    }
                }
            }
            sum += cnt[u];
        }
        const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
        int incl = sum;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += x;
        }
        if (lane == 31) s_warp[warp] = incl;
        __syncthreads();
        int first = incl - sum;
        for (int w = 0; w < warp; ++w) first += s_warp[w];
#pragma unroll
        for (int u = 0; u < 4; ++u) {
            const int e = threadIdx.x * 4 + u;
            if (e < E) {
                s_next[e] = first + mine[u];
                if (blockIdx.x == 0) {
                    counts[e] = cnt[u];
                    if (starts) { starts[e] = first; ends[e] = first + cnt[u]; }
                }
                first += cnt[u];
            }
        }
    }
    __syncthreads();
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int t_begin = blockIdx.x * tokens_per_cta;
    const int n_tok = min(tokens_per_cta, T - t_begin);
    const int n_pairs = n_tok * top_k;
    const int64_t pair0 = (int64_t)t_begin * top_k;
    // A pair's row: the expert's next free one, behind those of lower warps and lower lanes that are the same expert's.  (Warp after warp, with a
    // barrier between them: eight turns instead of three barriers.)
    for (int base = 0; base < n_pairs; base += 256) {
        const int p = base + threadIdx.x;
        const bool live = p < n_pairs;
        const int e = live ? top_experts[pair0 + p] : -1 - lane;              // dead lanes match nobody
        const unsigned peers = __match_any_sync(0xffffffffu, e);
        const bool leads = live && lane == __ffs(peers) - 1;
        if (leads) atomicAdd(&s_warps[e], (unsigned long long)__popc(peers) << (8 * warp));
        __syncthreads();
        int row = 0, all = 0;
        bool first = false;
        if (live) {
            const unsigned long long counts_of = s_warps[e], lower = counts_of & ((1ull << (8 * warp)) - 1ull);
            const auto bytes = [](unsigned long long v) { return __dp4a((unsigned)v, 0x01010101u, __dp4a((unsigned)(v >> 32), 0x01010101u, 0u)); };
            row = s_next[e] + (int)bytes(lower) + __popc(peers & ((1u << lane) - 1u));
            all = (int)bytes(counts_of);
            first = leads && lower == 0ull;
            s_pos[p] = row;
            token_indices[row] = t_begin + p / top_k;
            sorted_scores[row] = top_gates[pair0 + p];
            sorted_experts[row] = e;
        }
        __syncthreads();
        if (first) { s_next[e] += all; s_warps[e] = 0ull; }
        __syncthreads();
    }
    // per token: its rows in ascending order, gates alongside; a pair's place is how many of its token's rows come before its own
    for (int p = threadIdx.x; p < n_pairs; p += 256) {
        const int tl = p / top_k, mine = s_pos[p];
        int place = 0;
        for (int j = 0; j < top_k; ++j) place += s_pos[tl * top_k + j] < mine;
        pair_pos[pair0 + tl * top_k + place] = mine;
        pair_gate[pair0 + tl * top_k + place] = top_gates[pair0 + p];
    }
}

// Tokens per CTA of the other forms: CTAs of 256 threads that are all resident at once (five per SM up to 256 experts, two beyond), so that none
// waits for a second turn; full turns of them for more tokens.
static inline int form_tokens_per_cta(int64_t T, int E) {
    const int64_t slots = (E <= 256 ? 5 : 2) * (int64_t)sm_count();
    const int64_t turns = (T + slots * ROUTE_MAX_TOKENS_PER_CTA - 1) / (slots * ROUTE_MAX_TOKENS_PER_CTA);
    const int64_t ctas = slots * (turns < 1 ? 1 : turns), per = ((T + ctas - 1) / ctas + 7) / 8 * 8;
    return (int)(per < 8 ? 8 : per);
}
int64_t moe_route_form_workspace_ints(int64_t T, int E) {
    const int per = form_tokens_per_cta(T, E);
    return ((T + per - 1) / per) * (int64_t)E + E;
}

int64_t moe_route_workspace_ints(int64_t T, int E) {
    const int per = route_tokens_per_cta(T, E);
    return ((T + per - 1) / per) * (int64_t)E + E;
}

template <typename L>
static void launch_topk(const L* logits, const float* bias, int T, int E, int top_k, int per, int n_ctas, int* top_experts,
                        float* top_gates, int* hist, cudaStream_t st) {
#define CINN_TOPK(V) launch_dependent(route_topk_kernel<V, L>, dim3(n_ctas), dim3(256), 0, st, logits, bias, T, E, top_k, per, top_experts, top_gates, hist)
    if (E <= 32) CINN_TOPK(1);
    else if (E <= 64) CINN_TOPK(2);
    else if (E <= 128) CINN_TOPK(4);
    else if (E <= 256) CINN_TOPK(8);
    else if (E <= 512) CINN_TOPK(16);
    else CINN_TOPK(32);
#undef CINN_TOPK
}

#define CINN_FORM_VPL(CALL) \
    do { if (E <= 32) { CALL(1); } else if (E <= 64) { CALL(2); } else if (E <= 128) { CALL(4); } else if (E <= 256) { CALL(8); } \
         else if (E <= 512) { CALL(16); } else { CALL(32); } } while (0)

template <typename L>
static void launch_form(const L* logits, const float* bias, int T, int E, int top_k, const RouteForm& form, bool softmax, int per, int n_ctas,
                        int* top_experts, float* top_gates, int* hist, cudaStream_t st) {
    const bool aligned = (reinterpret_cast<uintptr_t>(logits) & 15) == 0;
#define CINN_CALL(V) \
    const int vec = aligned && E % V == 0; \
    if (softmax) launch_dependent(route_form_kernel<V, L, true>, dim3(n_ctas), dim3(256), 0, st, logits, bias, T, E, top_k, form, per, vec, top_experts, top_gates, hist); \
    else launch_dependent(route_form_kernel<V, L, false>, dim3(n_ctas), dim3(256), 0, st, logits, bias, T, E, top_k, form, per, vec, top_experts, top_gates, hist)
    CINN_FORM_VPL(CINN_CALL);
#undef CINN_CALL
}

template <typename L>
static void launch_form_backward(const L* logits, const int* top, const int64_t* se, const int64_t* pos, const float* d_top, const float* d_pair,
                                 const float* d_sorted, const RouteForm& form, bool softmax, L* out, int64_t T, int E, int top_k, cudaStream_t st) {
    const int64_t want = (T + 7) / 8, cap = (int64_t)sm_count() * 16;
    const unsigned grid = (unsigned)(want < cap ? want : cap);
#define CINN_CALL(V) \
    if (softmax) launch_dependent(route_form_backward_kernel<V, L, true>, dim3(grid), dim3(256), 0, st, logits, top, se, pos, d_top, d_pair, d_sorted, form, out, T, E, top_k); \
    else launch_dependent(route_form_backward_kernel<V, L, false>, dim3(grid), dim3(256), 0, st, logits, top, se, pos, d_top, d_pair, d_sorted, form, out, T, E, top_k)
    CINN_FORM_VPL(CINN_CALL);
#undef CINN_CALL
}

static int check_form(int scores, int n_groups, int top_groups, int E, int top_k) {
    CINN_CHECK_ARG(scores == 0 || scores == 1, "moe_route: scores %d (0 sigmoid, 1 softmax)", scores);
    CINN_CHECK_ARG(n_groups >= 1 && n_groups <= ROUTE_MAX_GROUPS && E % n_groups == 0, "moe_route: %d experts in %d groups (1 to %d groups of equally many)",
                   E, n_groups, ROUTE_MAX_GROUPS);
    CINN_CHECK_ARG(top_groups >= 1 && top_groups <= n_groups && top_k <= top_groups * (E / n_groups),
                   "moe_route: %d experts out of %d of %d groups of %d", top_k, top_groups, n_groups, E / n_groups);
    return CINN_OK;
}

// logits_dtype: CINN_F32, or a 16-bit type that is widened on load.  starts / ends (E each): null, or every expert's rows.  form: null, or what
// the scores and gates are (with a bias that may be null then).
static int moe_route(const void* logits, int logits_dtype, const float* bias, int64_t T, int E, int top_k, int* workspace, int* top_experts,
              float* top_gates, int64_t* token_indices, float* sorted_scores, int64_t* sorted_experts, int64_t* counts,
              int64_t* starts, int64_t* ends, int64_t* pair_pos, float* pair_gate, cudaStream_t st, const RouteForm* form, bool softmax) {
    CINN_CHECK_ARG(T >= 0 && E >= 1 && E <= ROUTE_MAX_EXPERTS, "moe_route: 1 <= E <= %d experts (got %d)", ROUTE_MAX_EXPERTS, E);
    CINN_CHECK_ARG(top_k >= 1 && top_k <= ROUTE_MAX_TOPK && top_k <= E, "moe_route: 1 <= top_k <= min(E, %d) (got %d)",
                   ROUTE_MAX_TOPK, top_k);
    CINN_CHECK_ARG(T * (int64_t)top_k < (1LL << 31), "moe_route: too many (token, expert) pairs");
    CINN_CHECK_ARG(counts != nullptr && (starts == nullptr) == (ends == nullptr), "moe_route: null pointer");
    CINN_CHECK_ARG(logits_dtype == CINN_F32 || logits_dtype == CINN_BF16 || logits_dtype == CINN_F16, "moe_route: unknown dtype tag %d",
                   logits_dtype);
    if (T == 0) {
        CINN_CHECK_CUDA(cudaMemsetAsync(counts, 0, sizeof(int64_t) * E, st));
        if (starts) {
            CINN_CHECK_CUDA(cudaMemsetAsync(starts, 0, sizeof(int64_t) * E, st));
            CINN_CHECK_CUDA(cudaMemsetAsync(ends, 0, sizeof(int64_t) * E, st));
        }
        return CINN_OK;
    }
    CINN_CHECK_ARG(logits && (bias || form) && workspace && top_experts && top_gates && token_indices && sorted_scores &&
                   sorted_experts && pair_pos && pair_gate, "moe_route: null pointer");
    const int per = form ? form_tokens_per_cta(T, E) : route_tokens_per_cta(T, E), n_ctas = (int)((T + per - 1) / per);
    int* hist = workspace;
    int* totals = n_ctas > ROUTE_FEW_CTAS ? workspace + (int64_t)n_ctas * E : nullptr;
    if (form) {
        if (logits_dtype == CINN_F32) launch_form((const float*)logits, bias, (int)T, E, top_k, *form, softmax, per, n_ctas, top_experts, top_gates, hist, st);
        else if (logits_dtype == CINN_BF16) launch_form((const __nv_bfloat16*)logits, bias, (int)T, E, top_k, *form, softmax, per, n_ctas, top_experts, top_gates, hist, st);
        else launch_form((const __half*)logits, bias, (int)T, E, top_k, *form, softmax, per, n_ctas, top_experts, top_gates, hist, st);
    } else if (logits_dtype == CINN_F32) launch_topk((const float*)logits, bias, (int)T, E, top_k, per, n_ctas, top_experts, top_gates, hist, st);
    else if (logits_dtype == CINN_BF16) launch_topk((const __nv_bfloat16*)logits, bias, (int)T, E, top_k, per, n_ctas, top_experts, top_gates, hist, st);
    else launch_topk((const __half*)logits, bias, (int)T, E, top_k, per, n_ctas, top_experts, top_gates, hist, st);
    CINN_CHECK_LAUNCH();
    if (totals) {
        if ((int64_t)n_ctas * E > 1 << 16) launch_dependent(route_scan_wide_kernel, dim3((E + 31) / 32), dim3(1024), 0, st, hist, n_ctas, E, totals);
        else launch_dependent(route_scan_kernel, dim3((E + 7) / 8), dim3(256), 0, st, hist, n_ctas, E, totals);
        CINN_CHECK_LAUNCH();
    }
    launch_dependent(route_scatter_kernel, dim3(n_ctas), dim3(256), 0, st, top_experts, top_gates, hist, totals, (int)T, E, top_k, per, token_indices, sorted_scores,
                                                 sorted_experts, counts, starts, ends, pair_pos, pair_gate);
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

int moe_route(const void* logits, int logits_dtype, const float* bias, int64_t T, int E, int top_k, int* workspace, int* top_experts,
              float* top_gates, int64_t* token_indices, float* sorted_scores, int64_t* sorted_experts, int64_t* counts,
              int64_t* starts, int64_t* ends, int64_t* pair_pos, float* pair_gate, cudaStream_t st) {
    return moe_route(logits, logits_dtype, bias, T, E, top_k, workspace, top_experts, top_gates, token_indices, sorted_scores, sorted_experts, counts,
                     starts, ends, pair_pos, pair_gate, st, nullptr, false);
}

int moe_route_form(const void* logits, int logits_dtype, const float* bias, int64_t T, int E, int top_k, int scores, int n_groups, int top_groups,
                   int renormalise, float scale, int* workspace, int* top_experts, float* top_gates, int64_t* token_indices, float* sorted_scores,
                   int64_t* sorted_experts, int64_t* counts, int64_t* starts, int64_t* ends, int64_t* pair_pos, float* pair_gate, cudaStream_t st) {
    CINN_CHECK_ARG(E >= 1, "moe_route: no experts");
    int rc = check_form(scores, n_groups, top_groups, E, top_k);
    if (rc) return rc;
    const RouteForm form{n_groups, top_groups, renormalise != 0, scale};
    return moe_route(logits, logits_dtype, bias, T, E, top_k, workspace, top_experts, top_gates, token_indices, sorted_scores, sorted_experts, counts,
                     starts, ends, pair_pos, pair_gate, st, &form, scores == 1);
}

int moe_route_form_backward(const void* logits, int logits_dtype, const int* top_experts, const int64_t* sorted_experts, const int64_t* pair_pos,
                            const float* d_top, const float* d_pair, const float* d_sorted, int64_t T, int E, int top_k, int scores, int renormalise, float scale,
                            void* d_logits, cudaStream_t st) {
    CINN_CHECK_ARG(T >= 0 && E >= 1 && E <= ROUTE_MAX_EXPERTS && top_k >= 1 && top_k <= ROUTE_MAX_TOPK && top_k <= E && (scores == 0 || scores == 1),
                   "moe_route backward: bad shape");
    CINN_CHECK_ARG(logits_dtype == CINN_F32 || logits_dtype == CINN_BF16 || logits_dtype == CINN_F16, "moe_route: unknown dtype tag %d", logits_dtype);
    if (T == 0) return CINN_OK;
    CINN_CHECK_ARG(logits && top_experts && d_logits && ((!d_pair && !d_sorted) || (sorted_experts && pair_pos)), "moe_route backward: null pointer");
    const RouteForm form{1, 1, renormalise != 0, scale};
    if (logits_dtype == CINN_F32) launch_form_backward((const float*)logits, top_experts, sorted_experts, pair_pos, d_top, d_pair, d_sorted, form, scores == 1, (float*)d_logits, T, E, top_k, st);
    else if (logits_dtype == CINN_BF16) launch_form_backward((const __nv_bfloat16*)logits, top_experts, sorted_experts, pair_pos, d_top, d_pair, d_sorted, form, scores == 1, (__nv_bfloat16*)d_logits, T, E, top_k, st);
    else launch_form_backward((const __half*)logits, top_experts, sorted_experts, pair_pos, d_top, d_pair, d_sorted, form, scores == 1, (__half*)d_logits, T, E, top_k, st);
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

// ---------------------------------------------------------------------------
// The same routing for callers that cannot hand over a workspace.  The scratch lives in a fixed array inside
// the library image: every GPU that loads the library holds these 2 MiB until the process exits.  All calls on
// a device share it, so two calls that overlap on that GPU (different streams, different threads) race; the
// routing kernels overwrite every word they later read, so nothing has to be cleared between calls.
// ---------------------------------------------------------------------------
static __device__ __align__(256) int g_route_scratch[ROUTE_STATIC_MAX_INTS];

constexpr int ROUTE_MAX_DEVICES = 64;
static std::mutex g_route_scratch_mutex;
static int* g_route_scratch_ptr[ROUTE_MAX_DEVICES] = {};               // device address of the array, per device

// In host code `g_route_scratch` is only a handle for the symbol, not an address a kernel can use; the device
// address is asked for once per device, with that device current.
static int route_scratch_address(int** out) {
    int dev = -1;
    CINN_CHECK_CUDA(cudaGetDevice(&dev));
    CINN_CHECK_ARG(dev >= 0 && dev < ROUTE_MAX_DEVICES, "moe_route_static: device ordinal %d is beyond %d", dev,
                   ROUTE_MAX_DEVICES);
    std::lock_guard<std::mutex> lock(g_route_scratch_mutex);
    if (g_route_scratch_ptr[dev] == nullptr) {
        void* p = nullptr;
        CINN_CHECK_CUDA(cudaGetSymbolAddress(&p, g_route_scratch));
        g_route_scratch_ptr[dev] = static_cast<int*>(p);
    }
    *out = g_route_scratch_ptr[dev];
    return CINN_OK;
}

int64_t moe_route_static_max_ints() { return ROUTE_STATIC_MAX_INTS; }

int moe_route_static(const float* logits, const float* bias, int64_t T, int E, int top_k, int* top_experts, float* top_gates,
                     int64_t* token_indices, float* sorted_scores, int64_t* sorted_experts, int64_t* counts,
                     int64_t* pair_pos, float* pair_gate, cudaStream_t st) {
    CINN_CHECK_ARG(T >= 0 && E >= 1 && E <= ROUTE_MAX_EXPERTS, "moe_route_static: 1 <= E <= %d experts (got %d)",
                   ROUTE_MAX_EXPERTS, E);
    const int64_t need = moe_route_workspace_ints(T, E);
    CINN_CHECK_ARG(need <= ROUTE_STATIC_MAX_INTS,
                   "moe_route_static: %lld tokens x %d experts need %lld ints of scratch, the built-in array holds %lld; "
                   "use cinn_moe_route with a workspace of your own",
                   (long long)T, E, (long long)need, (long long)ROUTE_STATIC_MAX_INTS);
    int* scratch = nullptr;
    int rc = route_scratch_address(&scratch);
    if (rc) return rc;
    return moe_route(logits, CINN_F32, bias, T, E, top_k, scratch, top_experts, top_gates, token_indices, sorted_scores,
                     sorted_experts, counts, nullptr, nullptr, pair_pos, pair_gate, st);
}

}  // namespace cinn
