// Rotary positions: pairs of a head's elements turned by position x frequency, for queries and keys in one launch.
//
//   (a, b) -> m (a cos t - b sin t, b cos t + a sin t),  t = position * frequency[i] (the inverse: -t)
//
// Pairs are neighbours (interleaved) or half of the rotated part apart; the rest of the head is copied (or, in place, left alone).
//
// The angle of a far position loses its bits in fp32 (at 10^6 radians a step is 0.06) and a table of cosines has a length.  Here a
// frequency is a fraction of a turn in 64 bits and position x frequency a 64-bit product: what overflows is whole turns, so
// the angle is exact to 2^-53 of the frequency times the position.  The top two bits (rounded) are the quadrant, and the rest,
// within an eighth of a turn, goes to sincospif in fp32.
//
// Bound by memory: every element is read and written once, 16 bytes a thread.  A CTA takes a few tokens and some of their heads; it
// works out the tokens' cosines and sines once, in shared memory, for all of its heads.
#include "common.cuh"
#include <algorithm>

namespace cinn {
namespace rope {

constexpr int THREADS = 256;
constexpr int MAX_ANGLES = 2048;           // of a CTA's tokens; also the most pairs of a head

struct Side {                              // queries or keys
    const void* in;
    void* out;
    int64_t in_b, in_h, in_l, out_b, out_h, out_l;
    int heads, d, start;                   // elements of a head; where the rotated part starts
    int head_chunks, heads_per_chunk;      // the CTAs of a token tile share its heads
};
struct Params {
    Side side[2];
    int64_t blocks0;                       // CTAs of side 0
    int64_t tokens;
    int L, tile;                           // positions of a sequence; tokens of a CTA
    const int64_t* positions;
    int64_t pos_b, pos_l;
    const double* freq;                    // radians a position
    int pairs;
    float magnitude, sign;
    int copy_rest;                         // 0: in place, the rest of a head is left alone
};

template <typename T> __device__ __forceinline__ float widen(T v);
template <> __device__ __forceinline__ float widen<float>(float v) { return v; }
template <> __device__ __forceinline__ float widen<__nv_bfloat16>(__nv_bfloat16 v) { return __bfloat162float(v); }
template <> __device__ __forceinline__ float widen<__half>(__half v) { return __half2float(v); }
template <typename T> __device__ __forceinline__ T narrow(float v);
template <> __device__ __forceinline__ float narrow<float>(float v) { return v; }
template <> __device__ __forceinline__ __nv_bfloat16 narrow<__nv_bfloat16>(float v) { return __float2bfloat16_rn(v); }
template <> __device__ __forceinline__ __half narrow<__half>(float v) { return __float2half_rn(v); }

template <typename T, int VEC> struct alignas(sizeof(T) * VEC) Piece { T v[VEC]; };

// cosine and sine of position * freq radians
__device__ __forceinline__ float2 turn_of(int64_t position, double freq) {
    double turns = freq * 0.15915494309189533577;
    turns -= floor(turns);
    const uint64_t unit = __double2ull_rn(turns * 18446744073709551616.0);           // 2^64 (a whole turn saturates: off by 2^-64)
    const uint64_t at = unit * (uint64_t)position;
    const uint64_t quadrant = (at + (1ull << 61)) >> 62;
    const float rest = (float)(int64_t)(at - (quadrant << 62)) * 0x1p-63f;           // half turns, within a quarter
    float s, c;
    sincospif(rest, &s, &c);
    if (quadrant & 1) { const float t = c; c = -s; s = t; }
    if (quadrant & 2) { c = -c; s = -s; }
    return make_float2(c, s);
}

// VEC: elements a thread moves at a time (16 bytes, or one where the layout does not allow it)
template <typename T, int VEC, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS)
rotary_kernel(const Params p) {
    pdl_wait();
    pdl_trigger();
    __shared__ float2 s_turn[MAX_ANGLES];
    const bool second = blockIdx.x >= p.blocks0;
    const Side& sd = p.side[second];
    const int64_t block = blockIdx.x - (second ? p.blocks0 : 0);
    const int64_t tile = block / sd.head_chunks;
    const int chunk = (int)(block - tile * sd.head_chunks);
    const int64_t t0 = tile * p.tile;
    const int n_tok = (int)min((int64_t)p.tile, p.tokens - t0);
    const int h0 = chunk * sd.heads_per_chunk, n_heads = min(sd.heads_per_chunk, sd.heads - h0);
    for (int i = threadIdx.x; i < n_tok * p.pairs; i += THREADS) {
        const int t = i / p.pairs, f = i - t * p.pairs;
        const int64_t tok = t0 + t, b = tok / p.L, l = tok - b * p.L;
        float2 cs = turn_of(p.positions[b * p.pos_b + l * p.pos_l], p.freq[f]);
        s_turn[i] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude * p.sign);
    }
    __syncthreads();
    using V = Piece<T, VEC>;
    constexpr int UNIT = VEC > 1 ? VEC : 2;                               // of neighbours: whole pairs
    const int rest = p.copy_rest ? (sd.d - 2 * p.pairs) / VEC : 0;        // pieces that are copied
    const int turned = INTERLEAVED ? 2 * p.pairs / UNIT : p.pairs / VEC;   // units that are rotated
    const int units = rest + turned;
    const int wide = min(units, THREADS), rows = THREADS / wide;          // threads of a row, rows at a time
    const int r0 = threadIdx.x / wide, u0 = threadIdx.x - r0 * wide;
    if (r0 >= rows) return;
    const int step_t = rows / n_heads, step_h = rows - step_t * n_heads;
    int t = r0 / n_heads, h = r0 - t * n_heads;
    while (t < n_tok) {
        const int64_t tok = t0 + t, b = tok / p.L, l = tok - b * p.L;
        const T* in = static_cast<const T*>(sd.in) + b * sd.in_b + (h0 + h) * sd.in_h + l * sd.in_l;
        T* out = static_cast<T*>(sd.out) + b * sd.out_b + (h0 + h) * sd.out_h + l * sd.out_l;
        const float2* turn = s_turn + t * p.pairs;
        for (int u = u0; u < units; u += wide) {
            if (u < rest) {
                int at = u * VEC;
                if (at >= sd.start) at += 2 * p.pairs;                   // (the rotated part lies in between)
                *reinterpret_cast<V*>(out + at) = *reinterpret_cast<const V*>(in + at);
            } else if constexpr (INTERLEAVED) {
                const int at = (u - rest) * UNIT;
                Piece<T, UNIT> x;
#pragma unroll
                for (int j = 0; j < UNIT; j += VEC) *reinterpret_cast<V*>(x.v + j) = *reinterpret_cast<const V*>(in + sd.start + at + j);
#pragma unroll
                for (int j = 0; j < UNIT; j += 2) {
                    const float2 cs = turn[(at + j) >> 1];
                    const float a = widen<T>(x.v[j]), c = widen<T>(x.v[j + 1]);
                    x.v[j] = narrow<T>(fmaf(a, cs.x, -c * cs.y));
                    x.v[j + 1] = narrow<T>(fmaf(c, cs.x, a * cs.y));
                }
#pragma unroll
                for (int j = 0; j < UNIT; j += VEC) *reinterpret_cast<V*>(out + sd.start + at + j) = *reinterpret_cast<const V*>(x.v + j);
            } else {
                const int at = (u - rest) * VEC;
                V x = *reinterpret_cast<const V*>(in + sd.start + at), y = *reinterpret_cast<const V*>(in + sd.start + p.pairs + at);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float2 cs = turn[at + j];
                    const float a = widen<T>(x.v[j]), c = widen<T>(y.v[j]);
                    x.v[j] = narrow<T>(fmaf(a, cs.x, -c * cs.y));
                    y.v[j] = narrow<T>(fmaf(c, cs.x, a * cs.y));
                }
                *reinterpret_cast<V*>(out + sd.start + at) = x;
                *reinterpret_cast<V*>(out + sd.start + p.pairs + at) = y;
            }
        }
        t += step_t;
        h += step_h;
        if (h >= n_heads) { h -= n_heads; ++t; }
    }
}

template <typename T>
static void launch(bool vec, bool interleaved, const Params& p, unsigned blocks, cudaStream_t st) {
    constexpr int W = 16 / (int)sizeof(T);
    if (vec && interleaved) launch_dependent(rotary_kernel<T, W, true>, dim3(blocks), dim3(THREADS), 0, st, p);
    else if (vec) launch_dependent(rotary_kernel<T, W, false>, dim3(blocks), dim3(THREADS), 0, st, p);
    else if (interleaved) launch_dependent(rotary_kernel<T, 1, true>, dim3(blocks), dim3(THREADS), 0, st, p);
    else launch_dependent(rotary_kernel<T, 1, false>, dim3(blocks), dim3(THREADS), 0, st, p);
}

}  // namespace rope

// in / out: q and k (k's null: q alone), each (B, heads, L, d) with strides {batch, head, position} in elements, the elements of a head
// contiguous; in and out of a side may be the same memory.
int rotary(const void* const* in, void* const* out, const int64_t* in_strides, const int64_t* out_strides, const int64_t* heads, const int64_t* d,
           const int64_t* start, int dtype, int64_t B, int64_t L, const int64_t* positions, int64_t pos_b, int64_t pos_l, const double* freq, int64_t pairs,
           int interleaved, int inverse, float magnitude, cudaStream_t st) {
    using namespace rope;
    CINN_CHECK_ARG(in && out && in_strides && out_strides && heads && d && start, "rotary: null pointer");
    CINN_CHECK_ARG(dtype == CINN_BF16 || dtype == CINN_F16 || dtype == CINN_F32, "rotary: unknown dtype tag %d", dtype);
    CINN_CHECK_ARG(B >= 0 && L >= 0 && B < (1LL << 31) && L < (1LL << 31) && heads[0] >= 0 && heads[1] >= 0 && heads[0] < (1 << 30) && heads[1] < (1 << 30),
                   "rotary: bad shape");
    CINN_CHECK_ARG(pairs >= 1 && pairs <= MAX_ANGLES, "rotary: 1 to %d pairs of a head are rotated (got %lld)", MAX_ANGLES, (long long)pairs);
    const int64_t size = dtype == CINN_F32 ? 4 : 2, width = 16 / size, tokens = B * L;
    Params p{};
    p.tokens = tokens; p.L = (int)L; p.positions = positions; p.pos_b = pos_b; p.pos_l = pos_l; p.freq = freq; p.pairs = (int)pairs;
    p.magnitude = magnitude; p.sign = inverse ? -1.0f : 1.0f;
    bool vec = (interleaved ? 2 * pairs : pairs) % width == 0;
    int sides = 0;
    bool in_place = true;
    for (int i = 0; i < 2; ++i) {
        const bool used = in[i] != nullptr && heads[i] > 0;
        Side& sd = p.side[i];
        sd.heads = used ? (int)heads[i] : 0;
        if (!used || tokens == 0) continue;
        ++sides;
        CINN_CHECK_ARG(out[i] && positions && freq, "rotary: null pointer");
        CINN_CHECK_ARG(start[i] >= 0 && start[i] + 2 * pairs <= d[i] && d[i] < (1LL << 30), "rotary: %lld elements from %lld on do not fit a head of %lld",
                       (long long)(2 * pairs), (long long)start[i], (long long)d[i]);
        sd.in = in[i]; sd.out = out[i]; sd.d = (int)d[i]; sd.start = (int)start[i];
        sd.in_b = in_strides[3 * i]; sd.in_h = in_strides[3 * i + 1]; sd.in_l = in_strides[3 * i + 2];
        sd.out_b = out_strides[3 * i]; sd.out_h = out_strides[3 * i + 1]; sd.out_l = out_strides[3 * i + 2];
        in_place = in_place && in[i] == out[i];
        vec = vec && ((reinterpret_cast<uintptr_t>(in[i]) | reinterpret_cast<uintptr_t>(out[i])) & 15) == 0 && start[i] % width == 0 && d[i] % width == 0;
        for (int s = 0; s < 3; ++s) vec = vec && in_strides[3 * i + s] % width == 0 && out_strides[3 * i + s] % width == 0;
    }
    if (sides == 0) return CINN_OK;
    p.copy_rest = !in_place;
    // A CTA: eight tokens and up to 32 of their heads, fewer where that leaves SMs without work
    const int64_t want = 4LL * sm_count();
    int tile = (int)std::min<int64_t>({8, MAX_ANGLES / pairs, tokens}), most = 32;
    auto blocks_of = [&](int i) {
        return p.side[i].heads ? (tokens + tile - 1) / tile * ((p.side[i].heads + most - 1) / most) : 0;
    };
    while (blocks_of(0) + blocks_of(1) < want && (tile > 1 || most > 4)) {
        if (tile > 1) tile /= 2;
        else most /= 2;
    }
    p.tile = tile;
    for (int i = 0; i < 2; ++i) {
        p.side[i].head_chunks = p.side[i].heads ? (p.side[i].heads + most - 1) / most : 1;
        p.side[i].heads_per_chunk = most;
    }
    p.blocks0 = blocks_of(0);
    const int64_t blocks = p.blocks0 + blocks_of(1);
    CINN_CHECK_ARG(blocks < (1LL << 31), "rotary: too many tokens");
    if (dtype == CINN_F32) launch<float>(vec, interleaved, p, (unsigned)blocks, st);
    else if (dtype == CINN_BF16) launch<__nv_bfloat16>(vec, interleaved, p, (unsigned)blocks, st);
    else launch<__half>(vec, interleaved, p, (unsigned)blocks, st);
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

}  // namespace cinn
