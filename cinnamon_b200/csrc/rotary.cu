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
// Every element is read and written once, and where up to half of a head is rotated that is what bounds it.  Whole heads in 16 bits are bound by
// shared memory: cosines and sines are read anew for every head, 8 bytes a pair, neighbouring lanes 64 bytes apart on the same banks (32 query and
// 8 key heads x 4 x 4096 positions x 128 in bf16, 336 MB in and out: 128 of 128 rotated 78 us, 4.3 TB/s, interleaved 84; 64 of 128 57 us, 5.9 TB/s).
//
// A CTA takes jobs of up to 24 KiB (a few positions of a sequence and some of
// their heads), two of them on their way into shared memory by TMA while a third is turned in place and leaves the same way.  A job is
// one box of a tensor map over (part of a head, parts, heads, positions, sequences), so any strides of whole 16 bytes are one instruction of one
// thread: with loads and stores of the threads' own, resident CTAs did not keep enough bytes in flight (queries and keys of 32 x 8
// heads x 1024 positions x 192 in bf16, 403 MB in and out, 145 us; with four rows ahead per thread, and the registers for it, 212), and a bulk
// copy for each head of 384 bytes left its issuing warp the bound (195).  Cosines and sines are worked out once per job, for all of its
// heads.  What TMA cannot read goes through a kernel of plain loads and stores.
#include "tma.cuh"
#include <algorithm>
#include <cmath>

namespace cinn {
namespace rope {

constexpr int THREADS = 256;
constexpr int MAX_ANGLES = 2048;           // of a CTA's tokens; also the most pairs of a head
constexpr int STAGE = 24576;               // bytes of a job
constexpr int STAGES = 3;
constexpr int MAX_TILE = 32;               // positions of a job
constexpr int MAX_HEADS = 256;             // heads of a job
constexpr size_t SMEM = (size_t)STAGES * STAGE + 128;
constexpr long long WAIT_LIMIT = 4000000000LL;                             // cycles: about two seconds

__device__ int g_status = 0;               // 0, or (role << 8) | reason of a bounded wait that ran out

struct Side {                              // queries or keys
    const void* in;
    void* out;
    int64_t in_b, in_h, in_l, out_b, out_h, out_l;
    int heads, d, start;                   // elements of a head; where the rotated part starts
    int tile, heads_per_job;               // positions and heads of a job
    int tiles, head_chunks;                // jobs of a sequence: tiles x head_chunks
    int row, skip, parts;                  // elements of a head that a job moves (all, or in place the rotated ones), the rotated part's
                                           // place in them, and how many parts the tensor map has them in
    int64_t jobs;
};
struct Params {
    Side side[2];
    int B, L;
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
    if (!(turns >= 0.0)) return make_float2(NAN, NAN);                               // (a frequency that is no number, or infinite)
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

struct Job { int second, b, l0, n_pos, h0, n_heads; };
__device__ __forceinline__ Job job_at(const Params& p, int64_t j) {
    Job r;
    r.second = j >= p.side[0].jobs;
    const Side& sd = p.side[r.second];
    const unsigned at = (unsigned)(r.second ? j - p.side[0].jobs : j), of_b = (unsigned)sd.tiles * sd.head_chunks;
    r.b = (int)(at / of_b);
    const unsigned in = at - r.b * of_b, tile = in / (unsigned)sd.head_chunks;
    r.l0 = (int)tile * sd.tile;
    r.n_pos = min(sd.tile, p.L - r.l0);
    r.h0 = (int)(in - tile * sd.head_chunks) * sd.heads_per_job;
    r.n_heads = min(sd.heads_per_job, sd.heads - r.h0);
    return r;
}
__device__ __forceinline__ void turns_of_job(const Params& p, const Job& w, float2* turn) {
    for (int i = threadIdx.x; i < w.n_pos * p.pairs; i += THREADS) {
        const int t = i / p.pairs, f = i - t * p.pairs;
        const float2 cs = turn_of(p.positions[w.b * p.pos_b + (w.l0 + t) * p.pos_l], p.freq[f]);
        turn[i] = make_float2(cs.x * p.magnitude, cs.y * p.magnitude * p.sign);
    }
}
__device__ __forceinline__ void load_5d(const CUtensorMap* map, uint32_t bar, uint32_t dst, int h, int l, int b) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %3, %4, %5, %6}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar), "r"(0), "r"(h), "r"(l), "r"(b) : "memory");
}
__device__ __forceinline__ void store_5d(const CUtensorMap* map, uint32_t src, int h, int l, int b) {
    asm volatile("cp.async.bulk.tensor.5d.global.shared::cta.bulk_group [%0, {%2, %2, %3, %4, %5}], [%1];"
                 ::"l"(map), "r"(src), "r"(0), "r"(h), "r"(l), "r"(b) : "memory");
}
struct Maps { CUtensorMap in[2], out[2]; };

template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS)
rotary_kernel(const __grid_constant__ Maps maps, const __grid_constant__ Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ float2 s_turn[MAX_ANGLES];
    uint64_t* bars = reinterpret_cast<uint64_t*>(smem + (size_t)STAGES * STAGE);
    constexpr int VEC = 16 / (int)sizeof(T);
    const uint32_t bar0 = smem_u32(bars), data0 = smem_u32(smem);
    if (threadIdx.x == 0) {
        for (int s = 0; s < STAGES; ++s) mbar_init(bar0 + 8 * s, 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncthreads();
    pdl_wait();
    pdl_trigger();
    const int64_t n_jobs = p.side[0].jobs + p.side[1].jobs;
    const int mine = n_jobs > blockIdx.x ? (int)((n_jobs - blockIdx.x + gridDim.x - 1) / gridDim.x) : 0;
    auto fetch = [&](int i) {                              // by one thread: this CTA's i-th job into its stage
        const Job w = job_at(p, blockIdx.x + (int64_t)i * gridDim.x);
        const Side& sd = p.side[w.second];
        const int s = i % STAGES;
        // (the whole box: what lies outside is filled with zeros and counted)
        mbar_expect_tx(bar0 + 8 * s, (uint32_t)(sd.tile * sd.heads_per_job * sd.row * (int)sizeof(T)));
        load_5d(&maps.in[w.second], bar0 + 8 * s, data0 + s * STAGE, w.h0, w.l0, w.b);
    };
    if (threadIdx.x == 0)
        for (int i = 0; i < STAGES - 1 && i < mine; ++i) fetch(i);
    for (int i = 0; i < mine; ++i) {
        const Job w = job_at(p, blockIdx.x + (int64_t)i * gridDim.x);
        const Side& sd = p.side[w.second];
        const int s = i % STAGES;
        turns_of_job(p, w, s_turn);
        auto landed = [&](int job) {
            const uint32_t bar = bar0 + 8 * (uint32_t)(job % STAGES), parity = (uint32_t)(job / STAGES) & 1;
            bool ok = mbar_try_wait(bar, parity);
            for (const long long since = clock64(); !ok && clock64() - since < WAIT_LIMIT;) ok = mbar_try_wait(bar, parity);
            return ok;
        };
        if (__syncthreads_or(!landed(i))) {                // (also: the turns are there)
            if (threadIdx.x == 0) atomicCAS(&g_status, 0, (15 << 8) | 1);
            for (int j = i + 1; j < mine && j < i + STAGES - 1; ++j) landed(j);
            break;
        }
        T* stage = reinterpret_cast<T*>(smem + (size_t)s * STAGE) + sd.skip;
        // rows in the box: heads_per_job of each position (those that are not there as well: nothing of them is stored)
        const int per_row = (INTERLEAVED ? 2 * p.pairs : p.pairs) / VEC, per_pos = sd.heads_per_job * per_row, units = w.n_pos * per_pos;
        using V = Piece<T, VEC>;
        for (int u = threadIdx.x; u < units; u += THREADS) {
            const int t = u / per_pos, in_pos = u - t * per_pos, h = in_pos / per_row, at = (in_pos - h * per_row) * VEC;
            const float2* turn = s_turn + t * p.pairs;
            T* row = stage + (t * sd.heads_per_job + h) * sd.row;
            V x = *reinterpret_cast<V*>(row + at);
            if constexpr (INTERLEAVED) {
#pragma unroll
                for (int j = 0; j < VEC; j += 2) {
                    const float2 cs = turn[(at + j) >> 1];
                    const float a = widen<T>(x.v[j]), c = widen<T>(x.v[j + 1]);
                    x.v[j] = narrow<T>(fmaf(a, cs.x, -c * cs.y));
                    x.v[j + 1] = narrow<T>(fmaf(c, cs.x, a * cs.y));
                }
            } else {
                V y = *reinterpret_cast<V*>(row + p.pairs + at);
#pragma unroll
                for (int j = 0; j < VEC; ++j) {
                    const float2 cs = turn[at + j];
                    const float a = widen<T>(x.v[j]), c = widen<T>(y.v[j]);
                    x.v[j] = narrow<T>(fmaf(a, cs.x, -c * cs.y));
                    y.v[j] = narrow<T>(fmaf(c, cs.x, a * cs.y));
                }
                *reinterpret_cast<V*>(row + p.pairs + at) = y;
            }
            *reinterpret_cast<V*>(row + at) = x;
        }
        fence_async_smem();
        __syncthreads();
        if (threadIdx.x == 0) {
            store_5d(&maps.out[w.second], data0 + s * STAGE, w.h0, w.l0, w.b);
            tma_store_commit();
            if (i + STAGES - 1 < mine) {                   // into the stage whose job left before this one
                asm volatile("cp.async.bulk.wait_group.read 1;" ::: "memory");
                fetch(i + STAGES - 1);
            }
        }
    }
    if (threadIdx.x == 0) tma_store_wait_all();
}

// Element by element, for what TMA cannot read: a thread moves a pair, or an element of the rest.
template <typename T, bool INTERLEAVED>
__global__ void __launch_bounds__(THREADS)
rotary_plain_kernel(const __grid_constant__ Params p) {
    pdl_wait();
    pdl_trigger();
    __shared__ float2 s_turn[MAX_ANGLES];
    const Job w = job_at(p, blockIdx.x);
    const Side& sd = p.side[w.second];
    turns_of_job(p, w, s_turn);
    __syncthreads();
    const int rest = p.copy_rest ? sd.d - 2 * p.pairs : 0, units = rest + p.pairs;
    for (int64_t i = threadIdx.x; i < (int64_t)w.n_pos * w.n_heads * units; i += THREADS) {
        const int r = (int)(i / units), u = (int)(i - (int64_t)r * units), t = r / w.n_heads, h = w.h0 + r - t * w.n_heads;
        const T* in = static_cast<const T*>(sd.in) + w.b * sd.in_b + (w.l0 + t) * sd.in_l + h * sd.in_h;
        T* out = static_cast<T*>(sd.out) + w.b * sd.out_b + (w.l0 + t) * sd.out_l + h * sd.out_h;
        if (u < rest) {
            const int at = u < sd.start ? u : u + 2 * p.pairs;             // (the rotated part lies in between)
            out[at] = in[at];
        } else {
            const int f = u - rest, at = sd.start + (INTERLEAVED ? 2 * f : f), other = at + (INTERLEAVED ? 1 : p.pairs);
            const float2 cs = s_turn[t * p.pairs + f];
            const float a = widen<T>(in[at]), c = widen<T>(in[other]);
            out[at] = narrow<T>(fmaf(a, cs.x, -c * cs.y));
            out[other] = narrow<T>(fmaf(c, cs.x, a * cs.y));
        }
    }
}

template <typename T, bool INTERLEAVED>
static int launch(const Maps* maps, const Params& p, int64_t jobs, cudaStream_t st) {
    if (maps) {
        int rc = allow_smem_once<rotary_kernel<T, INTERLEAVED>>(SMEM);
        if (rc) return rc;
        const unsigned grid = (unsigned)std::min<int64_t>(jobs, 2LL * sm_count());        // two CTAs of an SM
        launch_dependent(rotary_kernel<T, INTERLEAVED>, dim3(grid), dim3(THREADS), SMEM, st, *maps, p);
    } else {
        launch_dependent(rotary_plain_kernel<T, INTERLEAVED>, dim3((unsigned)jobs), dim3(THREADS), 0, st, p);
    }
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

// A head's `row` elements in equal parts that a box can hold (256 of a dimension at most), each of whole 16 bytes; 0: there are none
static int parts_of(int row, int width) {
    for (int parts = (row + 255) / 256; parts <= 256; ++parts)
        if (row % parts == 0 && row / parts % width == 0) return parts;
    return 0;
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
    const int64_t size = dtype == CINN_F32 ? 4 : 2, width = 16 / size;
    const bool swap = L == 1;
    if (swap) {                                              // one position of many sequences: as many positions of one
        L = B;
        B = 1;
        pos_l = pos_b;
        pos_b = 0;
    }
    Params p{};
    p.B = (int)B; p.L = (int)L; p.positions = positions; p.pos_b = pos_b; p.pos_l = pos_l; p.freq = freq; p.pairs = (int)pairs;
    p.magnitude = magnitude; p.sign = inverse ? -1.0f : 1.0f;
    bool tma = (interleaved ? 2 * pairs : pairs) % width == 0, in_place = true;
    int sides = 0;
    for (int i = 0; i < 2; ++i) {
        const bool used = in[i] != nullptr && heads[i] > 0 && B > 0 && L > 0;
        Side& sd = p.side[i];
        sd.heads = used ? (int)heads[i] : 0;
        sd.tiles = sd.head_chunks = sd.tile = sd.heads_per_job = 1;
        if (!used) continue;
        ++sides;
        CINN_CHECK_ARG(out[i] && positions && freq, "rotary: null pointer");
        CINN_CHECK_ARG(start[i] >= 0 && start[i] + 2 * pairs <= d[i] && d[i] < (1LL << 24), "rotary: %lld elements from %lld on do not fit a head of %lld",
                       (long long)(2 * pairs), (long long)start[i], (long long)d[i]);
        sd.in = in[i]; sd.out = out[i]; sd.d = (int)d[i]; sd.start = (int)start[i];
        const int64_t *si = in_strides + 3 * i, *so = out_strides + 3 * i;
        sd.in_b = swap ? 0 : si[0]; sd.in_h = si[1]; sd.in_l = swap ? si[0] : si[2];
        sd.out_b = swap ? 0 : so[0]; sd.out_h = so[1]; sd.out_l = swap ? so[0] : so[2];
        in_place = in_place && in[i] == out[i];
    }
    if (sides == 0) return CINN_OK;
    p.copy_rest = !in_place;
    for (int i = 0; i < 2; ++i) {
        Side& sd = p.side[i];
        if (!sd.heads) continue;
        sd.row = in_place ? (int)(2 * pairs) : sd.d;
        sd.skip = in_place ? 0 : sd.start;
        sd.parts = parts_of(sd.row, (int)width);
        const int64_t from = in_place ? sd.start : 0;
        const uintptr_t bases = (uintptr_t)sd.in | (uintptr_t)sd.out;
        tma = tma && sd.parts > 0 && (bases & 15) == 0 && from % width == 0 && sd.start % width == 0 && sd.row * size <= STAGE;
        // (a stride along one entry is never taken; one of 0, or below, is none that a tensor map has)
        const int64_t counts[3] = {sd.heads, L, B}, strides[6] = {sd.in_h, sd.in_l, sd.in_b, sd.out_h, sd.out_l, sd.out_b};
        for (int s = 0; s < 6; ++s) tma = tma && (counts[s % 3] == 1 || (strides[s] > 0 && strides[s] % width == 0 && strides[s] * size < (1LL << 40)));
    }
    // Jobs: as many heads of a position as fit, then as many positions; smaller ones where there would not be two for every SM
    int64_t jobs = 0;
    for (int64_t most = STAGE;; most /= 2) {
        jobs = 0;
        bool smaller = false;
        for (int i = 0; i < 2; ++i) {
            Side& sd = p.side[i];
            if (!sd.heads) continue;
            const int64_t rows = std::max<int64_t>(1, most / (sd.row * size));
            sd.heads_per_job = (int)std::min<int64_t>({(int64_t)sd.heads, rows, (int64_t)MAX_HEADS});
            sd.tile = (int)std::max<int64_t>(1, std::min<int64_t>({rows / sd.heads_per_job, (int64_t)MAX_TILE, MAX_ANGLES / pairs, L}));
            sd.head_chunks = (sd.heads + sd.heads_per_job - 1) / sd.heads_per_job;
            sd.tiles = (int)((L + sd.tile - 1) / sd.tile);
            sd.jobs = B * sd.tiles * sd.head_chunks;
            jobs += sd.jobs;
            smaller = smaller || rows > 4;
        }
        if (jobs >= 2LL * sm_count() || !smaller) break;
    }
    CINN_CHECK_ARG(jobs < (1LL << 31), "rotary: too many positions");
    Maps maps;
    for (int i = 0; i < 2 && tma; ++i) {
        const Side& sd = p.side[i];
        if (!sd.heads) continue;
        const uint64_t part = (uint64_t)(sd.row / sd.parts);
        const uint64_t dims[5] = {part, (uint64_t)sd.parts, (uint64_t)sd.heads, (uint64_t)L, (uint64_t)B};
        const uint32_t box[5] = {(uint32_t)part, (uint32_t)sd.parts, (uint32_t)sd.heads_per_job, (uint32_t)sd.tile, 1};
        const int64_t from = in_place ? sd.start * size : 0;
        auto encode = [&](CUtensorMap* m, const void* base, int64_t h, int64_t l, int64_t b) {
            const auto bytes = [&](int64_t stride, int64_t count) { return (uint64_t)(count == 1 ? 16 : stride * size); };
            const uint64_t strides[4] = {part * size, bytes(h, sd.heads), bytes(l, L), bytes(b, B)};
            return encode_map(m, static_cast<const uint8_t*>(base) + from, 5, dims, strides, box,
                              size == 4 ? CU_TENSOR_MAP_DATA_TYPE_UINT32 : CU_TENSOR_MAP_DATA_TYPE_UINT16, CU_TENSOR_MAP_SWIZZLE_NONE);
        };
        int rc = encode(&maps.in[i], sd.in, sd.in_h, sd.in_l, sd.in_b);
        if (!rc) rc = encode(&maps.out[i], sd.out, sd.out_h, sd.out_l, sd.out_b);
        if (rc) return rc;
    }
    const Maps* m = tma ? &maps : nullptr;
    if (dtype == CINN_F32) return interleaved ? launch<float, true>(m, p, jobs, st) : launch<float, false>(m, p, jobs, st);
    if (dtype == CINN_BF16) return interleaved ? launch<__nv_bfloat16, true>(m, p, jobs, st) : launch<__nv_bfloat16, false>(m, p, jobs, st);
    return interleaved ? launch<__half, true>(m, p, jobs, st) : launch<__half, false>(m, p, jobs, st);
}

int read_rotary_status(int* out, int reset) {
    int v = 0;
    CINN_CHECK_CUDA(cudaMemcpyFromSymbol(&v, rope::g_status, sizeof(int)));
    if (reset && v) {
        const int z = 0;
        CINN_CHECK_CUDA(cudaMemcpyToSymbol(rope::g_status, &z, sizeof(int)));
    }
    *out = v;
    return CINN_OK;
}

}  // namespace cinn
