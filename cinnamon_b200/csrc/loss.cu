// Output projection and softmax cross entropy in one operator, forward and backward, without the logits in memory.
//
//   z = x W^T                      x (T, d), W (V, d), 16-bit operands, fp32 sums in tensor memory
//   loss_t = log sum_v e^z_tv - z_t,target(t)
//   dz_tv = g_t (e^(z_tv - lse_t) - [v = target(t)]),   dx = dz W,   dW = dz^T x
//
// Forward: a tile of 256 tokens x 256 words is multiplied by a pair of SMs and read out of tensor memory once, into a running
// maximum and sum per token (two fp32 numbers); tiles of one run of words are joined in registers, runs by a small pass
// at the end.  Backward, one of two ways:
//   late    The words in pieces; a piece's product is made again, turned into dz in the epilogue and rounded to the operands' type
//           (bf16, or fp16 times 2^14, so that small probabilities keep their bits), and two products over the piece add up dx
//           (fp32, in L2) and write the piece's rows of dW.  2 T V d forward and 6 T V d backward, one 2 T V d more than with kept logits.
//   early   The tokens in pieces; a piece's e^(z - maximum of its 128 words) is written in fp16, times 2^15, by the forward's product, turned into dz by one
//           pass over it once the sums are known, and the two products add up dx and dW in fp32, all in the forward.  What is left for the
//           backward is the loss's gradient, one number, and the one rounding.  6 T V d in all.  The sums stay until the backward, and a
//           loss whose gradient is never asked for has cost three times as much.  For sums and means over many and wide rows (early_pays).
// The memory is that of one piece, and early that of the gradients' sums.
//
// Tokens whose target is ignored take part in nothing: the others' rows are gathered first (where none is ignored, x is read
// as it is), so that what stands in ignored rows, infinities and NaN as well, reaches neither gradient, and half a batch of
// prompts costs half.
//
// Sums, maxima and the two statistics per token are fp32; the logarithm of the sum is kept apart from the maximum, since
// their sum would round away what e^(z - lse) - 1 of a well-predicted token is made of.
#include "tcgen05.cuh"
#include <algorithm>
#include <cmath>

namespace cinn {

int gemm_sm_count();                       // SMs that the persistent kernels may take (gemm.cu)

namespace ce {

__device__ int g_status = 0;               // 0, or (role << 8) | reason of a bounded wait that ran out

enum Mode { STATS = 0, SOFT = 1, KEEP = 2, DX = 3, DW = 4 };

constexpr int M = 256, N = 256;            // the pair's tile
constexpr int KE = 64;                     // elements of a K block: 128 bytes
constexpr int SIDE = 128 * 128;            // bytes of one operand's stage in one CTA: 128 rows (or columns) x 64 elements
constexpr int EPI = 8, COLS = 128;         // epilogue warps: four lane quarters x two halves of the columns
constexpr int W_TMA = EPI, W_MMA = EPI + 1;
constexpr int THREADS = (EPI + 2) * 32;
constexpr int BOX = 32 * 128;              // a TMA-store box: 32 rows of 128 bytes
// The operands' ring takes what shared memory there is: with four stages the logits' product waited for operands 1800 of a tile's 4600 cycles, and
// where dz is written to memory at the same time 3900 of 6100.
constexpr int STAGES_Z = 7;                // product_kernel, which stores from registers
constexpr int STAGES_G = 5, BOXES = 2;     // grads_kernel; boxes of an epilogue warp, filled in turn
constexpr int C_BYTES = EPI * BOXES * BOX;
constexpr size_t SMEM_Z = (size_t)STAGES_Z * 2 * SIDE + 256 + 1024, SMEM_G = (size_t)STAGES_G * 2 * SIDE + C_BYTES + 256 + 1024;
constexpr int GROUP = 16;                  // tiles of tokens that meet a run of words before the next ones do (L2)
constexpr int SCAN = 1024;                 // tokens per CTA of the passes that gather
// Of the exponentials that the early way keeps in fp16: the largest of 128 words is 1, and so becomes 2^15.  Words down to 2^-29 of it (20 nats) keep all
// their bits and those down to 2^-40 (27 nats) some; unscaled, fp16's smallest numbers began at 2^-14 (10 nats) and a rare word's row of dW was
// zero from 17 nats on.
constexpr float KEPT_SCALE = 32768.0f;
constexpr float LOG2E = 1.4426950408889634f;
constexpr float FP16_SCALE = 16384.0f;     // of dz in fp16: the smallest probability with all its bits is then 2^-28

struct Params {
    const int* n_valid;                    // rows in use (device)
    int T, V, d;                           // T: x itself is read where all of so many rows are in use (-1: never)
    int v0, vc;                            // a piece of the words: its first, how many
    int t0, tc;                            // a piece of the rows in use
    int parts;                             // STATS, KEEP: runs of words per tile of tokens
    int dx_splits, dw_splits;              // pieces that the reductions are cut into, each with sums of its own; 0: not wanted
    int dx_rows, dw_rows;                  // rows of one such piece's sums
    int add_dx, add_dw;                    // add to the sums of earlier pieces
    int per_row;                           // SOFT: gradients per token (reduction "none")
    int half;                              // few tokens: dz's second rows, what the rounding of the first left; 0: none
    int64_t part_ld;
    float2* part;                          // STATS, KEEP: (parts * 2, part_ld) maximum and sum, a row for every one of the piece
    float* tile_max;                       // KEEP: (two for each tile of words, part_ld) maximum of 128 words
    float* target_logit;
    const int* target;                     // per row in use
    const int* rows;                       // the token of every row in use
    const float2* stat;                    // per row: maximum, log2 of the sum
    const float* grad;                     // the loss's gradient: one number, or one per token
    const unsigned* grad_max;              // the bits of the largest finite |gradient| (reduction "none")
    int mean;
    float log2e;                           // of one unit of the logits as they stand in tensor memory (see growth)
    uint16_t* dz;                          // the piece's (KEEP: what it will be made of), rows of dz_ld (a multiple of 64)
    int dz_ld;
};

__device__ __forceinline__ bool wait(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
    return mbar_wait_bounded(bar, parity, abort_flag, code, &g_status);
}
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity, volatile int* abort_flag, int code) {
    return __all_sync(0xffffffffu, wait(bar, parity, abort_flag, code));
}
__device__ __forceinline__ uint32_t cta_rank() {
    uint32_t r;
    asm volatile("mov.u32 %0, %%cluster_ctarank;" : "=r"(r));
    return r;
}
__device__ __forceinline__ uint32_t mapa(uint32_t addr, uint32_t rank) {
    uint32_t r;
    asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(addr), "r"(rank));
    return r;
}
__device__ __forceinline__ void cluster_sync() {
    asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");
    asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// relaxed: it hands over a buffer of tensor memory whose reads are complete (see gemm_pair.cuh)
__device__ __forceinline__ void arrive_remote(uint32_t cluster_addr) {
    asm volatile("mbarrier.arrive.relaxed.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_addr) : "memory");
}
__device__ __forceinline__ void load_2d(const CUtensorMap* map, uint32_t bar_cluster, uint32_t dst, int x, int y) {
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];"
        ::"r"(dst), "l"(map), "r"(bar_cluster), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void add_2d(const CUtensorMap* map, uint32_t src, int x, int y) {
    asm volatile("cp.reduce.async.bulk.tensor.2d.global.shared::cta.add.bulk_group [%0, {%2, %3}], [%1];"
                 ::"l"(map), "r"(src), "r"(x), "r"(y) : "memory");
}
__device__ __forceinline__ void commit_pair(uint32_t own, uint32_t peer) {
    asm volatile(
        "{\n\t.reg .pred e;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t"
        "@e tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.b64 [%1];\n\t}"
        ::"r"(own), "r"(peer) : "memory");
}
// The four steps of a K block by one election; low words of the descriptors, STEP in units of 16 bytes.
template <int STEP_A, int STEP_B>
__device__ __forceinline__ void mma_block(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool fresh) {
    asm volatile(
        "{\n\t.reg .pred p, e;\n\t.reg .b64 a, b;\n\t.reg .b32 x, y;\n\t"
        "elect.sync _|e, 0xffffffff;\n\t"
        "setp.ne.b32 p, %5, 0;\n\t"
        "mov.b64 a, {%1, %4};\n\tmov.b64 b, {%2, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, p;\n\t"
        "add.u32 x, %1, %6;\n\tadd.u32 y, %2, %7;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, %8;\n\tadd.u32 y, %2, %9;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t"
        "add.u32 x, %1, %10;\n\tadd.u32 y, %2, %11;\n\tmov.b64 a, {x, %4};\n\tmov.b64 b, {y, %4};\n\t"
        "@e tcgen05.mma.cta_group::2.kind::f16 [%0], a, b, %3, 1;\n\t}"
        ::"r"(d), "r"(a), "r"(b), "r"(idesc), "r"(DESC_HI), "r"(fresh ? 0u : 1u), "n"(STEP_A), "n"(STEP_B), "n"(2 * STEP_A), "n"(2 * STEP_B),
          "n"(3 * STEP_A), "n"(3 * STEP_B) : "memory");
}
__device__ __forceinline__ void ld32(uint32_t taddr, uint32_t (&r)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, "
        "%19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
          "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
          "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
          "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
        : "r"(taddr));
}
__device__ __forceinline__ void ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ float exp2_approx(float x) {          // relative error 2^-22; a result below 2^-126 is 0
    float r;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(r) : "f"(x));
    return r;
}
template <bool BF16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    if constexpr (BF16) {
        const __nv_bfloat162 t = __floats2bfloat162_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    } else {
        const __half2 t = __floats2half2_rn(a, b);
        return *reinterpret_cast<const uint32_t*>(&t);
    }
}

template <bool BF16>
__device__ __forceinline__ float2 unpack2(uint32_t v) {
    if constexpr (BF16) return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(&v));
    else return __half22float2(*reinterpret_cast<const __half2*>(&v));
}

// What the gradients are multiplied by once their sums are complete: the loss's gradient (over the number of targets for a
// mean), or the largest of the tokens' gradients, to which SOFT has related each.
__device__ __forceinline__ float final_scale(const Params& p, bool bf16) {
    // (a mean over nothing: no gradient, not 0 times infinity)
    const float s = p.per_row ? __uint_as_float(*p.grad_max) : !p.mean ? *p.grad : *p.n_valid ? *p.grad / (float)*p.n_valid : 0.0f;
    return bf16 ? s : s * (1.0f / FP16_SCALE);
}

// rows in use of the piece
__device__ __forceinline__ int rows_of(const Params& p) { return min(max(*p.n_valid - p.t0, 0), p.tc); }

// rows of dz that dW sums over
__device__ __forceinline__ int summed(const Params& p, int valid) { return valid ? valid + p.half : 0; }

struct Unit { int m0, n_first, n_last, kb0, KB, split; };

// Work of one cluster at a time: a tile (a run of them along the words for STATS and KEEP).  Groups of GROUP row tiles, rows fastest inside.
template <int MODE>
__device__ __forceinline__ int unit_count(const Params& p, int valid) {
    const int rows = MODE == DW ? p.vc : valid, cols = MODE == SOFT ? p.vc : MODE <= KEEP ? p.V : p.d;
    const int tiles = ((rows + M - 1) / M) * (MODE == STATS || MODE == KEEP ? p.parts : (cols + N - 1) / N);
    return MODE == DX ? tiles * p.dx_splits : MODE == DW ? tiles * p.dw_splits : tiles;
}
template <int MODE>
__device__ __forceinline__ Unit unit_at(const Params& p, int valid, int u) {
    const int rows = MODE == DW ? p.vc : valid, cols = MODE == SOFT ? p.vc : MODE <= KEEP ? p.V : p.d;
    const int m_tiles = (rows + M - 1) / M, n_tiles = (cols + N - 1) / N, across = MODE == STATS || MODE == KEEP ? p.parts : n_tiles;
    const int red = MODE == DX ? p.vc : MODE == DW ? summed(p, valid) : p.d, blocks = (red + KE - 1) / KE;
    Unit r;
    r.split = 0; r.kb0 = 0; r.KB = blocks;
    if constexpr (MODE >= DX) {
        const int splits = MODE == DX ? p.dx_splits : p.dw_splits;
        r.split = u / (m_tiles * across);
        u -= r.split * (m_tiles * across);
        r.kb0 = (int)((int64_t)blocks * r.split / splits);
        r.KB = (int)((int64_t)blocks * (r.split + 1) / splits) - r.kb0;
    }
    const int g = u / (GROUP * across), first = g * GROUP, size = min(GROUP, m_tiles - first);
    const int in = u - g * GROUP * across, n = in / size;
    r.m0 = (first + in - n * size) * M;
    if constexpr (MODE == STATS || MODE == KEEP) {
        const int run = (n_tiles + p.parts - 1) / p.parts;             // (all of one length but the last)
        r.n_first = n * run;
        r.n_last = min(r.n_first + run, n_tiles);
    } else {
        r.n_first = n; r.n_last = n + 1;
    }
    return r;
}

// The two gradients' tiles as one list for each cluster: first its share of those with the longer reduction; then, where the last round of
// these leaves clusters over, the shorter ones that fit beside it; then the rest in turn.  (One kernel for each: 128 x 2 tiles of dx and 32 x 2
// of dW on 74 pairs end in rounds that are half or nearly empty, 219 + 198 us of which 163 + 163 are products at the STATS kernel's rate.)
struct Schedule {
    int n_long, n_short, clusters, cluster, rem, pre, fit;
    bool dx_long;
    __device__ Schedule(const Params& p, int valid, int cluster_, int clusters_) : clusters(clusters_), cluster(cluster_) {
        const int n_dx = unit_count<DX>(p, valid), n_dw = unit_count<DW>(p, valid);
        const int l_dx = p.dx_splits ? ((p.vc + KE - 1) / KE + p.dx_splits - 1) / p.dx_splits : 0;
        const int l_dw = p.dw_splits ? ((summed(p, valid) + KE - 1) / KE + p.dw_splits - 1) / p.dw_splits : 0;
        dx_long = l_dx >= l_dw;
        n_long = dx_long ? n_dx : n_dw;
        n_short = dx_long ? n_dw : n_dx;
        const int l_long = max(l_dx, l_dw), l_short = max(1, min(l_dx, l_dw));
        rem = n_long % clusters;
        fit = rem ? l_long / l_short : 0;
        pre = rem ? (int)min((int64_t)n_short, (int64_t)(clusters - rem) * fit) : 0;
    }
    // this cluster's i-th tile: its number among dx's or dW's; false: there are no more
    __device__ __forceinline__ bool at(int i, bool& dx, int& u) const {
        const int longs = n_long > cluster ? (n_long - cluster + clusters - 1) / clusters : 0;
        if (i < longs) { dx = dx_long; u = cluster + i * clusters; return true; }
        i -= longs;
        dx = !dx_long;
        const int room = clusters - rem;
        int here = 0;                                       // of the shorter ones beside the last long round
        if (rem && cluster >= rem && pre > cluster - rem) here = (pre - (cluster - rem) + room - 1) / room;
        if (i < here) { u = cluster - rem + i * room; return true; }
        const int64_t v = pre + cluster + (int64_t)(i - here) * clusters;
        if (v >= n_short) return false;
        u = (int)v;
        return true;
    }
};

__device__ __forceinline__ void store32(uint16_t* at, const uint32_t* v) {             // 32 bytes
    asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(at), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]),
                 "r"(v[6]), "r"(v[7]) : "memory");
}

// What every product kernel sets up: barriers, tensor memory, the roles' view of both.
template <int STAGES, int SMEM_C>
struct Setup {
    uint8_t *smem_a, *smem_b, *c_stage;
    volatile int* abort_flag;
    uint32_t full0, empty0, tfull0, tempty0, rank, tmem;
    int warp, lane;

    __device__ __forceinline__ Setup(uint8_t* raw) {
        uint8_t* smem = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(raw) + 1023) & ~(uintptr_t)1023);
        smem_a = smem;
        smem_b = smem + STAGES * SIDE;
        c_stage = smem + STAGES * 2 * SIDE;
        uint64_t* bars = reinterpret_cast<uint64_t*>(c_stage + SMEM_C);
        // [0, S) full (used in the leader), [S, 2S) empty, then: tensor memory full (2), empty (2, leader)
        uint32_t* tmem_slot = reinterpret_cast<uint32_t*>(bars + 2 * STAGES + 4);
        abort_flag = reinterpret_cast<volatile int*>(tmem_slot + 1);
        warp = threadIdx.x >> 5; lane = threadIdx.x & 31;
        rank = cta_rank();
        full0 = smem_u32(bars); empty0 = smem_u32(bars + STAGES);
        tfull0 = smem_u32(bars + 2 * STAGES); tempty0 = smem_u32(bars + 2 * STAGES + 2);
        if (threadIdx.x == 0) *abort_flag = 0;
        if (warp == W_TMA && lane == 0) {
            for (int s = 0; s < STAGES; ++s) { mbar_init(full0 + 8 * s, 1); mbar_init(empty0 + 8 * s, 1); }
            for (int b = 0; b < 2; ++b) { mbar_init(tfull0 + 8 * b, 1); mbar_init(tempty0 + 8 * b, 2 * EPI); }
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
        if (warp == W_MMA) {
            asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
            asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
        }
        pdl_wait();
        if (warp == W_MMA) pdl_trigger();
        tc_fence_before();
        __syncthreads();
        cluster_sync();
        tc_fence_after();
        tmem = *tmem_slot;
    }
    // nobody leaves while the other CTA may still read this CTA's shared memory or signal its barriers
    __device__ __forceinline__ void finish() {
        tc_fence_before();
        __syncthreads();
        cluster_sync();
        if (warp == W_MMA) {
            tc_fence_after();
            asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
        }
    }
    // The producer gives up: time for the copies already issued to land (their barrier may be the other CTA's)
    __device__ __forceinline__ void drain() {
        const long long t0 = clock64();
        while (clock64() - t0 < 2000000LL) { }
    }
    // by the MMA warp, after its last tile: every MMA issued must have retired before tensor memory is freed
    __device__ __forceinline__ void retire(uint32_t tiles, bool alive) {
        if (alive && tiles) wait(tfull0 + 8 * ((tiles - 1) & 1), (tiles - 1) >> 1 & 1, abort_flag, (12 << 8) | 3);
    }
};

// 16 bytes of a box's row: 16-byte pieces, 128-byte swizzle
__device__ __forceinline__ void stage16(uint32_t box, int row, int piece, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
    asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(box + row * 128 + ((piece ^ (row & 7)) << 4)), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
// An epilogue warp's two boxes, in turn: `open` waits until the one to be filled has been read by its last store (the one after may still
// be on its way), `send` hands it over: a tile's conversion and its stores run beside one another, where one warp for all of a tile's stores, behind a
// barrier of all warps, put them one after the other.
struct Boxes {
    uint32_t slot, turn = 0;
    __device__ __forceinline__ Boxes(uint32_t s) : slot(s) {}
    __device__ __forceinline__ uint32_t open(int lane) {
        if (lane == 0) asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(BOXES - 1) : "memory");
        __syncwarp();
        return slot + turn * BOX;
    }
    __device__ __forceinline__ void send(int lane, const CUtensorMap* map, int col, int row, bool store, bool add) {
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
            const uint32_t box = slot + turn * BOX;
            if (store) {
                if (add) add_2d(map, box, col, row);
                else tma_store_2d(map, box, col, row);
            }
            tma_store_commit();
        }
        turn = turn + 1 == BOXES ? 0 : turn + 1;
    }
    __device__ __forceinline__ void drain(int lane) { if (lane == 0) tma_store_wait_all(); }
};
__device__ __forceinline__ uint64_t pair2(float a, float b) {
    uint64_t r;
    asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(a), "f"(b));
    return r;
}

// The logits' product: A = x, B = W, both K-major.  STATS leaves maxima and sums of its runs, SOFT dz of the piece, KEEP both maxima and sums, and
// e^(z - maximum) in fp16 (times KEPT_SCALE), of each half tile.  xg: x's rows in use, gathered; read in x's place where some token is ignored.  Bound by the tensor cores
// (active 87.6 % of STATS at 8192 x 32000 x 512, 74 % of SOFT, which also writes dz) and, in long calls, by the power that they draw.
template <int MODE, bool BF16>
__global__ void __launch_bounds__(THREADS, 1)
product_kernel(const __grid_constant__ CUtensorMap tm_a, const __grid_constant__ CUtensorMap tm_b, const __grid_constant__ CUtensorMap tm_xg,
               const Params p) {
    constexpr int STAGES = STAGES_Z;
    extern __shared__ uint8_t smem_raw[];
    Setup<STAGES, 0> s(smem_raw);
    const int warp = s.warp, lane = s.lane, rank = (int)s.rank;
    const int valid = rows_of(p);
    const int n_units = unit_count<MODE>(p, valid);
    const int cluster = blockIdx.x >> 1, n_clusters = gridDim.x >> 1;

    if (warp == W_TMA) {
        // ------------------------------ TMA producer (both CTAs) ------------------------------
        if (lane == 0) {
            const uint32_t full_leader = mapa(s.full0, 0);
            const CUtensorMap* map_a = *p.n_valid != p.T ? &tm_xg : &tm_a;
            uint32_t it = 0;
            bool alive = true;
            for (int u = cluster; u < n_units && alive; u += n_clusters) {
                const Unit w = unit_at<MODE>(p, valid, u);
                for (int nt = w.n_first; nt < w.n_last && alive; ++nt) {
                    const int ma = p.t0 + w.m0 + 128 * rank, nb = p.v0 + nt * N + 128 * rank;
                    for (int kb = 0; kb < w.KB; ++kb, ++it) {
                        const int st = it % STAGES;
                        if (!wait(s.empty0 + 8 * st, (it / STAGES & 1) ^ 1, s.abort_flag, (11 << 8) | 1)) { alive = false; break; }
                        if (rank == 0) mbar_expect_tx(s.full0 + 8 * st, 4 * SIDE);
                        load_2d(map_a, full_leader + 8 * st, smem_u32(s.smem_a + st * SIDE), kb * KE, ma);
                        load_2d(&tm_b, full_leader + 8 * st, smem_u32(s.smem_b + st * SIDE), kb * KE, nb);
                    }
                }
            }
            if (!alive) s.drain();
        }
    } else if (warp == W_MMA) {
        // ------------------------------ MMA issuer (leader; a whole warp, one elected lane) ------------------------------
        if (rank == 0) {
            constexpr uint32_t idesc = make_idesc_f16(BF16, M, N);
            const uint32_t a0 = panel_desc(smem_u32(s.smem_a)), b0 = panel_desc(smem_u32(s.smem_b));
            const uint32_t tfull_own = mapa(s.tfull0, 0), tfull_peer = mapa(s.tfull0, 1);
            const uint32_t empty_own = mapa(s.empty0, 0), empty_peer = mapa(s.empty0, 1);
            uint32_t it = 0, tile = 0;
            bool alive = true;
            for (int u = cluster; u < n_units && alive; u += n_clusters) {
                const Unit w = unit_at<MODE>(p, valid, u);
                for (int nt = w.n_first; nt < w.n_last && alive; ++nt, ++tile) {
                    const uint32_t b = tile & 1;
                    if (!wait_warp(s.tempty0 + 8 * b, (tile >> 1 & 1) ^ 1, s.abort_flag, (12 << 8) | 2)) { alive = false; break; }
                    tc_fence_after();
                    for (int kb = 0; kb < w.KB; ++kb, ++it) {
                        const uint32_t st = it % STAGES;
                        if (!wait_warp(s.full0 + 8 * st, it / STAGES & 1, s.abort_flag, (12 << 8) | 1)) { alive = false; break; }
                        tc_fence_after();
                        mma_block<2, 2>(s.tmem + b * N, a0 + st * (SIDE >> 4), b0 + st * (SIDE >> 4), idesc, kb == 0);
                        commit_pair(empty_own + 8 * st, empty_peer + 8 * st);
                    }
                    if (!alive) break;
                    commit_pair(tfull_own + 8 * b, tfull_peer + 8 * b);
                }
            }
            s.retire(tile, alive);
        }
    } else {
        // ------------------------------ epilogue (both CTAs) ------------------------------
        const int q = warp & 3, h = warp >> 2;
        const uint32_t tempty_leader = mapa(s.tempty0, 0);
        uint32_t tile = 0;
        bool alive = true;
        float most = 0.0f;                                 // SOFT, gradients per token: the largest
        if constexpr (MODE == SOFT) {
            if (p.per_row) most = __uint_as_float(*p.grad_max);
        }
        for (int u = cluster; u < n_units && alive; u += n_clusters) {
            const Unit w = unit_at<MODE>(p, valid, u);
            const int row = w.m0 + 128 * rank + q * 32 + lane;
            const bool low = MODE == SOFT && p.half && row >= p.half;          // (the same for the warp)
            const int own = low ? row - p.half : row;
            const bool live = own < valid;
            float mx = -INFINITY, sum = 0.0f, rel = 0.0f;
            int target = -1;
            if (live) {
                target = p.target[p.t0 + own];
                if constexpr (MODE == SOFT) {
                    const float2 st = p.stat[own];
                    mx = st.x; sum = st.y;
                    rel = 1.0f;
                    if (p.per_row) {
                        const float g = p.grad[p.rows[own]];
                        rel = most > 0.0f ? g / most : g;              // (0: they are zeros, infinities and NaN)
                    }
                    if (!BF16) rel *= FP16_SCALE;
                }
            }
            for (int nt = w.n_first; nt < w.n_last; ++nt, ++tile) {
                const uint32_t b = tile & 1;
                if (!wait_warp(s.tfull0 + 8 * b, tile >> 1 & 1, s.abort_flag, (13 << 8) | 1)) { alive = false; break; }
                tc_fence_after();
                const uint32_t taddr = s.tmem + ((uint32_t)(q * 32) << 16) + b * N + h * COLS;
                const int col0 = p.v0 + nt * N + h * COLS;                     // of this warp, among all words
                if constexpr (MODE == STATS) {
#pragma unroll 1
                    for (int c = 0; c < COLS / 32; ++c) {
                        uint32_t r[32];
                        ld32(taddr + c * 32, r);
                        ld_wait();
                        const int at = col0 + c * 32;
                        if (at >= p.V) break;
                        const int hit = target - at;
                        if ((unsigned)hit < 32u) {
                            float z = 0.0f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) z = j == hit ? __uint_as_float(r[j]) : z;
                            p.target_logit[p.t0 + row] = z;
                        }
                        if (at + 32 > p.V) {               // words past the last one
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (at + j >= p.V) r[j] = __float_as_uint(-INFINITY);
                        }
                        float top = mx;
#pragma unroll
                        for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(r[j]));
                        const float base = top == -INFINITY ? 0.0f : top;
                        float part[4] = {sum * exp2_approx((mx - base) * p.log2e), 0.0f, 0.0f, 0.0f};
#pragma unroll
                        for (int j = 0; j < 32; ++j) part[j & 3] += exp2_approx((__uint_as_float(r[j]) - base) * p.log2e);
                        sum = (part[0] + part[1]) + (part[2] + part[3]);
                        mx = top;
                    }
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_remote(tempty_leader + 8 * b);
                } else if constexpr (MODE == KEEP) {
                    uint32_t r[2][32];                     // 32 words at work, the next ones on their way
                    float top = -INFINITY;
                    ld32(taddr, r[0]);
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        ld_wait();
                        ld32(taddr + (c + 1) % (COLS / 32) * 32, r[(c + 1) & 1]);      // (after the last: the first again)
                        const uint32_t(&z)[32] = r[c & 1];
                        const int at = col0 + c * 32, hit = target - at, left = p.V - at;
                        if ((unsigned)hit < 32u) {
                            float v = 0.0f;
#pragma unroll
                            for (int j = 0; j < 32; ++j) v = j == hit ? __uint_as_float(z[j]) : v;
                            p.target_logit[p.t0 + row] = v;
                        }
                        if (left >= 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j) top = fmaxf(top, __uint_as_float(z[j]));
                        } else {
#pragma unroll
                            for (int j = 0; j < 32; ++j) top = j < left ? fmaxf(top, __uint_as_float(z[j])) : top;
                        }
                    }
                    const float base = top == -INFINITY ? 0.0f : top;
                    const uint64_t minus = pair2(-base, -base), scale = pair2(p.log2e, p.log2e), kept = pair2(KEPT_SCALE, KEPT_SCALE);
                    float part[4] = {0.0f, 0.0f, 0.0f, 0.0f};
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        ld_wait();
                        if (c + 1 < COLS / 32) ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
                        else {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) arrive_remote(tempty_leader + 8 * b);       // all of the tile is in registers
                        }
                        uint32_t(&z)[32] = r[c & 1];
                        const int left = p.V - (col0 + c * 32);
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            asm("{\n\t.reg .b64 a;\n\t"
                                "mov.b64 a, {%0, %1};\n\t"
                                "add.rn.f32x2 a, a, %2;\n\t"
                                "mul.rn.f32x2 a, a, %3;\n\t"
                                "mov.b64 {%0, %1}, a;\n\t"
                                "ex2.approx.ftz.f32 %0, %0;\n\tex2.approx.ftz.f32 %1, %1;\n\t}" : "+r"(z[j]), "+r"(z[j + 1]) : "l"(minus), "l"(scale));
                        if (!live || left < 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!live || j >= left) z[j] = 0u;
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) part[j & 3] += __uint_as_float(z[j]);
                        const int col = nt * N + h * COLS + c * 32;
                        if (col < p.dz_ld) {
                            uint32_t v[16];
#pragma unroll
                            for (int j = 0; j < 32; j += 2)
                                asm("{\n\t.reg .b64 a;\n\t"
                                    "mov.b64 a, {%0, %1};\n\t"
                                    "mul.rn.f32x2 a, a, %2;\n\t"
                                    "mov.b64 {%0, %1}, a;\n\t}" : "+r"(z[j]), "+r"(z[j + 1]) : "l"(kept));
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = pack2<false>(__uint_as_float(z[2 * j]), __uint_as_float(z[2 * j + 1]));
                            store32(p.dz + (int64_t)row * p.dz_ld + col, v);
                            store32(p.dz + (int64_t)row * p.dz_ld + col + 16, v + 8);
                        }
                    }
                    if (live) p.tile_max[(int64_t)(nt * 2 + h) * p.part_ld + row] = base;
                    const float best = fmaxf(mx, top), from = best == -INFINITY ? 0.0f : best;
                    sum = sum * exp2_approx((mx - from) * p.log2e) + ((part[0] + part[1]) + (part[2] + part[3])) * exp2_approx((top - from) * p.log2e);
                    mx = best;
                } else {
                    const uint64_t minus = pair2(-mx, -mx), scale = pair2(p.log2e, p.log2e), logs = pair2(-sum, -sum), rels = pair2(rel, rel);
                    uint32_t r[2][32];                     // a chunk of 32 words at work, the next one on its way
                    ld32(taddr, r[0]);
#pragma unroll
                    for (int c = 0; c < COLS / 32; ++c) {
                        ld_wait();
                        if (c + 1 < COLS / 32) ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
                        else {
                            tc_fence_before();
                            __syncwarp();
                            if (lane == 0) arrive_remote(tempty_leader + 8 * b);       // all of the tile is in registers
                        }
                        uint32_t(&z)[32] = r[c & 1];
                        const int hit = target - (col0 + c * 32), left = p.v0 + p.vc - (col0 + c * 32);      // words of the piece from here on
                        // two at a time: e^(z - lse), rounded once in the difference and once with the logarithm of the sum
#pragma unroll
                        for (int j = 0; j < 32; j += 2)
                            asm("{\n\t.reg .b64 a;\n\t"
                                "mov.b64 a, {%0, %1};\n\t"
                                "add.rn.f32x2 a, a, %2;\n\t"
                                "fma.rn.f32x2 a, a, %3, %4;\n\t"
                                "mov.b64 {%0, %1}, a;\n\t"
                                "ex2.approx.ftz.f32 %0, %0;\n\tex2.approx.ftz.f32 %1, %1;\n\t}"
                                : "+r"(z[j]), "+r"(z[j + 1]) : "l"(minus), "l"(scale), "l"(logs));
                        if ((unsigned)hit < 32u) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (j == hit) z[j] = __float_as_uint(__uint_as_float(z[j]) - 1.0f);
                        }
                        if (!BF16 || p.per_row) {
#pragma unroll
                            for (int j = 0; j < 32; j += 2)
                                asm("{\n\t.reg .b64 a;\n\t"
                                    "mov.b64 a, {%0, %1};\n\t"
                                    "mul.rn.f32x2 a, a, %2;\n\t"
                                    "mov.b64 {%0, %1}, a;\n\t}" : "+r"(z[j]), "+r"(z[j + 1]) : "l"(rels));
                        }
                        if (!live || left < 32) {
#pragma unroll
                            for (int j = 0; j < 32; ++j)
                                if (!live || j >= left) z[j] = 0u;
                        }
                        // A lane's 64 bytes as two whole sectors.  (dz has rows for whole tiles, and zeros in its last columns.)
                        const int col = nt * N + h * COLS + c * 32;
                        if (col < p.dz_ld) {
                            uint32_t v[16];
#pragma unroll
                            for (int j = 0; j < 16; ++j) v[j] = pack2<BF16>(__uint_as_float(z[2 * j]), __uint_as_float(z[2 * j + 1]));
                            if (low) {
#pragma unroll
                                for (int j = 0; j < 16; ++j) {
                                    const float2 high = unpack2<BF16>(v[j]);
                                    v[j] = pack2<BF16>(__uint_as_float(z[2 * j]) - high.x, __uint_as_float(z[2 * j + 1]) - high.y);
                                }
                            }
                            store32(p.dz + (int64_t)row * p.dz_ld + col, v);
                            store32(p.dz + (int64_t)row * p.dz_ld + col + 16, v + 8);
                        }
                    }
                }
            }
            if constexpr (MODE == STATS || MODE == KEEP) {
                // (a part holds two halves of the columns, each a warp's)
                const int across = p.parts, m_tiles = (valid + M - 1) / M;
                const int g = u / (GROUP * across), size = min(GROUP, m_tiles - g * GROUP);
                const int n = (u - g * GROUP * across) / size;
                if (alive && live) p.part[(int64_t)(n * 2 + h) * p.part_ld + row] = make_float2(mx, sum);
            }
        }
    }
    s.finish();
}

// Both gradients of a piece.  dx tiles: A = dz as stored, B = W, MN-major; fp32 sums, stored or added (the pieces run one after the other, so
// the order of a sum is always the same).  dW tiles: A = dz's transpose, B = x, both MN-major; the piece's rows of dW, complete, scaled and
// rounded, or with DW_SUMS the fp32 sums of a cut reduction.  Bound as the logits' product is (tensor cores active 84.5 % at 8192 x 32000 x 512).
struct GradMaps { CUtensorMap z_rows, z_cols, w_cols, x_cols, xg_cols, c_dx, c_dw; };

template <bool BF16, bool DW_SUMS>
__global__ void __launch_bounds__(THREADS, 1)
grads_kernel(const __grid_constant__ GradMaps maps, const Params p) {
    constexpr int STAGES = STAGES_G;
    extern __shared__ uint8_t smem_raw[];
    Setup<STAGES, C_BYTES> s(smem_raw);
    const int warp = s.warp, lane = s.lane, rank = (int)s.rank;
    const int valid = rows_of(p);
    const Schedule plan(p, valid, blockIdx.x >> 1, gridDim.x >> 1);
    bool dx;
    int u;

    if (warp == W_TMA) {
        // ------------------------------ TMA producer (both CTAs) ------------------------------
        if (lane == 0) {
            const uint32_t full_leader = mapa(s.full0, 0);
            const CUtensorMap* map_x = *p.n_valid != p.T ? &maps.xg_cols : &maps.x_cols;
            uint32_t it = 0;
            bool alive = true;
            for (int i = 0; alive && plan.at(i, dx, u); ++i) {
                const Unit w = dx ? unit_at<DX>(p, valid, u) : unit_at<DW>(p, valid, u);
                const int ma = w.m0 + 128 * rank, nb = w.n_first * N + 128 * rank;
                const CUtensorMap* map_b = dx ? &maps.w_cols : map_x;
                for (int kb = 0; kb < w.KB; ++kb, ++it) {
                    const int st = it % STAGES;
                    if (!wait(s.empty0 + 8 * st, (it / STAGES & 1) ^ 1, s.abort_flag, (11 << 8) | 2)) { alive = false; break; }
                    if (rank == 0) mbar_expect_tx(s.full0 + 8 * st, 4 * SIDE);
                    const uint32_t bar = full_leader + 8 * st, da = smem_u32(s.smem_a + st * SIDE), db = smem_u32(s.smem_b + st * SIDE);
                    const int k = (w.kb0 + kb) * KE, y = dx ? p.v0 + k : p.t0 + k;
                    if (dx) {
                        load_2d(&maps.z_rows, bar, da, k, ma);
                    } else {
                        load_2d(&maps.z_cols, bar, da, ma, k);
                        load_2d(&maps.z_cols, bar, da + SIDE / 2, ma + 64, k);
                    }
                    load_2d(map_b, bar, db, nb, y);
                    load_2d(map_b, bar, db + SIDE / 2, nb + 64, y);
                }
            }
            if (!alive) s.drain();
        }
    } else if (warp == W_MMA) {
        // ------------------------------ MMA issuer (leader; a whole warp, one elected lane) ------------------------------
        if (rank == 0) {
            constexpr uint32_t idesc_dx = make_idesc_f16(BF16, M, N, false, true), idesc_dw = make_idesc_f16(BF16, M, N, true, true);
            // K-major: a step of 16 elements is 32 bytes of the row.  MN-major: 16 rows of 128 bytes; the second 64 columns are a panel
            // of their own, SIDE / 2 bytes on (the leading offset).
            constexpr uint32_t LEAD = (SIDE / 2) >> 4;
            const uint32_t a0 = (smem_u32(s.smem_a) >> 4) & 0x3FFF, b0 = ((smem_u32(s.smem_b) >> 4) & 0x3FFF) | (LEAD << 16);
            const uint32_t tfull_own = mapa(s.tfull0, 0), tfull_peer = mapa(s.tfull0, 1);
            const uint32_t empty_own = mapa(s.empty0, 0), empty_peer = mapa(s.empty0, 1);
            uint32_t it = 0, tile = 0;
            bool alive = true;
            for (; alive && plan.at((int)tile, dx, u); ++tile) {
                const Unit w = dx ? unit_at<DX>(p, valid, u) : unit_at<DW>(p, valid, u);
                const uint32_t b = tile & 1;
                if (!wait_warp(s.tempty0 + 8 * b, (tile >> 1 & 1) ^ 1, s.abort_flag, (12 << 8) | 5)) { alive = false; break; }
                tc_fence_after();
                for (int kb = 0; kb < w.KB; ++kb, ++it) {
                    const uint32_t st = it % STAGES;
                    if (!wait_warp(s.full0 + 8 * st, it / STAGES & 1, s.abort_flag, (12 << 8) | 4)) { alive = false; break; }
                    tc_fence_after();
                    if (dx) mma_block<2, 128>(s.tmem + b * N, (a0 + st * (SIDE >> 4)) | (1u << 16), b0 + st * (SIDE >> 4), idesc_dx, kb == 0);
                    else mma_block<128, 128>(s.tmem + b * N, (a0 + st * (SIDE >> 4)) | (LEAD << 16), b0 + st * (SIDE >> 4), idesc_dw, kb == 0);
                    commit_pair(empty_own + 8 * st, empty_peer + 8 * st);
                }
                if (!alive) break;
                commit_pair(tfull_own + 8 * b, tfull_peer + 8 * b);
            }
            s.retire(tile, alive);
        }
    } else {
        // ------------------------------ epilogue (both CTAs) ------------------------------
        const int q = warp & 3, h = warp >> 2;
        const uint32_t tempty_leader = mapa(s.tempty0, 0);
        Boxes boxes(smem_u32(s.c_stage) + warp * BOXES * BOX);
        const float scale = DW_SUMS ? 1.0f : final_scale(p, BF16);
        for (int i = 0; plan.at(i, dx, u); ++i) {
            const Unit w = dx ? unit_at<DX>(p, valid, u) : unit_at<DW>(p, valid, u);
            const uint32_t b = i & 1;
            if (!wait_warp(s.tfull0 + 8 * b, i >> 1 & 1, s.abort_flag, (13 << 8) | 3)) break;
            tc_fence_after();
            const uint32_t taddr = s.tmem + ((uint32_t)(q * 32) << 16) + b * N + h * COLS;
            const int row = w.m0 + 128 * rank + q * 32, col0 = w.n_first * N + h * COLS;
            const bool sums = dx || DW_SUMS;
            uint32_t box = 0, r[2][32];                    // 32 columns at work, the next ones on their way
            ld32(taddr, r[0]);
#pragma unroll
            for (int c = 0; c < COLS / 32; ++c) {
                ld_wait();
                if (c + 1 < COLS / 32) ld32(taddr + (c + 1) * 32, r[(c + 1) & 1]);
                else {
                    tc_fence_before();
                    __syncwarp();
                    if (lane == 0) arrive_remote(tempty_leader + 8 * b);       // all of the tile is in registers
                }
                uint32_t(&v)[32] = r[c & 1];
                if (!w.KB) {                               // nothing to sum: no product either
#pragma unroll
                    for (int j = 0; j < 32; ++j) v[j] = 0u;
                }
                if (sums) {                                // a box: 32 columns
                    box = boxes.open(lane);
#pragma unroll
                    for (int j = 0; j < 8; ++j) stage16(box, lane, j, v[4 * j], v[4 * j + 1], v[4 * j + 2], v[4 * j + 3]);
                    const int col = col0 + c * 32;
                    if (dx) boxes.send(lane, &maps.c_dx, col, w.split * p.dx_rows + p.t0 + row, col < p.d, p.add_dx);
                    else boxes.send(lane, &maps.c_dw, col, w.split * p.dw_rows + row, col < p.d, p.add_dw);
                } else {                                   // 64 columns
                    if ((c & 1) == 0) box = boxes.open(lane);
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        uint32_t o[4];
#pragma unroll
                        for (int k = 0; k < 4; ++k) o[k] = pack2<BF16>(__uint_as_float(v[j * 8 + 2 * k]) * scale, __uint_as_float(v[j * 8 + 2 * k + 1]) * scale);
                        stage16(box, lane, (c & 1) * 4 + j, w.KB ? o[0] : 0u, w.KB ? o[1] : 0u, w.KB ? o[2] : 0u, w.KB ? o[3] : 0u);
                    }
                    if (c & 1) {
                        const int col = col0 + (c >> 1) * 64;
                        boxes.send(lane, &maps.c_dw, col, p.v0 + row, col < p.d && p.v0 + row < p.V, false);
                    }
                }
            }
        }
        boxes.drain(lane);
    }
    s.finish();
}

// ---------------------------------------------------------------------------------------------------------------------
// rows in use
// ---------------------------------------------------------------------------------------------------------------------
struct State {                             // what the forward leaves for the backward (one allocation of the caller's)
    int* n_valid;                          // [0] rows in use, [1] a ticket of the pass that adds up the losses
    int* rows;                             // the token of every row in use
    int* slot;                             // the row of every token; -1: ignored, -2: a target that is no word
    int* target;                           // per row in use
    float2* stat;                          // per row: maximum and log2 of the sum
};

__device__ __forceinline__ int slot_kind(int64_t t, int64_t ignore, int V) { return t == ignore ? -1 : (t < 0 || t >= V) ? -2 : 0; }

__global__ void __launch_bounds__(SCAN)
count_kernel(const int64_t* __restrict__ target, int T, int64_t ignore, int V, int* __restrict__ counts) {
    pdl_wait();
    pdl_trigger();
    const int t = blockIdx.x * SCAN + threadIdx.x;
    const int n = __syncthreads_count(t < T && slot_kind(target[t < T ? t : 0], ignore, V) == 0);
    if (threadIdx.x == 0) counts[blockIdx.x] = n;
}

// counts: of all blocks
__global__ void __launch_bounds__(SCAN)
place_kernel(const int64_t* __restrict__ target, int T, int64_t ignore, int V, const int* __restrict__ counts, State s) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_warp[32], s_base;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * SCAN + threadIdx.x;
    int before = 0;
    for (int b = threadIdx.x; b < (int)blockIdx.x; b += SCAN) before += counts[b];
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) before += __shfl_xor_sync(0xffffffffu, before, o);
    if (lane == 0) s_warp[warp] = before;
    __syncthreads();
    if (threadIdx.x == 0) {
        int sum = 0;
        for (int w = 0; w < 32; ++w) sum += s_warp[w];
        s_base = sum;
    }
    __syncthreads();
    before = s_base;
    const int64_t goal = t < T ? target[t] : ignore;
    const int kind = t < T ? slot_kind(goal, ignore, V) : -1;
    const unsigned has = __ballot_sync(0xffffffffu, kind == 0);
    if (lane == 0) s_warp[warp] = __popc(has);
    __syncthreads();
    int in_block = 0;
    for (int w = 0; w < warp; ++w) in_block += s_warp[w];
    const int row = before + in_block + __popc(has & ((1u << lane) - 1u));
    if (t < T) s.slot[t] = kind == 0 ? row : kind;
    if (kind == 0) { s.rows[row] = t; s.target[row] = (int)goal; }
    if (blockIdx.x == gridDim.x - 1 && threadIdx.x == SCAN - 1) {
        s.n_valid[0] = row + (kind == 0);
        s.n_valid[1] = 0;
    }
}

// x's rows in use, one after the other, and zeros up to a whole K block behind them (dz^T x reduces over rows: nothing else may
// stand there).  Where every token is in use nothing is copied: x itself is read.  half: the rows once more from that one on, zeros between.
__global__ void __launch_bounds__(256)
gather_kernel(const uint4* __restrict__ x, int64_t ld, int T, int vecs, const int* __restrict__ n_valid, const int* __restrict__ rows,
              uint4* __restrict__ out, int half) {
    pdl_wait();
    pdl_trigger();
    const int valid = *n_valid;
    if (valid == T && !half) return;
    const int padded = (valid + (valid ? half : 0) + KE - 1) / KE * KE;
    const int64_t n = (int64_t)padded * vecs;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / vecs), c = (int)(i - (int64_t)r * vecs);
        const int own = half && r >= half ? r - half : r;
        out[i] = own < valid ? x[(int64_t)rows[own] * ld + c] : make_uint4(0, 0, 0, 0);
    }
}

// The three passes above in one, for up to SMALL tokens: every CTA places all of them for itself, the first one writes it down, and each gathers the
// rows of every gridDim.x-th token: one or two launches less (130 tokens of 512 to 32000 words in training 89 -> 84 us, host and all).
constexpr int SMALL = 4096;

__global__ void __launch_bounds__(SCAN)
place_gather_kernel(const int64_t* __restrict__ target, int T, int64_t ignore, int V, State s, const uint4* __restrict__ x, int64_t ld, int vecs,
                    uint4* __restrict__ out) {
    pdl_wait();
    pdl_trigger();
    __shared__ int s_warp[32], s_row[SMALL];                 // the rows of this CTA's tokens
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, G = gridDim.x, me = blockIdx.x;
    int valid = 0;
    for (int base = 0; base < T; base += SCAN) {
        const int t = base + threadIdx.x;
        const int64_t goal = t < T ? target[t] : ignore;
        const int kind = t < T ? slot_kind(goal, ignore, V) : -1;
        const unsigned has = __ballot_sync(0xffffffffu, kind == 0);
        __syncthreads();
        if (lane == 0) s_warp[warp] = __popc(has);
        __syncthreads();
        int before = 0, all = 0;
#pragma unroll
        for (int w = 0; w < 32; ++w) {
            before += w < warp ? s_warp[w] : 0;
            all += s_warp[w];
        }
        const int row = valid + before + __popc(has & ((1u << lane) - 1u));
        if (me == 0) {
            if (t < T) s.slot[t] = kind == 0 ? row : kind;
            if (kind == 0) { s.rows[row] = t; s.target[row] = (int)goal; }
        }
        if (t < T && t % G == me) s_row[t / G] = kind == 0 ? row : -1;
        valid += all;
    }
    if (me == 0 && threadIdx.x == 0) { s.n_valid[0] = valid; s.n_valid[1] = 0; }
    if (valid == T) return;
    __syncthreads();
    const int mine = me < T ? (T - me + G - 1) / G : 0;
    for (int i = warp; i < mine; i += 32) {
        const int row = s_row[i];
        if (row < 0) continue;
        const uint4* from = x + (int64_t)(me + i * G) * ld;
        for (int c = lane; c < vecs; c += 32) out[(int64_t)row * vecs + c] = from[c];
    }
    const int padded = (valid + KE - 1) / KE * KE;
    for (int row = valid + me; row < padded; row += G)
        for (int c = threadIdx.x; c < vecs; c += SCAN) out[(int64_t)row * vecs + c] = make_uint4(0, 0, 0, 0);
}

// ---------------------------------------------------------------------------------------------------------------------
// loss
// ---------------------------------------------------------------------------------------------------------------------
constexpr int JOIN = 16;                   // warps of a block: each joins every JOINth run of the same 32 tokens

// Per token: the runs' maxima and sums joined, always in the same order; the loss; and for a sum or mean the blocks' sums, added up in 64
// bits and in their order by the block that comes last.  (One thread for all of a token's runs: 70 us for 130 tokens of 250 runs, which are
// read one after the other.)
//
// The tensor cores cut off what a step of 16 products leaves below the running sum's last bit, which puts a logit off by up to d / 16 such bits, towards zero.
// Among the other words most of that averages out; the target's logit is the one that a loss hangs on.  So it is multiplied once more in plain fp32, and its
// term in the sum exchanged for that: loss = log(1 + sum of the others e^(z - z_target)).  Relative errors for 5000 words: one token of 512 up to
// 1.2e-5 -> 3.1e-7, 200 of 2048 8e-7 -> 2.2e-7, and with growth 7e-8; of 7168 2.8e-6 -> 2.4e-6, and with growth 3e-7; 1531 tokens of 512 to 32000 words scored 53.5 -> 54.6 us.
template <bool BF16>
__global__ void __launch_bounds__(32 * JOIN)
loss_kernel(const float2* __restrict__ part, int64_t part_ld, int parts, const float* __restrict__ target_logit, State s, int T, int reduction,
            double* __restrict__ block_sum, float* __restrict__ loss, int t0, int tc, int last, const uint4* __restrict__ x, int64_t ldx,
            const uint4* __restrict__ w, int64_t ldw, int vecs, float grown) {
    const float log2e = LOG2E * grown;
    pdl_wait();
    pdl_trigger();
    __shared__ float2 s_part[JOIN][32];
    __shared__ double s_sum[JOIN];
    __shared__ float s_logit[32];
    __shared__ bool s_last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, t = blockIdx.x * 32 + lane;
    const int slot = t < T ? s.slot[t] : -1, row = slot >= t0 && slot - t0 < tc ? slot : -1;       // (of this piece)
    float mx = -INFINITY, sum = 0.0f;
    auto join = [&](float2 v) {
        const float top = fmaxf(mx, v.x), base = top == -INFINITY ? 0.0f : top;
        sum = sum * exp2f((mx - base) * log2e) + v.y * exp2f((v.x - base) * log2e);
        mx = top;
    };
    if (row >= 0) {
#pragma unroll 4
        for (int i = warp; i < parts; i += JOIN) join(part[(int64_t)i * part_ld + row - t0]);
    }
    s_part[warp][lane] = make_float2(mx, sum);
    for (int i = warp; i < 32; i += JOIN) {                // a warp a token
        const int at = __shfl_sync(0xffffffffu, row, i);
        if (at < 0) continue;
        const uint4 *a = x + (int64_t)(blockIdx.x * 32 + i) * ldx, *b = w + (int64_t)s.target[at] * ldw;
        float z = 0.0f;
        for (int c = lane; c < vecs; c += 32) {
            const uint4 u = a[c], v = b[c];
            const uint32_t ua[4] = {u.x, u.y, u.z, u.w}, va[4] = {v.x, v.y, v.z, v.w};
            float eight = 0.0f;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const float2 p = unpack2<BF16>(ua[j]), q = unpack2<BF16>(va[j]);
                eight = fmaf(p.x, q.x, fmaf(p.y, q.y, eight));
            }
            z += eight;
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) z += __shfl_xor_sync(0xffffffffu, z, o);
        if (lane == 0) s_logit[i] = z;
    }
    __syncthreads();
    double mine = 0.0;
    if (warp == 0 && t < T) {
        float l = slot == -2 && t0 == 0 ? NAN : 0.0f;
        if (row >= 0) {
#pragma unroll
            for (int w = 1; w < JOIN; ++w) join(s_part[w][lane]);
            s.stat[row] = make_float2(mx, log2f(sum));
            float others = sum - exp2f((target_logit[row] - mx) * log2e);      // (the term as it was added: exact where it is the largest)
            others = others < 0.0f ? 0.0f : others;
            const float over = mx * grown - s_logit[lane];
            l = over > 0.0f ? over + logf(others + exp2f(-over * LOG2E)) : log1pf(others * exp2f(over * LOG2E));
        }
        if (reduction == 0) loss[t] = l;
        mine = l;
    }
    if (reduction == 0) return;
    auto warp_total = [](double v) {
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
        return v;
    };
    if (warp == 0) {
        mine = warp_total(mine);
        if (lane == 0) {
            if (t0) mine += block_sum[blockIdx.x];           // of earlier pieces
            block_sum[blockIdx.x] = mine;
            __threadfence();
            s_last = last && atomicAdd(&s.n_valid[1], 1) == (int)gridDim.x - 1;
        }
    }
    __syncthreads();
    if (!s_last) return;
    __threadfence();
    mine = 0.0;
    for (int b = threadIdx.x; b < (int)gridDim.x; b += 32 * JOIN) mine += __ldcg(block_sum + b);
    mine = warp_total(mine);
    if (lane == 0) s_sum[warp] = mine;
    __syncthreads();
    if (threadIdx.x == 0) {
        double total = 0.0;
        for (int w = 0; w < JOIN; ++w) total += s_sum[w];
        *loss = (float)(reduction == 1 ? total / (double)s.n_valid[0] : total);
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// gradients: what is left around the products
// ---------------------------------------------------------------------------------------------------------------------
// What KEEP left, turned into dz in its place: e^(z - m) e^(m - lse) - [the target], m the maximum of the 128 words.  A warp a row, 256 words at a time; bound by
// reading and writing them.  Where the target is the likeliest word, its e^0 is exact, and so 1 - p keeps the bits of p's fp32.
template <bool BF16>
__global__ void __launch_bounds__(256)
soften_kernel(const Params p) {
    pdl_wait();
    pdl_trigger();
    const int lane = threadIdx.x & 31, valid = rows_of(p), vecs = p.dz_ld / 8;
    const int per = (vecs + 31) / 32;                      // turns of a row
    for (int64_t i = (int64_t)blockIdx.x * 8 + (threadIdx.x >> 5); i < (int64_t)valid * per; i += (int64_t)gridDim.x * 8) {
        const int row = (int)(i / per), at = (int)(i - (int64_t)row * per) * 32 + lane;
        if (at >= vecs) continue;
        const float2 st = p.stat[p.t0 + row];
        const float f = exp2_approx((p.tile_max[(int64_t)(at / 16) * p.part_ld + row] - st.x) * p.log2e - st.y) * (1.0f / KEPT_SCALE);
        uint4* q = reinterpret_cast<uint4*>(p.dz + (int64_t)row * p.dz_ld) + at;
        uint4 v = *q;
        uint32_t* h = &v.x;
        const int hit = p.target[p.t0 + row] - at * 8;
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 e = __half22float2(*reinterpret_cast<const __half2*>(&h[j]));
            e.x = e.x * f - (hit == 2 * j ? 1.0f : 0.0f);
            e.y = e.y * f - (hit == 2 * j + 1 ? 1.0f : 0.0f);
            h[j] = BF16 ? pack2<true>(e.x, e.y) : pack2<false>(e.x * FP16_SCALE, e.y * FP16_SCALE);
        }
        *q = v;
    }
}

// the largest finite |gradient| among the tokens in use, as bits; *out starts at 0.  (An infinity or NaN is its own token's affair: related to one, every
// other token's gradient would be 0 times infinity.)
__global__ void __launch_bounds__(256)
grad_max_kernel(const float* __restrict__ grad, const int* __restrict__ slot, int T, unsigned* __restrict__ out) {
    pdl_wait();
    pdl_trigger();
    unsigned most = 0;
    for (int t = blockIdx.x * 256 + threadIdx.x; t < T; t += gridDim.x * 256)
        if (slot[t] >= 0 && fabsf(grad[t]) < INFINITY) most = max(most, __float_as_uint(fabsf(grad[t])));
    most = __reduce_max_sync(0xffffffffu, most);
    if ((threadIdx.x & 31) == 0 && most) atomicMax(out, most);
}

// out[r] = scale * sum of the splits' sums of r's row (and of the row `half` further on), rounded once; slot (null: every row its own) -1 or -2:
// zeros.  Eight columns a thread.
template <bool BF16>
__global__ void __launch_bounds__(256)
finish_kernel(const float* __restrict__ sums, int splits, int64_t split_elems, int rows, int d, const int* __restrict__ slot, const Params p,
              uint4* __restrict__ out) {
    pdl_wait();
    pdl_trigger();
    const int vecs = d / 8;
    const int64_t n = (int64_t)rows * vecs;
    const float scale = final_scale(p, BF16);
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        const int r = (int)(i / vecs), c = (int)(i - (int64_t)r * vecs);
        const int from = slot ? slot[r] : r;
        float a[8] = {};
        if (from >= 0) {
            const float* first = sums + (int64_t)from * d + c * 8;
            for (int s = 0; s < splits * (slot && p.half ? 2 : 1); ++s) {
                const float* at = first + (s >= splits ? (int64_t)p.half * d + (s - splits) * split_elems : s * split_elems);
                const float4 u = __ldcs(reinterpret_cast<const float4*>(at)), v = __ldcs(reinterpret_cast<const float4*>(at) + 1);
                a[0] += u.x; a[1] += u.y; a[2] += u.z; a[3] += u.w;
                a[4] += v.x; a[5] += v.y; a[6] += v.z; a[7] += v.w;
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) a[j] *= scale;
        }
        out[i] = make_uint4(pack2<BF16>(a[0], a[1]), pack2<BF16>(a[2], a[3]), pack2<BF16>(a[4], a[5]), pack2<BF16>(a[6], a[7]));
    }
}

// ---------------------------------------------------------------------------------------------------------------------
// plans
// ---------------------------------------------------------------------------------------------------------------------
static inline int64_t up(int64_t v, int64_t a) { return (v + a - 1) / a * a; }
static inline int64_t ceil_div(int64_t a, int64_t b) { return (a + b - 1) / b; }

struct Plan {
    int64_t T, V, d, Tp;                   // Tp: T in whole tiles
    int clusters, parts;
    int64_t vc;                            // words of a piece
    int pieces, dx_splits, dw_splits;
    int64_t dz_ld;
    bool early;
    int64_t tc;                            // early: tokens of a piece
    int64_t half;                          // late: see FEW
};

constexpr int64_t PART_BYTES = 48LL << 20;
constexpr int64_t DZ_BYTES = 512LL << 20;  // most of a piece of dz: smaller pieces cost passes over dx, larger ones only memory (32768 tokens x 512 to 32000 words
                                           // with 128 MiB 5.0 ms, 256 3.92, 512 3.89, 1024 3.85, 2048 3.87)

// Up to FEW tokens, dz stands in two parts, rounded and what the rounding left, in rows of their own: a tile has 256 anyway, x's rows stand twice behind
// one another, and dW sums over twice as many.  Where a gradient is made of a few tokens, each one's dz is a factor of all that it adds and its rounding
// does not average out: with targets of probability 0.47 dW was off by up to 0.32 % in bf16 where its own rounding is 0.17 % (1 token; 0.25 % with 20), and
// is now at its own rounding.  32 tokens x 512 to 32000 words 43 -> 47 us, 128 x 2048 to 128000 428 -> 464, 100 x 4096 852 -> 937.
constexpr int64_t FEW = 128;
constexpr int64_t EARLY_BYTES = 5LL << 28; // the same of a piece of tokens: beyond the first one dW is added to, in memory
constexpr int64_t EARLY_TOKENS = 2048, EARLY_WIDTH = 1024;               // see early_pays
constexpr int64_t EARLY_KEPT = 8LL << 30;  // most of what the early way leaves for the backward

static Plan make_plan(int64_t T, int64_t V, int64_t d, bool early) {
    Plan r{};
    r.T = T; r.V = V; r.d = d; r.Tp = up(T, M); r.early = early;
    r.clusters = std::max(1, sm_count() / 2);          // (not those under a cap: sizes must not change between two calls)
    const int64_t n_tiles = ceil_div(V, N), n_d = ceil_div(d, N);
    // reductions cut where their tiles would leave SMs idle, down to 16 K blocks a piece
    auto cut = [&](int64_t tiles, int64_t blocks) {
        return (int)std::max<int64_t>(1, std::min<int64_t>({(int64_t)r.clusters / std::max<int64_t>(1, tiles), blocks / 16, (int64_t)16}));
    };
    if (early) {
        r.dz_ld = up(V, KE);
        const int64_t fit = std::max<int64_t>(M, EARLY_BYTES / (2 * r.dz_ld) / M * M);
        r.pieces = (int)ceil_div(r.Tp, fit);
        r.tc = up(ceil_div(r.Tp, r.pieces), M);        // equal pieces, in whole tiles
        r.pieces = (int)ceil_div(r.Tp, r.tc);
        r.vc = V;
        r.dx_splits = cut(r.tc / M * n_d, ceil_div(V, KE));
        r.dw_splits = r.pieces > 1 ? 1 : cut(n_tiles * n_d, ceil_div(T, KE));
    } else {
        const int64_t fit = std::max<int64_t>(N, DZ_BYTES / (2 * r.Tp) / N * N);
        r.pieces = (int)ceil_div(V, fit);
        r.vc = up(ceil_div(V, r.pieces), N);
        r.pieces = (int)ceil_div(V, r.vc);
        r.dz_ld = up(std::min(r.vc, V), KE);
        r.tc = r.Tp;
        r.half = T <= FEW ? up(T, 32) : 0;
        r.dx_splits = cut(r.Tp / M * n_d, ceil_div(std::min(r.vc, V), KE));
        r.dw_splits = r.pieces > 1 ? 1 : cut(n_tiles * n_d, ceil_div(T + r.half, KE));
    }
    // runs of words: one tile each, for an even end, unless what they leave per token is more than PART_BYTES
    r.parts = (int)ceil_div(n_tiles, ceil_div(16 * n_tiles * r.tc, PART_BYTES));
    return r;
}

static int64_t dx_sums_bytes(const Plan& r) { return 4 * r.dx_splits * r.Tp * r.d; }
static int64_t dw_sums_bytes(const Plan& r) { return 4 * r.dw_splits * up(r.V, M) * r.d; }
// Whether both gradients of a sum or mean are made in the forward.  That saves a product, which goes with d, and costs a pass over the piece and
// an epilogue that reads its tile twice, which do not, and 10 bytes of sums for each element of dW, which does not go with the tokens.  us
// late and early, in bf16: 8192 tokens x 512 to 32000 words 970 and 1060, 768 1400 and 1370, 1024 1810 and 1700, 2048 3440 and 3050; 1024 tokens x 2048
// 490 and 513, 1536 697 and 676, 2048 891 and 847; 2048 x 4096 to 128000 6870 and 6490, 16384 x 2048 to 128000 27.5 and 24.7 ms.
static bool early_pays(int64_t T, int64_t V, int64_t d, int reduction) {
    if (reduction == 0 || T < EARLY_TOKENS || d < EARLY_WIDTH) return false;
    const Plan r = make_plan(T, V, d, true);
    return dx_sums_bytes(r) + dw_sums_bytes(r) <= EARLY_KEPT;
}

struct Carver {                            // sub-allocations of one workspace, 256 bytes apart
    uint8_t* base;
    int64_t used = 0;
    void* take(int64_t bytes) { void* at = base ? base + used : nullptr; used += up(bytes, 256); return at; }
};

static State carve_state(void* mem, int64_t T, int64_t* bytes) {
    Carver c{static_cast<uint8_t*>(mem)};
    State s;
    s.n_valid = static_cast<int*>(c.take(8));
    s.rows = static_cast<int*>(c.take(4 * T));
    s.slot = static_cast<int*>(c.take(4 * T));
    s.target = static_cast<int*>(c.take(4 * T));
    s.stat = static_cast<float2*>(c.take(8 * T));
    if (bytes) *bytes = c.used;
    return s;
}

struct Forward { int* counts; void* xg; float2* part; float* target_logit; double* block_sum; void* dz; float* tile_max; };
static Forward carve_forward(void* mem, const Plan& r, int64_t* bytes) {
    Carver c{static_cast<uint8_t*>(mem)};
    Forward f;
    f.counts = static_cast<int*>(c.take(4 * ceil_div(r.T, SCAN)));
    f.xg = c.take(up(r.T, KE) * r.d * 2);
    f.part = static_cast<float2*>(c.take(8LL * 2 * r.parts * r.tc));
    f.target_logit = static_cast<float*>(c.take(4 * r.T));
    f.block_sum = static_cast<double*>(c.take(8 * ceil_div(r.T, 32)));
    f.dz = c.take(r.early ? r.tc * r.dz_ld * 2 : 0);
    f.tile_max = static_cast<float*>(c.take(r.early ? 4 * 2 * ceil_div(r.V, N) * r.tc : 0));
    if (bytes) *bytes = c.used;
    return f;
}
static int64_t gathered_rows(const Plan& r) { return r.half ? 2 * r.half : up(r.T, KE); }      // (of the late backward)
struct Backward { void *xg, *dz; float *dx, *dw; unsigned* grad_max; };
static Backward carve_backward(void* mem, const Plan& r, bool want_dx, bool want_dw, int64_t* bytes) {
    Carver c{static_cast<uint8_t*>(mem)};
    Backward b;
    b.grad_max = static_cast<unsigned*>(c.take(4));
    b.xg = c.take(gathered_rows(r) * r.d * 2);
    b.dz = c.take(r.Tp * r.dz_ld * 2);
    b.dx = static_cast<float*>(c.take(want_dx ? dx_sums_bytes(r) : 0));
    b.dw = static_cast<float*>(c.take(want_dw && r.dw_splits > 1 ? dw_sums_bytes(r) : 0));
    if (bytes) *bytes = c.used;
    return b;
}

// What a logit z = x w has lost on its way through tensor memory is made good for by as much as it loses on average.  A step of 16 products cuts the running
// sum off below its last bit: half such a bit, about 0.36 2^-23 of the sum (mantissas spread as logarithms are); and after k of K steps the sum is z k / K
// on average, whatever the order.  That makes 0.36 K 2^-24 of z.  Measured, in units of K 2^-24, d from 256 to 7168: bf16 0.25 to 0.28 for the words that a
// softmax is made of, 0.29 to 0.42 for z of 12 to 30, scattered by a tenth of that; fp16 0.3 and, its products having more bits to lose, 0.5 to 1.1.
// Those are operands with normally distributed elements.  Where nothing is cut off (few non-zeros in a row, or a coarse grid) the factor is itself the error: at d =
// 7168 it is 8e-6 of a logit, 2.4e-4 of the loss where logits are 30.  It stays below the bound of any fp32 sum of d / 16 steps, d / 16 2^-24.
static float growth(int64_t d) { return 1.0f + 0.3f * (float)(d / 16) * 0x1p-24f; }

template <auto KERN, size_t SMEM_BYTES, typename... A>
static int launch(cudaStream_t st, A&&... args) {
    int rc = allow_smem_once<KERN>(SMEM_BYTES);
    if (rc) return rc;
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3(2 * std::max(1, gemm_sm_count() / 2)); cfg.blockDim = dim3(THREADS); cfg.dynamicSmemBytes = SMEM_BYTES; cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = 2; attr[0].val.clusterDim.y = 1; attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr; cfg.numAttrs = 2;
    CINN_CHECK_CUDA(cudaLaunchKernelEx(&cfg, KERN, args...));
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

static int map16(CUtensorMap* m, const void* base, int64_t inner, int64_t rows, int64_t ld, int box_rows, bool bf16) {
    return encode_map_2d(m, base, (uint64_t)inner, (uint64_t)rows, (uint64_t)ld * 2, 64, (uint32_t)box_rows,
                         bf16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, CU_TENSOR_MAP_SWIZZLE_128B);
}

static int map_sums(CUtensorMap* m, float* base, int64_t rows, int64_t d) {
    return encode_map_2d(m, base, (uint64_t)d, (uint64_t)rows, (uint64_t)d * 4, 32, 32, CU_TENSOR_MAP_DATA_TYPE_FLOAT32, CU_TENSOR_MAP_SWIZZLE_128B);
}

static unsigned grid_for(int64_t items, int64_t per_block) { return (unsigned)std::max<int64_t>(1, std::min<int64_t>(ceil_div(items, per_block), 8LL * sm_count())); }

static int check_shapes(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, int64_t T, int64_t V, int64_t d, int reduction) {
    CINN_CHECK_ARG(dtype == CINN_BF16 || dtype == CINN_F16, "linear_ce: operands are bf16 or fp16 (dtype tag %d)", dtype);
    CINN_CHECK_ARG(T >= 0 && V >= 1 && d >= 1, "linear_ce: bad shape");
    CINN_CHECK_ARG(T <= (1LL << 30) && V <= (1LL << 30) && d <= (1LL << 24) && (T / 256 + 1) * (V / 256 + 1) < (1LL << 31),
                   "linear_ce: dimension too large");
    CINN_CHECK_ARG(reduction >= 0 && reduction <= 2, "linear_ce: reduction %d (0 none, 1 mean, 2 sum)", reduction);
    CINN_CHECK_ARG(d % 8 == 0 && ldx % 8 == 0 && ldw % 8 == 0 && ldx >= d && ldw >= d,
                   "linear_ce: the row length (%lld) and pitches (%lld, %lld) must be multiples of 8 elements", (long long)d, (long long)ldx, (long long)ldw);
    CINN_CHECK_ARG(T == 0 || (x && w), "linear_ce: null pointer");
    CINN_CHECK_ARG(((reinterpret_cast<uintptr_t>(x) | reinterpret_cast<uintptr_t>(w)) & 15) == 0, "linear_ce: operands must be 16-byte aligned");
    return CINN_OK;
}

// store32 writes pieces of 32 bytes into the workspace (whose parts lie 256 bytes apart); the state's widest elements are of 8
static int check_scratch(const void* state, const void* workspace) {
    CINN_CHECK_ARG((reinterpret_cast<uintptr_t>(workspace) & 31) == 0 && (reinterpret_cast<uintptr_t>(state) & 7) == 0,
                   "linear_ce: the workspace must be 32-byte aligned and the state 8-byte aligned");
    return CINN_OK;
}

static int gather(const void* x, int64_t ldx, const Plan& r, const State& s, void* xg, int64_t half, cudaStream_t st) {
    launch_dependent(gather_kernel, dim3(grid_for((half + r.T) * (r.d / 8), 256)), dim3(256), 0, st, static_cast<const uint4*>(x), ldx / 8,
                     (int)r.T, (int)(r.d / 8), s.n_valid, s.rows, static_cast<uint4*>(xg), (int)half);
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

template <bool BF16>
static int forward(const void* x, int64_t ldx, const void* w, int64_t ldw, const int64_t* target, int64_t ignore, const Plan& r, int reduction,
                   float* loss, const State& s, const Forward& f, float* dx_sums, float* dw_sums, cudaStream_t st) {
    const int blocks = (int)ceil_div(r.T, SCAN);
    int rc = CINN_OK;
    if (r.T <= SMALL) {
        launch_dependent(place_gather_kernel, dim3((unsigned)std::min<int64_t>(r.T, sm_count())), dim3(SCAN), 0, st, target, (int)r.T, ignore, (int)r.V, s,
                         static_cast<const uint4*>(x), ldx / 8, (int)(r.d / 8), static_cast<uint4*>(f.xg));
        CINN_CHECK_LAUNCH();
    } else {
        launch_dependent(count_kernel, dim3(blocks), dim3(SCAN), 0, st, target, (int)r.T, ignore, (int)r.V, f.counts);
        CINN_CHECK_LAUNCH();
        launch_dependent(place_kernel, dim3(blocks), dim3(SCAN), 0, st, target, (int)r.T, ignore, (int)r.V, f.counts, s);
        CINN_CHECK_LAUNCH();
        if ((rc = gather(x, ldx, r, s, f.xg, 0, st))) return rc;
    }
    CUtensorMap ta, tb, tx;
    if ((rc = map16(&ta, x, r.d, r.T, ldx, 128, BF16))) return rc;
    if ((rc = map16(&tx, f.xg, r.d, up(r.T, KE), r.d, 128, BF16))) return rc;
    if ((rc = map16(&tb, w, r.d, r.V, ldw, 128, BF16))) return rc;
    Params p{};
    p.n_valid = s.n_valid; p.T = (int)r.T; p.V = (int)r.V; p.d = (int)r.d; p.vc = (int)r.V; p.tc = (int)r.tc; p.parts = r.parts;
    p.log2e = LOG2E * growth(r.d);
    p.part = f.part; p.part_ld = r.tc; p.target_logit = f.target_logit; p.target = s.target; p.stat = s.stat;
    auto join = [&](int last) {
        launch_dependent(loss_kernel<BF16>, dim3((unsigned)ceil_div(r.T, 32)), dim3(32 * JOIN), 0, st, f.part, r.tc, 2 * r.parts, f.target_logit, s, (int)r.T,
                         reduction, f.block_sum, loss, p.t0, p.tc, last, static_cast<const uint4*>(x), ldx / 8, static_cast<const uint4*>(w), ldw / 8,
                         (int)(r.d / 8), growth(r.d));
        CINN_CHECK_LAUNCH();
        return (int)CINN_OK;
    };
    if (!r.early) {
        if ((rc = launch<product_kernel<STATS, BF16>, SMEM_Z>(st, ta, tb, tx, p))) return rc;
        return join(1);
    }
    GradMaps g;
    if ((rc = map16(&g.x_cols, x, r.d, r.T, ldx, 64, BF16))) return rc;
    if ((rc = map16(&g.xg_cols, f.xg, r.d, up(r.T, KE), r.d, 64, BF16))) return rc;
    if ((rc = map16(&g.w_cols, w, r.d, r.V, ldw, 64, BF16))) return rc;
    if ((rc = map16(&g.z_rows, f.dz, r.V, r.tc, r.dz_ld, 128, BF16))) return rc;
    if ((rc = map16(&g.z_cols, f.dz, r.V, r.tc, r.dz_ld, 64, BF16))) return rc;
    g.c_dx = g.c_dw = g.x_cols;            // (one that is not wanted is not used)
    if (dx_sums && (rc = map_sums(&g.c_dx, dx_sums, r.dx_splits * r.Tp, r.d))) return rc;
    if (dw_sums && (rc = map_sums(&g.c_dw, dw_sums, r.dw_splits * up(r.V, M), r.d))) return rc;
    p.dz = static_cast<uint16_t*>(f.dz); p.dz_ld = (int)r.dz_ld; p.tile_max = f.tile_max;
    p.dx_splits = dx_sums ? r.dx_splits : 0; p.dx_rows = (int)r.Tp;
    p.dw_splits = dw_sums ? r.dw_splits : 0; p.dw_rows = (int)up(r.V, M);
    for (int i = 0; i < r.pieces; ++i) {
        p.t0 = (int)(i * r.tc);
        p.add_dw = i > 0;
        if ((rc = launch<product_kernel<KEEP, BF16>, SMEM_Z>(st, ta, tb, tx, p))) return rc;
        if ((rc = join(i + 1 == r.pieces))) return rc;
        launch_dependent(soften_kernel<BF16>, dim3((unsigned)(8 * sm_count())), dim3(256), 0, st, p);
        CINN_CHECK_LAUNCH();
        if ((rc = launch<grads_kernel<BF16, true>, SMEM_G>(st, g, p))) return rc;
    }
    return CINN_OK;
}

template <bool BF16>
static int finish(const float* sums, int splits, int64_t split_rows, int64_t rows, int64_t d, const int* slot, const Params& p, void* out, cudaStream_t st) {
    launch_dependent(finish_kernel<BF16>, dim3(grid_for(rows * (d / 8), 256)), dim3(256), 0, st, sums, splits, split_rows * d, (int)rows, (int)d, slot, p,
                     static_cast<uint4*>(out));
    CINN_CHECK_LAUNCH();
    return CINN_OK;
}

template <bool BF16>
static int backward(const void* x, int64_t ldx, const void* w, int64_t ldw, const float* grad, const Plan& r, int reduction, const State& s,
                    void* dx, void* dw, const Backward& b, cudaStream_t st) {
    int rc = gather(x, ldx, r, s, b.xg, r.half, st);
    if (rc) return rc;
    Params p{};
    p.n_valid = s.n_valid; p.T = r.half ? -1 : (int)r.T; p.V = (int)r.V; p.d = (int)r.d; p.tc = (int)r.Tp; p.half = (int)r.half;
    p.target = s.target; p.rows = s.rows; p.stat = s.stat; p.grad = grad; p.grad_max = b.grad_max;
    p.per_row = reduction == 0; p.mean = reduction == 1; p.log2e = LOG2E * growth(r.d);
    if (p.per_row) {
        CINN_CHECK_CUDA(cudaMemsetAsync(b.grad_max, 0, 4, st));
        launch_dependent(grad_max_kernel, dim3(grid_for(r.T, 1024)), dim3(256), 0, st, grad, s.slot, (int)r.T, b.grad_max);
        CINN_CHECK_LAUNCH();
    }
    CUtensorMap x_rows, xg_rows, w_rows;
    GradMaps g;
    if ((rc = map16(&x_rows, x, r.d, r.T, ldx, 128, BF16))) return rc;
    if ((rc = map16(&xg_rows, b.xg, r.d, gathered_rows(r), r.d, 128, BF16))) return rc;
    if ((rc = map16(&w_rows, w, r.d, r.V, ldw, 128, BF16))) return rc;
    if ((rc = map16(&g.x_cols, x, r.d, r.T, ldx, 64, BF16))) return rc;
    if ((rc = map16(&g.xg_cols, b.xg, r.d, gathered_rows(r), r.d, 64, BF16))) return rc;
    if ((rc = map16(&g.w_cols, w, r.d, r.V, ldw, 64, BF16))) return rc;
    g.c_dx = g.c_dw = g.x_cols;            // (one that is not wanted is not used)
    if (dx && (rc = map_sums(&g.c_dx, b.dx, r.dx_splits * r.Tp, r.d))) return rc;
    if (dw) {
        if (r.dw_splits > 1) rc = map_sums(&g.c_dw, b.dw, r.dw_splits * up(r.V, M), r.d);
        else rc = map16(&g.c_dw, dw, r.d, r.V, r.d, 32, BF16);
        if (rc) return rc;
    }
    p.dz = static_cast<uint16_t*>(b.dz); p.dz_ld = (int)r.dz_ld;
    p.dx_splits = dx ? r.dx_splits : 0; p.dx_rows = (int)r.Tp;
    p.dw_splits = dw ? r.dw_splits : 0; p.dw_rows = (int)up(r.V, M);
    for (int i = 0; i < r.pieces; ++i) {
        p.v0 = (int)(i * r.vc);
        p.vc = (int)std::min<int64_t>(r.vc, r.V - p.v0);
        p.add_dx = i > 0;
        if ((rc = map16(&g.z_rows, b.dz, p.vc, r.Tp, r.dz_ld, 128, BF16))) return rc;
        if ((rc = map16(&g.z_cols, b.dz, p.vc, r.Tp, r.dz_ld, 64, BF16))) return rc;
        if ((rc = launch<product_kernel<SOFT, BF16>, SMEM_Z>(st, x_rows, w_rows, xg_rows, p))) return rc;
        rc = r.dw_splits > 1 ? launch<grads_kernel<BF16, true>, SMEM_G>(st, g, p) : launch<grads_kernel<BF16, false>, SMEM_G>(st, g, p);
        if (rc) return rc;
    }
    if (dx && (rc = finish<BF16>(b.dx, r.dx_splits, r.Tp, r.T, r.d, s.slot, p, dx, st))) return rc;
    if (dw && r.dw_splits > 1) return finish<BF16>(b.dw, r.dw_splits, up(r.V, M), r.V, r.d, nullptr, p, dw, st);
    return CINN_OK;
}

}  // namespace ce

int64_t linear_ce_state_bytes(int64_t T) {
    int64_t n = 0;
    if (T > 0) ce::carve_state(nullptr, T, &n);
    return n;
}
// pass: 0 = forward, 1 = forward with early gradients, 4 = (late) backward, + 1 with dx, + 2 with dw
int64_t linear_ce_workspace_bytes(int64_t T, int64_t V, int64_t d, int pass) {
    if (T <= 0 || V <= 0 || d <= 0) return 0;
    int64_t n = 0;
    const ce::Plan r = ce::make_plan(T, V, d, pass == 1);
    if (pass < 4) ce::carve_forward(nullptr, r, &n);
    else ce::carve_backward(nullptr, r, pass & 1, pass & 2, &n);
    return n;
}
// which: 0 = whether the early way is taken, 1, 2 = bytes of the sums of dx, dw
int64_t linear_ce_early(int64_t T, int64_t V, int64_t d, int reduction, int which) {
    if (T <= 0 || V <= 0 || d <= 0) return 0;
    if (which == 0) return ce::early_pays(T, V, d, reduction);
    const ce::Plan r = ce::make_plan(T, V, d, true);
    return which == 1 ? ce::dx_sums_bytes(r) : ce::dw_sums_bytes(r);
}

int linear_ce_forward(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, const int64_t* target, int64_t ignore, int64_t T, int64_t V,
                      int64_t d, int reduction, float* loss, void* state, float* dx_sums, float* dw_sums, void* workspace, int64_t workspace_bytes,
                      cudaStream_t st) {
    int rc = ce::check_shapes(x, ldx, w, ldw, dtype, T, V, d, reduction);
    if (rc) return rc;
    CINN_CHECK_ARG(loss || (T == 0 && reduction == 0), "linear_ce: null pointer");
    const bool early = dx_sums || dw_sums;
    CINN_CHECK_ARG(!early || (reduction != 0 && T > 0), "linear_ce: early gradients are those of a sum or mean over some tokens");
    CINN_CHECK_ARG(((reinterpret_cast<uintptr_t>(dx_sums) | reinterpret_cast<uintptr_t>(dw_sums)) & 15) == 0, "linear_ce: sums must be 16-byte aligned");
    if (T == 0) {
        // a mean of nothing is NaN (all bits set), a sum 0
        if (reduction) CINN_CHECK_CUDA(cudaMemsetAsync(loss, reduction == 1 ? 0xff : 0, 4, st));
        return CINN_OK;
    }
    CINN_CHECK_ARG(target && state && workspace, "linear_ce: null pointer");
    if ((rc = ce::check_scratch(state, workspace))) return rc;
    const ce::Plan r = ce::make_plan(T, V, d, early);
    int64_t need = 0;
    const ce::Forward f = ce::carve_forward(workspace, r, &need);
    CINN_CHECK_ARG(workspace_bytes >= need, "linear_ce: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
    const ce::State s = ce::carve_state(state, T, nullptr);
    return dtype == CINN_BF16 ? ce::forward<true>(x, ldx, w, ldw, target, ignore, r, reduction, loss, s, f, dx_sums, dw_sums, st)
                              : ce::forward<false>(x, ldx, w, ldw, target, ignore, r, reduction, loss, s, f, dx_sums, dw_sums, st);
}

// what is left of the early way's backward: the loss's gradient, and one rounding
int linear_ce_finish(int dtype, const float* grad, int64_t T, int64_t V, int64_t d, int reduction, const void* state, const float* dx_sums,
                     const float* dw_sums, void* dx, void* dw, cudaStream_t st) {
    CINN_CHECK_ARG((dtype == CINN_BF16 || dtype == CINN_F16) && T > 0 && V > 0 && d > 0 && d % 8 == 0 && (reduction == 1 || reduction == 2), "linear_ce finish: bad arguments");
    CINN_CHECK_ARG(grad && state && (!dx || dx_sums) && (!dw || dw_sums), "linear_ce finish: null pointer");
    int rc = ce::check_scratch(state, nullptr);
    if (rc) return rc;
    CINN_CHECK_ARG(((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw) | reinterpret_cast<uintptr_t>(dx_sums) |
                     reinterpret_cast<uintptr_t>(dw_sums)) & 15) == 0, "linear_ce finish: pointers must be 16-byte aligned");
    const ce::Plan r = ce::make_plan(T, V, d, true);
    const ce::State s = ce::carve_state(const_cast<void*>(state), T, nullptr);
    ce::Params p{};
    p.n_valid = s.n_valid; p.grad = grad; p.mean = reduction == 1;
    const bool bf16 = dtype == CINN_BF16;
    if (dx) rc = bf16 ? ce::finish<true>(dx_sums, r.dx_splits, r.Tp, T, d, s.slot, p, dx, st) : ce::finish<false>(dx_sums, r.dx_splits, r.Tp, T, d, s.slot, p, dx, st);
    if (rc || !dw) return rc;
    return bf16 ? ce::finish<true>(dw_sums, r.dw_splits, ce::up(V, ce::M), V, d, nullptr, p, dw, st)
                : ce::finish<false>(dw_sums, r.dw_splits, ce::up(V, ce::M), V, d, nullptr, p, dw, st);
}

int linear_ce_backward(const void* x, int64_t ldx, const void* w, int64_t ldw, int dtype, const float* grad, int64_t T, int64_t V, int64_t d,
                       int reduction, const void* state, void* dx, void* dw, void* workspace, int64_t workspace_bytes, cudaStream_t st) {
    int rc = ce::check_shapes(x, ldx, w, ldw, dtype, T, V, d, reduction);
    if (rc) return rc;
    if (!dx && !dw) return CINN_OK;
    if (T == 0) {
        if (dw) CINN_CHECK_CUDA(cudaMemsetAsync(dw, 0, (size_t)(V * d * 2), st));
        return CINN_OK;
    }
    CINN_CHECK_ARG(grad && state && workspace, "linear_ce: null pointer");
    if ((rc = ce::check_scratch(state, workspace))) return rc;
    CINN_CHECK_ARG(((reinterpret_cast<uintptr_t>(dx) | reinterpret_cast<uintptr_t>(dw)) & 15) == 0, "linear_ce: gradients must be 16-byte aligned");
    const ce::Plan r = ce::make_plan(T, V, d, false);
    int64_t need = 0;
    const ce::Backward b = ce::carve_backward(workspace, r, dx != nullptr, dw != nullptr, &need);
    CINN_CHECK_ARG(workspace_bytes >= need, "linear_ce: workspace of %lld bytes, %lld are needed", (long long)workspace_bytes, (long long)need);
    const ce::State s = ce::carve_state(const_cast<void*>(state), T, nullptr);
    return dtype == CINN_BF16 ? ce::backward<true>(x, ldx, w, ldw, grad, r, reduction, s, dx, dw, b, st)
                              : ce::backward<false>(x, ldx, w, ldw, grad, r, reduction, s, dx, dw, b, st);
}

int read_loss_status(int* out, int reset) {
    int v = 0;
    CINN_CHECK_CUDA(cudaMemcpyFromSymbol(&v, ce::g_status, sizeof(int)));
    if (reset && v) {
        const int z = 0;
        CINN_CHECK_CUDA(cudaMemcpyToSymbol(ce::g_status, &z, sizeof(int)));
    }
    *out = v;
    return CINN_OK;
}

}  // namespace cinn
