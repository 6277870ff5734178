// Attention of a tree of drafted tokens over a paged KV cache, on tcgen05.mma.
//
// The query rows of a sequence and KV head (n drafts x G query heads) are the M side of the products, 128 rows (TMEM
// lanes) to a CTA; the cache is walked in blocks of 128 tokens:
//     S[row][token] = Q (shared memory) x K^T (shared memory, K-major)          fp32 in tensor memory
//     P = exp2(S * scale - m), rounded to 16 bits, in place of S                tensor memory
//     O[row][dim]  += P (tensor memory) x V (shared memory, MN-major: V lies [token][dim] as the cache has it)
// Two groups of four warps take the blocks in turn, thread = row = TMEM lane: no shuffles, and while one group is at its
// exponentials the other waits, loads or stores (eight warps on one block at a time: 2.8 to 3.2 thousand cycles a block,
// all latencies in a row).  A row's maximum goes from group to group through shared memory.
//
// What bounds it: K and V are read once per 128 rows, 4 * HD * 128 * 128 multiply-adds for 4 * HD * 128 bytes; at 128
// rows the tensor cores need a third of the time that HBM takes, so up to 128 rows the kernel's business is to keep
// loads in flight: a ring of 32 KB stages (128 tokens x 128 dimensions of K, 64 x 256 or 128 x 128 of V), each filled by
// a warp of its own with 16-byte cp.async straight into the swizzled places; each lane's arrival on the stage's barrier
// follows its copies.  (TMA boxes were measured first: pages allow boxes of 8 or 16 tokens only, and
// issuing sixteen 2 KB boxes a stage bounds the rate at 7.2 TB/s over the GPU even out of L2, where cp.async reaches 18.
// With four warps on every stage each of them paid four waits a block.)  More rows are more tiles: CTAs of the tiles
// of one sequence walk the same blocks at the same time and share them in L2.
// Work is split evenly whatever the lengths: the blocks of all (sequence, KV head) pairs form one line, every CTA
// takes an equal piece of it (found from the lengths on the device), and a pair that several CTAs share leaves partial
// sums with their maximum, which a second kernel joins in order (fixed order: the same bytes every run).  The change from
// one pair to the next costs a CTA 8 to 14 thousand cycles (the last products, the result out, new queries in), as much as
// two to five blocks, so that many empty places follow each pair's blocks on the line (without them the CTA with the most
// pairs ended 13 to 37 % after the others).
// The running maximum is only raised when it grows by more than 8 (a factor of 256 that the fp32 sums and the 16-bit
// probabilities hold easily), so O is seldom rescaled.
//
// Tokens nobody sees must not matter, whatever they hold: rows behind the end and rows on pages outside the pool are
// filled with zeros instead of read, and non-finite V values of drafts, which some rows see and others do not, are
// zeroed before the product and added to the rows that see them at the end (a path that finite caches never take).
//
// e4m3 caches: a pair of warps per stage fetches the 16 KB of rows into the stage's upper half and widens them in place,
// from the front, exactly to the 16-bit type of q in the swizzled places; the scales fold into the softmax scale and the
// normalisation.  The selections that keep the two halves of a row's lanes off each other's banks are worth it (60 against
// 63 us with the conflicts); bytes fetched to registers instead, all or half of them ahead of the stage's release, took 80 and
// 75 us at a time when this took 73 (57 now).
//
// Measured (device time, 24 query / 4 KV heads of 256 unless said; the GPUs differ by some per cent): 64 sequences x 16 drafts
// over 1000 .. 8192 tokens 220 to 250 us, 5.6 to 4.9 TB/s (the kernel without products and softmax: 214; HBM's time 190); 61 drafts
// over 32768 tokens, three tiles, 69 to 77 us, 714 TFLOP/s (58 without products and softmax); 32 x 8 drafts, e4m3, 57 us (52);
// 16 sequences of 1 .. 64 drafts, bf16, 32 / 8 heads of 128, 95 to 109 us (77); 5 drafts over 300 tokens 15 us (12).  So what
// bounds it away from HBM's rate is the ring: five stages, 160 KB a CTA (beside 128 dimensions, where the queries take 32 KB and not
// 64, a sixth would fit a CTA of the 16-bit caches; not measured), a stage's round trip 3 to 3.7 thousand cycles (issue 1.0 to 1.9,
// arrival 1.0 to 1.3, pick-up and release 0.5), with start-up, join and launches 12 us.  Not kept: two warps a stage for
// 16-bit caches (77 -> 81 us, 248 -> 243), three softmax groups at 128 dimensions (117 -> 121), the next stage's lines asked
// into L2 (+ 5 to 15 %), the queries loaded by the softmax warps (15.4 -> 14.7, but 248 -> 251 at the largest).
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_fp8.h>
#include <cuda_runtime.h>
#include <limits.h>
#include <math.h>
#include <stdint.h>

#include "exl3_common.cuh"
#include "exl3_paged.cuh"
#include "exl3_tcgen05.cuh"

namespace exl3 {
namespace tree {
using namespace t5;

constexpr int kM = 128;                       // rows of a tile
constexpr int kTok = 128;                     // tokens of a block
constexpr int kDims = 128;                    // dimensions of a stage
constexpr int kStageBytes = kTok * kDims * 2; // 32 KB
constexpr int kMostChange = 5;                // the largest Params::change
constexpr int kMaxTiles = 16;
constexpr int kMaxGrid = 148;
constexpr float kRaise = 8.f;                 // log2 units the maximum may lag behind

static __device__ unsigned g_tree_status;     // sticky: non-zero after a bounded wait ran out

struct Params {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const void *k, *v;
    long long page_stride, head_stride, tok_stride;
    const int *block_table, *seq_lens, *starts;
    const long long *mask;
    int bt_stride, width, num_pages, page_size;
    int batch, tokens, max_drafts, kvh, G, tiles;    // tiles: of the sequence with the most drafts
    int change;                               // places on the line behind a pair's blocks
    float scale_log2, v_scale;
    int negate;                               // the scale is negative: Q K^T is negated, scale_log2 is its size
    int rows_ws;                              // rows of a partial result (a multiple of 32)
    int4 *joins;                              // per CTA: the pair whose blocks begin in its piece and end behind it: (sequence,
                                              // KV head, parts, tile * 2 + slot of the first part); x < 0: none
    float *part_ml, *part_o;                  // [2 * grid][2][rows_ws], [2 * grid][HD / 4][rows_ws][4]: lane = row, full lines
};

struct Shared {
    // A stage has a barrier for K and one for V: each of the two threads that issue MMAs sees only the rounds that are
    // its own (with one barrier a thread could be a whole round behind another's, and parity would mislead it).
    uint64_t k_full[5], v_full[5], empty[5];
    uint64_t s_full[3], p_ready[3], v_here[3], pv_done[3], q_empty, o_free, drain[2];
    uint32_t tmem_base;
    int nonfinite[2];                         // of the current segment and the one before, in turn
    float top[kM];                            // of the rows
    union {
        int part[kMaxTiles][20];              // blocks per tile and warp (before the roles part)
        float sum[2][kM];                     // sums of the two groups
    };
    int first_seq, first_off;
};
static_assert(sizeof(Shared) <= 3 * 1024, "shared state");

template <bool FP8, int HD>
struct Cfg {
    static constexpr int kHalves = HD / kDims;                       // stages of a K or V block
    static constexpr int kBufs = (512 - HD) / kTok;                  // scores in tensor memory: 2 blocks beside 256 dimensions, 3 beside 128
    static constexpr int kQBytes = kM * HD * 2;
    static constexpr int kStages = 5;
    static constexpr int kThreads = 32 * (10 + (FP8 ? 2 : 1) * kStages);     // 2 MMA + 8 softmax warps, one or two per stage
    static constexpr int kSmem = kQBytes + kStages * kStageBytes + sizeof(Shared);
};


// Sixteen bytes into shared memory, or zeros.
__device__ __forceinline__ void copy16(uint32_t dst, const void *src, bool real) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(real ? 16 : 0) : "memory");
}
__device__ __forceinline__ void copy16(uint32_t dst, const void *src) {      // (without a size: a fifth quicker out of L2)
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(dst), "l"(src) : "memory");
}
__device__ __forceinline__ uint32_t pick(bool which, uint32_t a, uint32_t b) {      // (left to itself, the compiler branches)
    uint32_t v;
    asm("{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %3, 0;\n\tselp.b32 %0, %1, %2, p;\n\t}" : "=r"(v) : "r"(a), "r"(b), "r"((int)which));
    return v;
}
// This thread's arrival on the barrier once its copies so far have landed.
__device__ __forceinline__ void arrive_behind_copies(uint32_t bar) {
    asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
// Shared-memory operand, 128-byte swizzle.  K-major: rows of 128 bytes, groups of eight rows `sbo` bytes apart.
// MN-major: atoms of 64 values x 8 k, `lbo` bytes apart along the values, `sbo` along k.
__device__ __forceinline__ uint64_t desc_sw128(uint32_t addr, uint32_t lbo, uint32_t sbo) {
    return (uint64_t)((addr & 0x3FFFF) >> 4) | (uint64_t)(lbo >> 4) << 16 | (uint64_t)(sbo >> 4) << 32 | (uint64_t)1 << 46 |
           (uint64_t)2 << 61;
}
__device__ __forceinline__ void umma_f16_ss(uint32_t d_tmem, uint64_t a_desc, uint64_t b_desc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}"
        ::"r"(d_tmem), "l"(a_desc), "l"(b_desc), "r"(idesc), "r"(accumulate) : "memory");
}
// 32 consecutive columns of this thread's lane; the values are there after tmem_wait_ld.
__device__ __forceinline__ void tmem_ld32(uint32_t taddr, uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
        : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]),
          "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]), "=r"(v[14]), "=r"(v[15]), "=r"(v[16]), "=r"(v[17]),
          "=r"(v[18]), "=r"(v[19]), "=r"(v[20]), "=r"(v[21]), "=r"(v[22]), "=r"(v[23]), "=r"(v[24]), "=r"(v[25]), "=r"(v[26]),
          "=r"(v[27]), "=r"(v[28]), "=r"(v[29]), "=r"(v[30]), "=r"(v[31])
        : "r"(taddr) : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }
__device__ __forceinline__ void tmem_st32(uint32_t taddr, const uint32_t (&v)[32]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,"
        "%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]), "r"(v[16]), "r"(v[17]),
          "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]), "r"(v[24]), "r"(v[25]), "r"(v[26]),
          "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31]) : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile(
        "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};"
        ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]),
          "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]) : "memory");
}
__device__ __forceinline__ float ex2(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void fence_async() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }
// From a warp of one group to the warp of the same rows in the other (each id has one arriving and one waiting warp);
// all eight softmax warps.
__device__ __forceinline__ void pass_on(int id) { asm volatile("bar.arrive %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void take_over(int id) { asm volatile("bar.sync %0, 64;" ::"r"(id) : "memory"); }
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 9, 256;" ::: "memory"); }

// ---------------------------------------------------------------- the line of blocks
struct Seq { int first, n, len, rows, blocks, units; };    // first row of q, drafts, tokens, query rows per KV head, blocks, places on the line

__device__ __forceinline__ Seq seq_of(const Params &P, int b) {
    Seq s;
    const int lo = max(0, min(__ldg(P.starts + b), P.tokens)), hi = max(lo, min(__ldg(P.starts + b + 1), P.tokens));
    s.first = lo;
    s.n = hi - lo;
    s.len = max(0, min(__ldg(P.seq_lens + b), P.width * P.page_size));
    s.rows = min(s.n, P.max_drafts) * P.G;
    s.blocks = s.rows ? max(1, (s.len + kTok - 1) / kTok) : 0;
    s.units = s.rows ? s.blocks + P.change : 0;
    return s;
}

// One CTA's piece of the line of one tile: what is left of it, as segments (blocks of one sequence and KV head).
struct Walk {
    const Params &P;
    int m, b, off, left, index;
    Seq s;
    int hk, blk, nb, nblk;             // the current segment
    __device__ __forceinline__ Walk(const Params &p, int tile, int seq, int offset, int count)
        : P(p), m(tile), b(seq), off(offset), left(count), index(-1), hk(0), blk(0), nb(0), nblk(0) {
        if (left > 0) s = seq_of(P, b);
    }
    __device__ __forceinline__ bool next() {
        for (;;) {
            if (left <= 0) return false;
            const int units = s.rows > kM * m ? s.units : 0;
            if (off < units * P.kvh) {
                hk = off / units;
                blk = off - hk * units;
                nblk = s.blocks;
                if (blk < nblk) break;
                off += units - blk;
                left -= units - blk;
            } else {
                off -= units * P.kvh;
                if (++b >= P.batch) { left = 0; return false; }
                s = seq_of(P, b);
            }
        }
        nb = min(nblk - blk, left);
        off += nb;
        left -= nb;
        ++index;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return nb == nblk; }
    __device__ __forceinline__ int rows() const { return min(kM, s.rows - kM * m); }
};

// CTAs of tile `lane` out of `grid`, in proportion to its blocks (at least one).  Tiles of equal work get equal numbers,
// so that their CTAs walk the same blocks at the same time.  A whole warp; the first tile has the most blocks.
__device__ __forceinline__ int share_of(int blocks, int tiles, int grid, int lane) {
    if (tiles == 1) return lane == 0 && blocks ? grid : 0;
    const double u = blocks;
    double all = u;
#pragma unroll
    for (int o = 16; o; o >>= 1) all += __shfl_xor_sync(0xffffffffu, all, o);
    int w = u > 0 ? max(1, (int)(grid * u / all)) : 0;
    const int used = __reduce_add_sync(0xffffffffu, w);
    if (lane == 0) w -= max(0, used - grid);
    return w;
}
// First block of piece w when U blocks are cut into W pieces.
__device__ __forceinline__ int piece(int U, int W, int w) {
    const int q = U / W;
    return w * q + min(w, U - q * W);
}

// The page of the sixteen tokens at t of sequence b, -1 when they are on none.
__device__ __forceinline__ int page_of(const Params &P, int b, int t, int len, int &at) {
    const int idx = t / P.page_size;
    at = t - idx * P.page_size;
    return t < len ? __ldg(P.block_table + (size_t)b * P.bt_stride + idx) : -1;
}

// The stages of a segment in the order of the ring: K(0), then K(i + 1) (if there is one) and V(i) for every block i, H
// stages each.  Stage j of the segment:
struct Fill { int block, half; bool is_v; };
template <int H>
__device__ __forceinline__ Fill fill_of(int j, int nb) {
    if (j < H) return Fill{0, j, false};
    const int q = (j - H) / (2 * H), r = (j - H) % (2 * H);
    if (q < nb - 1 && r < H) return Fill{q + 1, r, false};
    return Fill{q, r % H, true};
}

// ---------------------------------------------------------------- e4m3 -> 16 bits
template <typename T>
__device__ __forceinline__ void widen4(uint32_t w, uint32_t &lo, uint32_t &hi) {
    asm("{\n\t.reg .b16 a, b;\n\tmov.b32 {a, b}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, a;\n\tcvt.rn.f16x2.e4m3x2 %1, b;\n\t}"
        : "=r"(lo), "=r"(hi) : "r"(w));
    if constexpr (sizeof(T) == 2 && !__is_same(T, __half)) {      // bf16 holds every e4m3 value too
        const float2 a = Type16<__half>::to_float2(lo), b = Type16<__half>::to_float2(hi);
        lo = Type16<T>::pack(a.x, a.y);
        hi = Type16<T>::pack(b.x, b.y);
    }
}
template <typename T>
__device__ __forceinline__ bool nonfinite2(uint32_t w, uint32_t &keep) {      // keep: the pair with non-finite values zeroed
    constexpr uint32_t kExp = __is_same(T, __half) ? 0x7C00u : 0x7F80u;
    const bool lo = (w & kExp) == kExp, hi = (w >> 16 & kExp) == kExp;
    keep = (lo ? 0u : w & 0xFFFFu) | (hi ? 0u : w & 0xFFFF0000u);
    return lo || hi;
}

template <typename T, bool FP8, int HD>
__global__ void __launch_bounds__(Cfg<FP8, HD>::kThreads, 1)
tree_attn_kernel(const __grid_constant__ Params P) {
    using C = Cfg<FP8, HD>;
    constexpr int H = C::kHalves;
    constexpr int kThreads = C::kThreads;
    extern __shared__ __align__(1024) unsigned char smem[];      // (swizzle atoms are 1 KB)
    unsigned char *const smQ = smem, *const ring = smQ + C::kQBytes;
    Shared &S = *reinterpret_cast<Shared *>(ring + C::kStages * kStageBytes);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned *const status = &g_tree_status;
    if (s32(smem) & 1023u) {
        asm volatile("griddepcontrol.wait;" ::: "memory");
        if (tid == 0) { atomicOr(status, 2u); P.joins[blockIdx.x] = make_int4(-1, 0, 0, 0); }
        return;
    }

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) { mbar_init(s32(&S.k_full[i]), FP8 ? 2 : 32); mbar_init(s32(&S.v_full[i]), FP8 ? 2 : 32); mbar_init(s32(&S.empty[i]), 1); }
        for (int i = 0; i < C::kBufs; ++i) { mbar_init(s32(&S.s_full[i]), 1); mbar_init(s32(&S.p_ready[i]), 4); mbar_init(s32(&S.v_here[i]), 1); mbar_init(s32(&S.pv_done[i]), 1); }
        mbar_init(s32(&S.q_empty), 1);
        mbar_init(s32(&S.o_free), 8); mbar_init(s32(&S.drain[0]), 1); mbar_init(s32(&S.drain[1]), 1);
        S.nonfinite[0] = S.nonfinite[1] = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (warp == 1) tmem_alloc(s32(&S.tmem_base), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = S.tmem_base;
    asm volatile("griddepcontrol.wait;" ::: "memory");       // lengths, queries, cache rows of the kernels before
    asm volatile("griddepcontrol.launch_dependents;");

    // ---- this CTA's piece of the line: a thread has a run of sequences
    constexpr int kWarps = kThreads / 32;
    static_assert(kWarps <= 20, "S.part");
    const int run = (P.batch + kThreads - 1) / kThreads, b0 = tid * run, b1 = min(P.batch, b0 + run);
    Seq s0 = {};
    if (b0 < b1) s0 = seq_of(P, b0);
    const auto blocks_of = [&](int m) {                      // of the run, in tile m
        int v = s0.rows > kM * m ? s0.units * P.kvh : 0;
        for (int b = b0 + 1; b < b1; ++b) { const Seq s = seq_of(P, b); v += s.rows > kM * m ? s.units * P.kvh : 0; }
        return v;
    };
    for (int t = 0; t < P.tiles; ++t) {
        const int sum = __reduce_add_sync(0xffffffffu, blocks_of(t));
        if (lane == 0) S.part[t][warp] = sum;
    }
    if (tid == 0) P.joins[blockIdx.x] = make_int4(-1, 0, 0, 0);
    __syncthreads();
    int m = 0, w = blockIdx.x, W = 0, U = 0;
    {
        int mine = 0;                                        // lane = tile: its blocks
        if (lane < P.tiles)
            for (int i = 0; i < kWarps; ++i) mine += S.part[lane][i];
        const int share = share_of(mine, P.tiles, gridDim.x, lane);
        int upto = share;                                    // CTAs of the tiles up to this lane's
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, upto, o);
            if (lane >= o) upto += y;
        }
        const uint32_t behind = __ballot_sync(0xffffffffu, upto > (int)blockIdx.x);
        if (behind) {
            m = __ffs(behind) - 1;
            W = __shfl_sync(0xffffffffu, share, m);
            U = __shfl_sync(0xffffffffu, mine, m);
            w -= __shfl_sync(0xffffffffu, upto - share, m);
        }
    }
    const int u0 = W ? piece(U, W, w) : 0, u1 = W ? piece(U, W, w + 1) : 0;
    if (u1 > u0) {                                           // whose run holds the first block?
        const int v = blocks_of(m);
        int x = v;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, x, o);
            if (lane >= o) x += y;
        }
        int off = u0 - (x - v);
        for (int i = 0; i < warp; ++i) off -= S.part[m][i];
        if (off >= 0 && off < v) {
            int b = b0;
            for (Seq s = s0;; s = seq_of(P, b)) {
                const int n = s.rows > kM * m ? s.units * P.kvh : 0;
                if (off < n) break;
                off -= n;
                ++b;
            }
            S.first_seq = b;
            S.first_off = off;
        }
    }
    __syncthreads();

    if (u1 > u0) {
        Walk wk(P, m, S.first_seq, S.first_off, u1 - u0);
        if (warp == 1) {
            // ---------------- Q into shared memory, then S = Q K^T.  Two threads issue the MMAs, one for each product: a thread's
            // waits, fences and commits cost it about as much as the tensor cores need for its share of a block (one thread for
            // both: 5050 cycles a block, of which the tensor cores worked 2300)
            constexpr uint32_t kType = __is_same(T, __half) ? 0u : (1u << 7 | 1u << 10);
            const uint32_t idesc = umma_idesc_f16(kM, kTok) | kType | (P.negate ? 1u << 13 : 0u);      // bit 13: -A
            const uint64_t qdesc = desc_sw128(s32(smQ), 16, 1024), kdesc = desc_sw128(s32(ring), 16, 2048);
            constexpr int kUnits = HD / 8, kRows = 32 / kUnits;   // 16-byte units of a row of Q, rows of an instruction
            const int u = lane % kUnits, sub = lane / kUnits;
            int written = kM;                                  // rows of Q that may hold something
            uint32_t phases = 0;                               // of the stages' K barriers
            int stage = 0, cnt = 0;
            bool ok = true;
            const auto here = [&](int st) {
                const bool is = mbar_wait(s32(&S.k_full[st]), phases >> st & 1, status);
                phases ^= 1u << st;
                return is;
            };
            while (ok && wk.next()) {
                // rows (swizzled, K-major); those behind the last one are zero
                if (wk.index) ok = __all_sync(0xffffffffu, mbar_wait(s32(&S.q_empty), (wk.index - 1) & 1, status));
                if (!ok) break;
                const int rows = wk.rows(), upto = max(written, rows);
                int r = sub, i = (kM * m + r) / P.G, g = kM * m + r - i * P.G;
                const T *src = static_cast<const T *>(P.q) + (size_t)(wk.s.first + i) * P.q_stride + (size_t)(wk.hk * P.G + g) * HD + 8 * u;
                const int di = kRows / P.G, dg = kRows - di * P.G;
                const long long step = di * P.q_stride + dg * HD, wrap = P.q_stride - (long long)P.G * HD;
                const uint32_t dst = s32(smQ) + (u >> 3) * (kM * 128);
#pragma unroll 4
                for (; r < rows; r += kRows) {
                    copy16(dst + r * 128 + (((u & 7) ^ (r & 7)) << 4), src);
                    src += step; g += dg;
                    if (g >= P.G) { g -= P.G; src += wrap; }
                }
                for (; r < upto; r += kRows)
                    *reinterpret_cast<uint4 *>(smQ + (u >> 3) * (kM * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = make_uint4(0, 0, 0, 0);
                written = rows;
                asm volatile("cp.async.wait_all;" ::: "memory");
                fence_async();
                __syncwarp();
                if (lane == 0) {
                    for (int i = 0; i < wk.nb && ok; ++i, ++cnt) {
                        const int buf = cnt % C::kBufs;
                        const uint32_t phase = cnt / C::kBufs & 1;
                        // (128 dimensions: K is mostly there, and P the last to come; 256: the first half need not wait for the second)
                        if constexpr (H == 1) ok = here(stage);
                        if (ok && cnt >= C::kBufs) ok = mbar_wait(s32(&S.pv_done[buf]), phase ^ 1u, status);    // the P that lay there was used
                        const uint32_t d = tmem + HD + buf * kTok;
                        for (int h = 0; h < H && ok; ++h) {
                            if constexpr (H > 1) ok = here(stage);
                            if (!ok) break;
                            if constexpr (!FP8) fence_async();     // the copies were other warps', plain ones
                            fence_after_sync();
                            const uint64_t kd = kdesc + (uint32_t)(stage * (kStageBytes >> 4)), qd = qdesc + (uint32_t)(h * (2 * kM * 128 >> 4));
#pragma unroll
                            for (int k = 0; k < kDims / 16; ++k)
                                umma_f16_ss(d, qd + ((k / 4) * (kM * 128) + (k % 4) * 32 >> 4), kd + ((k / 4) * 1024 + (k % 4) * 32 >> 4), idesc, h || k);
                            umma_commit(s32(&S.empty[stage]));
                            if (++stage == C::kStages) stage = 0;
                        }
                        umma_commit(s32(&S.s_full[buf]));
                        // over V(i - 1) to the next K; behind the last K lie V of the last two blocks
                        const int skip = i + 1 == wk.nb ? (wk.nb > 1 ? 2 * H : H) : i ? H : 0;
                        stage = (stage + skip) % C::kStages;
                    }
                    umma_commit(s32(&S.q_empty));
                }
                ok = __shfl_sync(0xffffffffu, ok, 0);
            }
            if (lane == 0) {
                umma_commit(s32(&S.drain[0]));
                mbar_wait(s32(&S.drain[0]), 0, status);
            }
        } else if (warp == 0) {
            // ---------------- O += P V
            if (lane == 0) {
                constexpr uint32_t kType = __is_same(T, __half) ? 0u : (1u << 7 | 1u << 10);
                const uint32_t idesc = umma_idesc_f16(kM, HD) | kType | 1u << 16;                          // bit 16: B is MN-major
                const uint64_t vdesc = desc_sw128(s32(ring), 1024, HD * 16);
                uint32_t phases = 0;
                int stage = 0, cnt = 0;
                bool ok = true;
                while (ok && wk.next()) {
                    for (int i = 0; i < wk.nb && ok; ++i, ++cnt) {
                        const int buf = cnt % C::kBufs;
                        // before V(i) lies K(i + 1), before V(0) also K(0)
                        stage = (stage + (i + 1 < wk.nb ? H : 0) + (i ? 0 : H)) % C::kStages;
                        // e4m3: V's halves are used and given back as they come (57 against 60 us; 16 bits: 79 against 77), but where
                        // drafts are looked over (`clean`) all of V has to be there before P is.
                        const int early = !FP8 || H == 1 || (wk.blk + i + 1) * kTok > wk.s.len - wk.s.n ? H : 1;
                        int st = stage, got = 0;
                        const auto here = [&] {
                            const bool is = mbar_wait(s32(&S.v_full[st]), phases >> st & 1, status);
                            phases ^= 1u << st;
                            if (++st == C::kStages) st = 0;
                            if (++got == H) mbar_arrive(s32(&S.v_here[buf]));
                            return is;
                        };
                        while (ok && got < early) ok = here();
                        if (ok) ok = mbar_wait(s32(&S.p_ready[buf]), cnt / C::kBufs & 1, status);
                        if (ok && i == 0 && wk.index) ok = mbar_wait(s32(&S.o_free), (wk.index - 1) & 1, status);
                        for (int h = 0; h < H && ok; ++h) {
                            if (got == h) ok = here();
                            if (!ok) break;
                            if constexpr (!FP8) fence_async();
                            fence_after_sync();
                            const uint64_t vd = vdesc + (uint32_t)(stage * (kStageBytes >> 4));
                            const uint32_t p = tmem + HD + buf * kTok + h * 32;
#pragma unroll
                            for (int k = 0; k < kTok / H / 16; ++k)
                                umma_f16_ts(tmem, p + k * 8, vd + (k * (HD * 32) >> 4), idesc, i || h || k);
                            umma_commit(s32(&S.empty[stage]));
                            if (++stage == C::kStages) stage = 0;
                        }
                        if (ok) umma_commit(s32(&S.pv_done[buf]));
                    }
                }
                umma_commit(s32(&S.drain[1]));
                mbar_wait(s32(&S.drain[1]), 0, status);
            }
        } else if (warp < 10) {
            // ---------------- softmax: thread = row = TMEM lane; group `side` takes the blocks of its parity
            const int quarter = warp & 3, row = 32 * quarter + lane, side = (warp - 2) >> 2;
            const uint32_t lane_base = (uint32_t)(32 * quarter) << 16;
            constexpr int kCols = HD / 2;                      // of the result, this thread's half
            const uint32_t o_t = tmem + lane_base + side * kCols;
            // These warps meet at barriers: after a wait that ran out they walk on without waiting (what they write is
            // garbage then, the status word says so).
            bool ok = true;
            const auto hold = [&](uint64_t *bar, uint32_t parity) {
                if (ok) ok = __all_sync(0xffffffffu, mbar_wait(s32(bar), parity, status, 40));
                fence_after_sync();
            };
            int cnt = 0, pos = 0;                              // blocks done; ring position of the segment
            while (wk.next()) {
                const int rows = wk.rows();
                const int R = kM * m + row, draft = R / P.G;
                const bool live = row < rows;
                const int ctx = wk.s.len - wk.s.n;             // first draft's token (negative: drafts that have none)
                unsigned long long bits = 0;
                if (live) bits = P.mask ? (unsigned long long)__ldg(P.mask + wk.s.first + draft) : (draft >= 63 ? ~0ull : (2ull << draft) - 1);
                float top = -INFINITY;
                float2 sum2 = make_float2(0.f, 0.f);           // over this group's blocks, relative to `top`
                // Non-finite values of drafts in V become zeros (see the top of the file).
                const auto clean = [&](int n, int i, int tok0) {
                    if (tok0 + kTok <= ctx) return;
                    const int from = max(0, ctx - tok0), upto = min(kTok, wk.s.len - tok0);
                    const int vpos = pos + H + 2 * H * i + (i + 1 < wk.nb ? H : 0);
                    hold(&S.v_here[n % C::kBufs], n / C::kBufs & 1);      // (announced by the MMA thread, which looks at every stage in its turn)
                    constexpr int kUnits = HD / 8, kRowsV = kTok / H;           // 16-byte units of a row, rows of a stage
                    for (int e = row; e < (upto - from) * kUnits; e += 128) {
                        const int r = from + e / kUnits, u = e % kUnits, st = (vpos + r / kRowsV) % C::kStages, q = r % kRowsV;
                        uint4 *const at = reinterpret_cast<uint4 *>(ring + (size_t)st * kStageBytes + (q >> 3) * (HD * 16) + (u >> 3) * 1024 +
                                                                    (q & 7) * 128 + (((u & 7) ^ (q & 7)) << 4));
                        const uint4 v = *at;
                        uint4 y;
                        const bool a = nonfinite2<T>(v.x, y.x), b2 = nonfinite2<T>(v.y, y.y), c = nonfinite2<T>(v.z, y.z),
                                   d = nonfinite2<T>(v.w, y.w);
                        if (a || b2 || c || d) { *at = y; S.nonfinite[wk.index & 1] = 1; }
                    }
                    fence_async();
                };
                const auto ready = [&](int n) {
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s32(&S.p_ready[n % C::kBufs]));
                };
                for (int i = (cnt ^ side) & 1; i < wk.nb; i += 2) {
                    const int n = cnt + i, tok0 = (wk.blk + i) * kTok;         // n: number of the block in the CTA
                    int at;
                    const int t8 = tok0 + 16 * (lane & 7), page = page_of(P, wk.b, t8, wk.s.len, at);
                    const uint32_t groups = __ballot_sync(0xffffffffu, t8 >= wk.s.len || (unsigned)page < (unsigned)P.num_pages) & 0xFFu;
                    const bool masked = tok0 + kTok > ctx || groups != 0xFFu;          // uniform in the warp
                    // which of the 32 tokens from tok0 + 32 k the row sees: context, then the drafts' bits shifted to their places
                    const auto seen = [&](int k) {
                        const int c = ctx - tok0 - 32 * k, l = wk.s.len - tok0 - 32 * k;
                        uint32_t v = 0;
                        if (c >= 32) v = ~0u;
                        else if (c > 0) v = (1u << c) - 1 | (uint32_t)(bits << c);
                        else v = -c < 64 ? (uint32_t)(bits >> -c) : 0u;
                        if (l < 32) v &= l > 0 ? (1u << l) - 1 : 0u;
                        v &= (groups >> (2 * k) & 1 ? 0xFFFFu : 0u) | (groups >> (2 * k) & 2 ? 0xFFFF0000u : 0u);
                        return live ? v : 0u;
                    };
                    // (The loops over four times 32 scores stay loops: unrolled, the code of the roles did not fit the instruction
                    // caches, and the warps waited for instructions more often than for anything but loads.  Nor did it pay to take
                    // the exponentials against the maximum known so far and read the scores once: 85 against 79 us at 61 drafts over
                    // 32768 tokens, the probabilities being in registers until that maximum is confirmed, and the loop unrolled.)
                    const uint32_t s_t = tmem + lane_base + HD + n % C::kBufs * kTok;
                    hold(&S.s_full[n % C::kBufs], n / C::kBufs & 1);
                    if (32 * quarter >= rows) {                // no rows in this quarter: whatever lies there as P stays in its lanes
                        clean(n, i, tok0);
                        ready(n);
                        continue;
                    }
                    float mx = -INFINITY;
                    const auto mask = [&](int k, uint32_t (&y)[32]) {          // minus infinity where nothing is seen
                        if (masked) {
                            const uint32_t vis = seen(k);
#pragma unroll
                            for (int e = 0; e < 32; ++e) y[e] = vis >> e & 1 ? y[e] : 0xFF800000u;
                        }
                    };
                    const auto greatest = [&](int k, uint32_t (&y)[32]) {
                        mask(k, y);
                        float m4[4] = {mx, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
                        for (int e = 0; e < 32; ++e) m4[e & 3] = fmaxf(m4[e & 3], __uint_as_float(y[e]));
                        mx = fmaxf(fmaxf(m4[0], m4[1]), fmaxf(m4[2], m4[3]));
                    };
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        uint32_t y[32];
                        tmem_ld32(s_t + 32 * k, y);
                        tmem_wait_ld();
                        greatest(k, y);
                    }
                    mx = mx == -INFINITY ? mx : mx * P.scale_log2;
                    if (i > 0) {                               // the maximum as the block before left it, and this group's sum with it
                        take_over(1 + 4 * (side ^ 1) + quarter);
                        const float before = top;
                        top = S.top[row];
                        if (top != before) { const float c = ex2(before - top); sum2.x *= c; sum2.y *= c; }
                    }
                    const bool raise = mx > top + kRaise || (top == -INFINITY && mx > top);
                    const float corr = raise ? ex2(top - mx) : 1.f;    // 0 when nothing was seen before
                    if (raise) { top = mx; sum2.x *= corr; sum2.y *= corr; }
                    if (raise || i == 0) S.top[row] = top;
                    if (__any_sync(0xffffffffu, raise) && i > 0) {
                        hold(&S.pv_done[(n - 1) % C::kBufs], (n - 1) / C::kBufs & 1);
#pragma unroll 1
                        for (int c = 0; c < HD; c += 32) {
                            uint32_t o[32];
                            tmem_ld32(tmem + lane_base + c, o);
                            tmem_wait_ld();
#pragma unroll
                            for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                            tmem_st32(tmem + lane_base + c, o);
                        }
                    }
                    if (i + 1 < wk.nb) pass_on(1 + 4 * side + quarter);
                    const float shift = top == -INFINITY ? 0.f : top;
                    const float2 mul = make_float2(P.scale_log2, P.scale_log2), sub = make_float2(-shift, -shift);
                    const auto exps = [&](int k, uint32_t (&y)[32]) {
                        uint32_t p[16];
                        mask(k, y);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float2 a = fma2(make_float2(__uint_as_float(y[2 * e]), __uint_as_float(y[2 * e + 1])), mul, sub);
                            a.x = ex2(a.x);
                            a.y = ex2(a.y);
                            sum2 = add2(sum2, a);
                            p[e] = Type16<T>::pack(a.x, a.y);
                        }
                        tmem_st16(s_t + 16 * k, p);            // over scores that were read
                    };
#pragma unroll 1
                    for (int k = 0; k < 4; ++k) {
                        uint32_t y[32];
                        tmem_ld32(s_t + 32 * k, y);
                        tmem_wait_ld();
                        exps(k, y);
                    }
                    clean(n, i, tok0);
                    tmem_wait_st();
                    ready(n);
                }
                // ---- the segment's result
                cnt += wk.nb;
                softmax_sync();                                // S.top is the last block's now; and (for the group that had not the
                                                               // last block) its scores have been there, so all products but two
                hold(&S.pv_done[(cnt - 1) % C::kBufs], (cnt - 1) / C::kBufs & 1);
                {
                    const float before = top;
                    top = S.top[row];
                    const float c = top != before ? ex2(before - top) : 1.f;
                    S.sum[side][row] = (sum2.x + sum2.y) * c;  // (0 * 0 when this group saw nothing)
                }
                softmax_sync();
                const float sum = S.sum[0][row] + S.sum[1][row];
                const bool mend = S.nonfinite[wk.index & 1] != 0;       // uniform: all have written it before the barrier
                if (tid == 64) S.nonfinite[wk.index & 1 ^ 1] = 0;      // read before the last barrier, written behind the next
                const bool whole = wk.whole();
                const float inv = sum == 0.f ? 0.f : P.v_scale / sum;
                const int slot = 2 * blockIdx.x + (wk.index ? 1 : 0);
                float4 *const pcol = reinterpret_cast<float4 *>(P.part_o) + ((size_t)slot * (HD / 4) + side * (kCols / 4)) * P.rows_ws + row;
                T *orow[4];                                    // rows 4 (lane / 4) + 0..3 of the quarter, this lane's sixteen bytes
                if (whole) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        const int r = 32 * quarter + (lane & 28) + k, Rk = kM * m + r, i = Rk / P.G;
                        orow[k] = r < rows ? static_cast<T *>(P.out) + (size_t)(wk.s.first + i) * P.out_stride +
                                                 (size_t)(wk.hk * P.G + Rk - i * P.G) * HD + side * kCols + 8 * (lane & 3) : nullptr;
                    }
                }
#pragma unroll 1
                for (int c = 0; c < kCols; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(o_t + c, o);
                    tmem_wait_ld();
                    if (mend && live) {
                        const int t_end = min(wk.s.len, (wk.blk + wk.nb) * kTok);
                        for (int t = max(max(0, ctx), wk.blk * kTok); t < t_end; ++t) {
                            if (t - ctx > 63 || !(bits >> (t - ctx) & 1)) continue;
                            const int page = __ldg(P.block_table + (size_t)wk.b * P.bt_stride + t / P.page_size);
                            if (page < 0 || page >= P.num_pages) continue;
                            const size_t at = (size_t)page * P.page_stride + (size_t)wk.hk * P.head_stride +
                                              (size_t)(t % P.page_size) * P.tok_stride + side * kCols + c;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                float v;
                                if constexpr (FP8) v = (float)static_cast<const __nv_fp8_e4m3 *>(P.v)[at + e];
                                else v = (float)static_cast<const T *>(P.v)[at + e];
                                if (!isfinite(v)) o[e] = __float_as_uint(__uint_as_float(o[e]) + v);
                            }
                        }
                    }
                    __syncwarp();
                    if (whole) {
                        // a lane's 64 bytes are four pieces; four lanes exchange pieces so that each writes one piece of four
                        // rows, 64 contiguous bytes of a row from four lanes (a lane's own row: a line per lane and store)
                        uint32_t w[4][4];
#pragma unroll
                        for (int e = 0; e < 16; ++e)
                            w[e >> 2][e & 3] = Type16<T>::pack(__uint_as_float(o[2 * e]) * inv, __uint_as_float(o[2 * e + 1]) * inv);
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
#pragma unroll
                            for (int q = 0; q < 4; q += 2) {
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & 1 ? w[q][k] : w[q + 1][k], 1);
                                if (lane & 1) w[q][k] = got; else w[q + 1][k] = got;
                            }
#pragma unroll
                            for (int q = 0; q < 2; ++q) {
                                const uint32_t got = __shfl_xor_sync(0xffffffffu, lane & 2 ? w[q][k] : w[q + 2][k], 2);
                                if (lane & 2) w[q][k] = got; else w[q + 2][k] = got;
                            }
                        }
#pragma unroll
                        for (int k = 0; k < 4; ++k)
                            if (orow[k]) *reinterpret_cast<uint4 *>(orow[k] + c) = make_uint4(w[k][0], w[k][1], w[k][2], w[k][3]);
                    } else if (live) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            pcol[(c + e) / 4 * P.rows_ws] = make_float4(__uint_as_float(o[e]), __uint_as_float(o[e + 1]),
                                                                        __uint_as_float(o[e + 2]), __uint_as_float(o[e + 3]));
                    }
                    __syncwarp();
                }
                if (!whole && wk.blk == 0 && tid == 64) {          // more parts follow in the next CTAs
                    const int q = U / W, r = U - q * W, last = u1 + wk.nblk - wk.nb - 1;     // the pair's last block
                    const int owner = last < r * (q + 1) ? last / (q + 1) : r + (last - r * (q + 1)) / q;
                    P.joins[blockIdx.x] = make_int4(wk.b, wk.hk, owner - w + 1, 2 * m + (wk.index ? 1 : 0));
                }
                if (live && !whole && side == 0) {
                    P.part_ml[(size_t)(2 * slot) * P.rows_ws + row] = top;
                    P.part_ml[(size_t)(2 * slot + 1) * P.rows_ws + row] = sum;
                }
                fence_before_sync();
                softmax_sync();
                if (lane == 0) mbar_arrive(s32(&S.o_free));
                pos += 2 * H * wk.nb;
            }
        } else if constexpr (!FP8) {
            // ---------------- cache rows into the ring: warp f fills stage f (one warp waits for all of a stage's releases: with
            // stages passed round it could be a whole round ahead of the others, and parity would mislead it)
            const int f = warp - 10;
            int filled = 0;
            bool ok = true;
            // wide stages (K, and V of 128 dimensions): an instruction is two rows of 256 bytes; tall ones: one of 512
            const int half = lane >> 4, uk = lane & 15;
            uint32_t wide_at[4], tall_at[8];                   // inside a stage, rows 2 j + half, rows j
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const int r = 2 * j + half;
                wide_at[j] = s32(ring) + (uk >> 3) * 1024 + r * 128 + (((uk & 7) ^ r) << 4);
            }
#pragma unroll
            for (int j = 0; j < 8; ++j) tall_at[j] = s32(ring) + (lane >> 3) * 1024 + j * 128 + (((lane & 7) ^ j) << 4);
            const long long two = 2 * P.tok_stride;
            int skip = 0;                                      // stages of the segment before this warp's first
            while (ok && wk.next()) {
                const int fills = 2 * H * wk.nb;
                int j = (f + C::kStages - skip) % C::kStages;
                skip = (skip + fills) % C::kStages;
                if (j >= fills) continue;
                const long long head = wk.hk * P.head_stride;
                Fill fl = fill_of<H>(j, wk.nb);
                int t = (wk.blk + fl.block) * kTok + 16 * (lane & 7), at;      // lanes 0..7: sixteen tokens each
                int page = page_of(P, wk.b, t, wk.s.len, at);
                for (;;) {
                    const bool there = (unsigned)page < (unsigned)P.num_pages;
                    const long long off = there ? page * P.page_stride + head + at * P.tok_stride : 0ll;
                    const int rows = there ? wk.s.len - t : 0;
                    const Fill now = fl;
                    const bool more = j + C::kStages < fills;
                    if (more) {                                // the pages of the warp's next stage
                        fl = fill_of<H>(j + C::kStages, wk.nb);
                        t = (wk.blk + fl.block) * kTok + 16 * (lane & 7);
                        page = page_of(P, wk.b, t, wk.s.len, at);
                    }
                    if (filled) ok = mbar_wait(s32(&S.empty[f]), (filled - 1) & 1, status, 40);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t stage = f * kStageBytes;
                    const T *const pool = static_cast<const T *>(now.is_v ? P.v : P.k);
                    if (H == 2 && now.is_v) {
#pragma unroll 1
                        for (int g = 0; g < 4; ++g) {
                            const T *src = pool + __shfl_sync(0xffffffffu, off, 4 * now.half + g) + 8 * lane;
                            const int n = __shfl_sync(0xffffffffu, rows, 4 * now.half + g);
                            if (n >= 16) {
#pragma unroll
                                for (int i = 0; i < 16; ++i, src += P.tok_stride) copy16(tall_at[i & 7] + stage + g * 8192 + (i >> 3) * 4096, src);
                            } else {
#pragma unroll
                                for (int i = 0; i < 16; ++i, src += P.tok_stride)
                                    copy16(tall_at[i & 7] + stage + g * 8192 + (i >> 3) * 4096, i < n ? src : pool, i < n);
                            }
                        }
                    } else {
#pragma unroll 1
                        for (int g = 0; g < 8; ++g) {
                            const T *src = pool + __shfl_sync(0xffffffffu, off, g) + half * P.tok_stride + now.half * kDims + 8 * uk;
                            const int n = __shfl_sync(0xffffffffu, rows, g) - half;
                            if (__all_sync(0xffffffffu, n >= 15)) {
#pragma unroll
                                for (int i = 0; i < 8; ++i, src += two) copy16(wide_at[i & 3] + stage + g * 4096 + (i >> 2) * 2048, src);
                            } else {
#pragma unroll
                                for (int i = 0; i < 8; ++i, src += two)
                                    copy16(wide_at[i & 3] + stage + g * 4096 + (i >> 2) * 2048, 2 * i < n ? src : pool, 2 * i < n);
                            }
                        }
                    }
                    arrive_behind_copies(s32(&(now.is_v ? S.v_full : S.k_full)[f]));
                    ++filled;
                    j += C::kStages;
                    if (!more) break;
                }
            }
            asm volatile("cp.async.wait_all;" ::: "memory");
        } else {
            // ---------------- e4m3 rows: warps 2 f and 2 f + 1 fill stage f, in eight quads of four instructions (two each): wide,
            // sixteen tokens of 128 bytes, four to an instruction; tall, eight tokens of 256 bytes, two to an instruction.  Quad b
            // arrives at 16 KB + 2 KB * b and becomes the 4 KB at 4 KB * b.
            const int f = (warp - 10) >> 1, part = (warp - 10) & 1;
            int filled = 0;
            bool ok = true;
            // a lane's sixteen bytes are two units of the swizzled row, and the lanes of a row start with different ones: no bank
            // conflicts
            const int wsub = lane >> 3, wu = lane & 7, tsub = lane >> 4, tu = lane & 15;
            const bool swap = lane & 4;
            uint32_t wide_at[2], tall_at[2];                   // rows 4 j + wsub, 4 part + 2 j + tsub of an atom
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 4 * j + wsub;
                wide_at[j] = (wu >> 2) * 1024 + r * 128 + ((((wu & 3) * 2 + (swap ? 1 : 0)) ^ r) << 4);
            }
#pragma unroll
            for (int j = 0; j < 2; ++j) {
                const int r = 4 * part + 2 * j + tsub;
                tall_at[j] = (tu >> 2) * 1024 + r * 128 + ((((tu & 3) * 2 + (swap ? 1 : 0)) ^ r) << 4);
            }
            const uint32_t raw = s32(ring) + f * kStageBytes + 16384 + part * 1024 + 16 * lane;
            const auto fetch = [&](const Fill &fl, long long off, int rows) {
                const unsigned char *const pool = static_cast<const unsigned char *>(fl.is_v ? P.v : P.k);
                const bool tall = H == 2 && fl.is_v;
                const int inc = tall ? 2 : 4;
                const long long step = inc * P.tok_stride, column = tall ? 16 * tu : fl.half * kDims + 16 * wu;
#pragma unroll 1
                for (int b = 0; b < 8; ++b) {
                    const int lane_of = tall ? 4 * fl.half + (b >> 1) : b, row0 = tall ? (b & 1) * 8 + 4 * part + tsub : 8 * part + wsub;      // whose page it is
                    const unsigned char *src = pool + __shfl_sync(0xffffffffu, off, lane_of) + row0 * P.tok_stride + column;
                    const int n = __shfl_sync(0xffffffffu, rows, lane_of) - row0;
#pragma unroll
                    for (int i = 0; i < 2; ++i, src += step) copy16(raw + b * 2048 + i * 512, inc * i < n ? src : pool, inc * i < n);
                }
            };
            int skip = 0;
            while (wk.next()) {
                const int fills = 2 * H * wk.nb;
                int j = (f + C::kStages - skip) % C::kStages;
                skip = (skip + fills) % C::kStages;
                if (j >= fills) continue;
                const long long head = wk.hk * P.head_stride;
                Fill fl = fill_of<H>(j, wk.nb);
                int t = (wk.blk + fl.block) * kTok + 16 * (lane & 7), at;      // lanes 0..7: sixteen tokens each
                int page = page_of(P, wk.b, t, wk.s.len, at);
                for (;;) {
                    const bool there = (unsigned)page < (unsigned)P.num_pages;
                    const long long off = there ? page * P.page_stride + head + at * P.tok_stride : 0ll;
                    const int rows = there ? wk.s.len - t : 0;
                    const Fill now = fl;
                    const bool more = j + C::kStages < fills;
                    if (more) {                                // the pages of the warp's next stage
                        fl = fill_of<H>(j + C::kStages, wk.nb);
                        t = (wk.blk + fl.block) * kTok + 16 * (lane & 7);
                        page = page_of(P, wk.b, t, wk.s.len, at);
                    }
                    // (the pair meets at a barrier: after a wait that ran out it walks on without waiting, as the softmax warps do)
                    if (ok && filled) ok = mbar_wait(s32(&S.empty[f]), (filled - 1) & 1, status, 40);
                    ok = __all_sync(0xffffffffu, ok);
                    fetch(now, off, rows);
                    asm volatile("cp.async.wait_all;" ::: "memory");
                    const bool tall = H == 2 && now.is_v;
                    const unsigned char *src = ring + f * kStageBytes + 16384 + part * 1024 + 16 * lane;
                    unsigned char *dst = ring + f * kStageBytes;
                    // wide: rows 16 b + 8 part + 4 i + wsub; tall: 8 b + 4 part + 2 i + tsub
                    const uint32_t at0 = tall ? tall_at[0] : wide_at[0] + part * 2048, at1 = tall ? tall_at[1] : wide_at[1] + part * 2048;
                    const auto write = [&](const uint4 &v, uint32_t to) {
                        uint4 one, two;
                        widen4<T>(pick(swap, v.z, v.x), one.x, one.y);
                        widen4<T>(pick(swap, v.w, v.y), one.z, one.w);
                        widen4<T>(pick(swap, v.x, v.z), two.x, two.y);
                        widen4<T>(pick(swap, v.y, v.w), two.z, two.w);
                        *reinterpret_cast<uint4 *>(dst + to) = one;
                        *reinterpret_cast<uint4 *>(dst + (to ^ 16)) = two;
                    };
                    // the first four quads become the lower half, which holds nothing; then both warps read the others and, when both
                    // have, write them over the upper half
#pragma unroll 1
                    for (int b = 0; b < 4; b += 2) {
                        uint4 x[4];
#pragma unroll
                        for (int i = 0; i < 4; ++i) x[i] = *reinterpret_cast<const uint4 *>(src + (b + (i >> 1)) * 2048 + (i & 1) * 512);
#pragma unroll
                        for (int i = 0; i < 4; ++i) write(x[i], (b + (i >> 1)) * 4096 + (i & 1 ? at1 : at0));
                    }
                    {
                        uint4 x[8];
#pragma unroll
                        for (int i = 0; i < 8; ++i) x[i] = *reinterpret_cast<const uint4 *>(src + (4 + (i >> 1)) * 2048 + (i & 1) * 512);
                        asm volatile("bar.sync %0, 64;" ::"r"(10 + f) : "memory");
#pragma unroll
                        for (int i = 0; i < 8; ++i) write(x[i], (4 + (i >> 1)) * 4096 + (i & 1 ? at1 : at0));
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s32(&(now.is_v ? S.v_full : S.k_full)[f]));
                    ++filled;
                    j += C::kStages;
                    if (!more) break;
                }
            }
        }
    }
    fence_before_sync();
    __syncthreads();
    if (warp == 1) {
        fence_after_sync();
        tmem_dealloc(tmem, 512);
    }
}

// Joins the partial results: CTA (c, y) takes the pair whose blocks begin in CTA c's piece and end behind it, 32 rows x 64
// dimensions of its tile; lane = row, a warp has eight dimensions; the result turns in shared memory.
constexpr int kMergeCols = 64;
template <typename T, int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ Params P) {
    __shared__ T turn[32][kMergeCols + 8];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int row0 = blockIdx.y / (HD / kMergeCols) * 32, col0 = blockIdx.y % (HD / kMergeCols) * kMergeCols;
    const int4 join = P.joins[blockIdx.x];
    if (join.x < 0) return;
    const int b = join.x, hk = join.y, parts = join.z, m = join.w >> 1;
    const Seq s = seq_of(P, b);
    const int rows = min(kM, s.rows - kM * m) - row0;          // of these 32
    if (rows <= 0) return;
    const int first = 2 * blockIdx.x + (join.w & 1), next = 2 * (blockIdx.x + 1);       // slots: first, next, next + 2, ..
    const int row = row0 + min(lane, rows - 1);
    const auto slot = [&](int k) { return (size_t)(k ? next + 2 * (k - 1) : first); };
    float top = -INFINITY;
#pragma unroll 4
    for (int k = 0; k < parts; ++k) top = fmaxf(top, __ldcg(P.part_ml + 2 * slot(k) * P.rows_ws + row));
    float acc[8] = {}, sum = 0.f;
#pragma unroll 2
    for (int k = 0; k < parts; ++k) {
        const float *const ml = P.part_ml + 2 * slot(k) * P.rows_ws + row;
        const float mk = __ldcg(ml), lk = __ldcg(ml + P.rows_ws);
        const float4 *const src = reinterpret_cast<const float4 *>(P.part_o) + (slot(k) * (HD / 4) + col0 / 4 + 2 * warp) * P.rows_ws + row;
        const float4 v0 = __ldcg(src), v1 = __ldcg(src + P.rows_ws);
        const float v[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
        if (mk != -INFINITY || lk != 0.f) {                    // parts in which the row saw nothing are zeros (a NaN is not)
            const float f = exp2f(mk - top);
            sum += lk * f;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] += v[e] * f;
        }
    }
    const float inv = sum == 0.f ? 0.f : P.v_scale / sum;
#pragma unroll
    for (int e = 0; e < 8; e += 2)
        *reinterpret_cast<uint32_t *>(&turn[lane][8 * warp + e]) = Type16<T>::pack(acc[e] * inv, acc[e + 1] * inv);
    __syncthreads();
    const int r = threadIdx.x >> 3, x = threadIdx.x & 7;       // eight lanes write the 128 bytes of a row
    if (r < rows) {
        const int R = kM * m + row0 + r, i = R / P.G;
        T *const out = static_cast<T *>(P.out) + (size_t)(s.first + i) * P.out_stride + (size_t)(hk * P.G + R - i * P.G) * HD + col0;
        *reinterpret_cast<uint4 *>(out + 8 * x) = *reinterpret_cast<const uint4 *>(&turn[r][8 * x]);
    }
}

// ---------------------------------------------------------------- host side
struct Sizes { int tiles, rows_ws; size_t joins, ml, total; };
static Sizes sizes_of(int G, int max_drafts, int hd) {
    Sizes z;
    const int rows = max_drafts * G;
    z.tiles = (rows + kM - 1) / kM;
    z.rows_ws = rows < kM ? (rows + 31) / 32 * 32 : kM;
    z.joins = (kMaxGrid * sizeof(int4) + 255) & ~(size_t)255;
    z.ml = ((size_t)2 * kMaxGrid * z.rows_ws * 8 + 255) & ~(size_t)255;
    z.total = z.joins + z.ml + (size_t)2 * kMaxGrid * z.rows_ws * hd * 4;
    return z;
}

template <typename T, bool FP8, int HD>
static int launch(const Params &P, cudaStream_t st) {
    using C = Cfg<FP8, HD>;
    auto kernel = tree_attn_kernel<T, FP8, HD>;
    static bool ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= 64 || !ready[dev]) {
        if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem) != cudaSuccess) {
            cudaGetLastError();
            return EXL3_E_LAUNCH;
        }
        if (dev >= 0 && dev < 64) ready[dev] = true;
    }
    if (launch_pdl(kernel, dim3(kMaxGrid), dim3(C::kThreads), C::kSmem, st, P) != cudaSuccess) return EXL3_E_LAUNCH;
    if (launch_pdl(tree_merge_kernel<T, HD>, dim3(kMaxGrid, P.rows_ws / 32 * (HD / kMergeCols)), dim3(256), 0, st, P) != cudaSuccess)
        return EXL3_E_LAUNCH;
    return launch_status();
}

__global__ void wait_selftest_kernel(unsigned long long limit_ns) {
    __shared__ __align__(8) unsigned long long bar;
    if (threadIdx.x == 0) {
        mbar_init(s32(&bar), 1);
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
    }
    __syncwarp();
    mbar_wait(s32(&bar), 0, &g_tree_status, 32, limit_ns);
}

}  // namespace tree
}  // namespace exl3

extern "C" size_t exl3_tree_attn_workspace_bytes(int batch, int q_heads, int max_drafts, const exl3_paged_cache *cache) {
    if (!cache || batch <= 0 || q_heads <= 0 || cache->kv_heads <= 0 || q_heads % cache->kv_heads || max_drafts < 1 ||
        max_drafts > EXL3_TREE_MAX_DRAFTS || (cache->head_dim != 128 && cache->head_dim != 256))
        return 0;
    return exl3::tree::sizes_of(q_heads / cache->kv_heads, max_drafts, cache->head_dim).total;
}

extern "C" int exl3_tree_attn(const void *q, long long q_stride, void *out, long long out_stride, const void *block_table,
                              int table_stride, int table_width, const void *seq_lens, const void *starts,
                              const void *mask, int batch, int tokens, int max_drafts, int q_heads, float scale,
                              int is_bf16, const exl3_paged_cache *cache, void *workspace, size_t workspace_bytes,
                              void *stream) {
    using namespace exl3;
    using namespace exl3::tree;
    if (!q || !out || !block_table || !seq_lens || !starts || !cache) return EXL3_E_NULL;
    const int rc = check_cache(*cache, is_bf16, true);
    if (rc != EXL3_OK) return rc;
    const int hd = cache->head_dim, kvh = cache->kv_heads;
    if (batch < 0 || batch > 65535 || tokens < 0 || q_heads <= 0 || q_heads > 65535 || q_heads % kvh || table_width <= 0 ||
        table_stride < table_width || (long long)table_width * cache->page_size > INT_MAX - 1024 || (q_stride & 7) ||
        (out_stride & 7) || q_stride < (long long)q_heads * hd || out_stride < (long long)q_heads * hd ||
        max_drafts < 1 || max_drafts > EXL3_TREE_MAX_DRAFTS ||
        (long long)batch * kvh * (((long long)table_width * cache->page_size + kTok - 1) / kTok + 1 + kMostChange) > INT_MAX)
        return EXL3_E_SHAPE;
    const float s2 = scale * cache->k_scale * 1.4426950408889634f;
    if (!(fabsf(s2) <= 3e38f)) return EXL3_E_SHAPE;
    if (q_heads / kvh > 2 * kMaxTiles) return EXL3_E_UNSUPPORTED;      // 64 drafts of as many heads are kMaxTiles tiles
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(starts, 4) ||
        !aligned(mask, 8))
        return EXL3_E_ALIGN;
    if (batch == 0 || tokens == 0) return EXL3_OK;
    const Sizes z = sizes_of(q_heads / kvh, max_drafts, hd);
    if (!workspace || workspace_bytes < z.total) return EXL3_E_WORKSPACE;
    if (!aligned(workspace, 16)) return EXL3_E_ALIGN;
    Params P = {};
    P.q = q; P.out = out; P.q_stride = q_stride; P.out_stride = out_stride;
    P.k = cache->k_pages; P.v = cache->v_pages;
    P.page_stride = cache->page_stride; P.head_stride = cache->head_stride; P.tok_stride = cache->token_stride;
    P.block_table = (const int *)block_table; P.seq_lens = (const int *)seq_lens; P.starts = (const int *)starts;
    P.mask = (const long long *)mask;
    P.bt_stride = table_stride; P.width = table_width; P.num_pages = cache->num_pages; P.page_size = cache->page_size;
    P.batch = batch; P.tokens = tokens; P.max_drafts = max_drafts; P.kvh = kvh; P.G = q_heads / kvh; P.tiles = z.tiles;
    P.negate = s2 < 0.f;
    P.scale_log2 = fmaxf(P.negate ? -s2 : s2, 1e-37f);       // (zero times the minus infinity of an unseen token would be NaN)
    P.v_scale = cache->v_scale;
    // Measured (us, with 0 / 1 / 2 / 3 / 4 places): 64 x 16 drafts 253 / 240 / 233 / 229 / 230, 61 drafts over 32768 tokens 80 / 79 /
    // 76 / 73 / 73, e4m3 71 / 60 / 59.5 / 60 / 62; 128 dimensions with 0 / 3 / 5 / 6 / 8: 127 / 107 / 100 / 102 / 106, e4m3 146 /
    // 124 / 119 / 120 / 122.
    P.change = hd == 128 ? kMostChange : cache->dtype == EXL3_KV_E4M3 ? 2 : 3;
    P.rows_ws = z.rows_ws;
    P.joins = (int4 *)workspace;
    P.part_ml = (float *)((char *)workspace + z.joins);
    P.part_o = (float *)((char *)workspace + z.joins + z.ml);
    const bool fp8 = cache->dtype == EXL3_KV_E4M3;
    cudaStream_t st = (cudaStream_t)stream;
    if (hd == 256) {
        if (is_bf16) return fp8 ? launch<__nv_bfloat16, true, 256>(P, st) : launch<__nv_bfloat16, false, 256>(P, st);
        return fp8 ? launch<__half, true, 256>(P, st) : launch<__half, false, 256>(P, st);
    }
    if (is_bf16) return fp8 ? launch<__nv_bfloat16, true, 128>(P, st) : launch<__nv_bfloat16, false, 128>(P, st);
    return fp8 ? launch<__half, true, 128>(P, st) : launch<__half, false, 128>(P, st);
}

extern "C" int exl3_tree_attn_status(unsigned *status_out) {
    if (!status_out) return EXL3_E_NULL;
    if (cudaMemcpyFromSymbol(status_out, exl3::tree::g_tree_status, sizeof(unsigned)) != cudaSuccess) { cudaGetLastError(); return EXL3_E_LAUNCH; }
    return EXL3_OK;
}
extern "C" int exl3_tree_attn_status_reset(void) {
    const unsigned v = 0;
    if (cudaMemcpyToSymbol(exl3::tree::g_tree_status, &v, sizeof(v)) != cudaSuccess) { cudaGetLastError(); return EXL3_E_LAUNCH; }
    return EXL3_OK;
}
extern "C" int exl3_tree_attn_selftest_wait(unsigned limit_us, void *stream) {
    if (limit_us == 0 || limit_us > 1000000u) return EXL3_E_SHAPE;
    exl3::tree::wait_selftest_kernel<<<1, 32, 0, static_cast<cudaStream_t>(stream)>>>((unsigned long long)limit_us * 1000ull);
    return exl3::launch_status();
}
