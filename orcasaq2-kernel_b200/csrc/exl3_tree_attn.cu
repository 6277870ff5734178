// Attention of a tree of drafted tokens over a paged KV cache, on tcgen05.mma.
//
// The query rows of a sequence and KV head (n drafts x G query heads) are the M side of the products, 128 rows (TMEM
// lanes) to a CTA; the cache is walked in blocks of 128 tokens:
//     S[row][token] = Q (shared memory) x K^T (shared memory, K-major)          fp32 in tensor memory
//     P = exp2(S * scale - m), rounded to 16 bits, in place of S                tensor memory
//     O[row][dim]  += P (tensor memory) x V (shared memory, MN-major: V lies [token][dim] as the cache has it)
// A row's statistics are one thread's: its TMEM lane holds all 128 scores of the block, no shuffles.
//
// What bounds it: K and V are read once per 128 rows, 4 * HD * 128 * 128 multiply-adds for 4 * HD * 128 bytes; at 128
// rows the tensor cores need a third of the time that HBM takes, so up to 128 rows the kernel's business is to keep
// loads in flight: a ring of 32 KB stages (128 tokens x 128 dimensions of K or of V) filled by TMA boxes of 8 tokens
// (eight rows of a swizzle atom; a page is a multiple of them), all boxes of a stage issued by one instruction of
// sixteen lanes.  More rows are more tiles: CTAs of the tiles of one sequence walk the same blocks at the same time
// and share them in L2.
// Work is split evenly whatever the lengths: the blocks of all (sequence, KV head) pairs form one line, every CTA
// takes an equal piece of it (found from the lengths on the device), and a pair that several CTAs share leaves partial
// sums with their maximum, which a second kernel joins in order (fixed order: the same bytes every run).
// The running maximum is only raised when it grows by more than 8 (a factor of 256 that the fp32 sums and the 16-bit
// probabilities hold easily), so O is seldom rescaled.
//
// Tokens nobody sees must not matter, whatever they hold: box rows behind the end and rows on pages outside the pool
// come in as zeros (TMA fill of an out-of-range page), the rest of the last box is zeroed, and non-finite V values of
// drafts, which some rows see and others do not, are zeroed before the product and added to the rows that see them at
// the end (a path that finite caches never take).
//
// e4m3 caches: raw stages, eight converter warps widen them exactly to the 16-bit type of q into the same swizzled
// stages; the scales fold into the softmax scale and the normalisation.
#include <cuda.h>
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
constexpr int kRawBytes = kTok * kDims;       // 16 KB of e4m3
constexpr int kMaxTiles = 32;
constexpr int kMaxGrid = 148;
constexpr int kConvWarps = 8;
constexpr float kRaise = 8.f;                 // log2 units the maximum may lag behind

static __device__ unsigned g_tree_status;     // sticky: non-zero after a bounded wait ran out

struct Params {
    const void *q;
    void *out;
    long long q_stride, out_stride;
    const void *v;                            // for the non-finite path only
    long long page_stride, head_stride, tok_stride;
    const int *block_table, *seq_lens, *starts;
    const long long *mask;
    int bt_stride, width, num_pages, page_size;
    int batch, tokens, max_drafts, kvh, G, tiles;    // tiles: of the sequence with the most drafts
    float scale_log2, v_scale;
    int negate;                               // the scale is negative: q is negated, scale_log2 is its size
    int rows_ws;                              // rows of a partial result
    int *plan;                                // [0..32) CTAs per tile, [32..64) blocks per tile, then per tile [batch + 1] prefix sums
    float *part_ml, *part_o;                  // [2 * grid][rows_ws][2], [2 * grid][rows_ws][HD]
};

template <bool FP8, int HD>
struct Cfg {
    static constexpr int kHalves = HD / kDims;                       // stages of a K or V block
    static constexpr int kQBytes = kM * HD * 2;
    static constexpr int kStages = FP8 ? 3 : (HD == 256 ? 5 : 6);
    static constexpr int kRaw = FP8 ? 4 : 0;
    static constexpr int kThreads = FP8 ? 256 + 32 * kConvWarps : 256;
    static constexpr int kSmem = kQBytes + kStages * kStageBytes + kRaw * kRawBytes + 1024 /*barriers*/ + 1024 /*alignment*/;
};

struct Shared {
    uint64_t full[6], empty[6], raw_full[4], raw_empty[4];
    uint64_t s_full[2], p_ready[2], v_here[2], pv_done[2], q_full, q_empty, o_free, drain;
    uint32_t tmem_base;
    int nonfinite;
    int total[kMaxTiles];
    int sums[16];
    int first_seq, first_off;
};
static_assert(sizeof(Shared) <= 1024, "shared state");

__device__ __forceinline__ void tma_5d(uint32_t dst, const CUtensorMap *map, int a, int b, int c, int d, int e, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];"
        ::"r"(dst), "l"(map), "r"(a), "r"(b), "r"(c), "r"(d), "r"(e), "r"(bar) : "memory");
}
__device__ __forceinline__ void tma_4d(uint32_t dst, const CUtensorMap *map, int a, int b, int c, int d, uint32_t bar) {
    asm volatile(
        "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], [%6];"
        ::"r"(dst), "l"(map), "r"(a), "r"(b), "r"(c), "r"(d), "r"(bar) : "memory");
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
    asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
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
__device__ __forceinline__ void softmax_sync() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

// ---------------------------------------------------------------- the line of blocks
struct Seq { int first, n, len, rows, blocks; };    // first row of q, drafts, tokens, query rows per KV head, blocks

__device__ __forceinline__ Seq seq_of(const Params &P, int b) {
    Seq s;
    const int lo = max(0, min(__ldg(P.starts + b), P.tokens)), hi = max(lo, min(__ldg(P.starts + b + 1), P.tokens));
    s.first = lo;
    s.n = hi - lo;
    s.len = max(0, min(__ldg(P.seq_lens + b), P.width * P.page_size));
    s.rows = min(s.n, P.max_drafts) * P.G;
    s.blocks = s.rows ? max(1, (s.len + kTok - 1) / kTok) : 0;
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
        if (left <= 0) return false;
        for (;;) {
            nblk = s.rows > kM * m ? s.blocks : 0;
            if (off < nblk * P.kvh) break;
            off -= nblk * P.kvh;
            if (++b >= P.batch) { left = 0; return false; }
            s = seq_of(P, b);
        }
        hk = off / nblk;
        blk = off - hk * nblk;
        nb = min(nblk - blk, left);
        off += nb;
        left -= nb;
        ++index;
        return true;
    }
    __device__ __forceinline__ bool whole() const { return nb == nblk; }
    __device__ __forceinline__ int rows() const { return min(kM, s.rows - kM * m); }
};

// CTAs of a tile out of `grid`, in proportion to its blocks (at least one).  Tiles of equal work get equal numbers, so
// that their CTAs walk the same blocks at the same time.  One thread; U[m] falls with m.
__device__ __forceinline__ int share_out(const int *U, int tiles, int grid, int m_wanted, int *m_of, int cta) {
    long long all = 0;
    for (int m = 0; m < tiles; ++m) all += U[m];
    int used = 0, first = 0;
    for (int m = 0; m < tiles; ++m) used += U[m] ? max(1, (int)((long long)grid * U[m] / all)) : 0;
    int at = 0;
    *m_of = -1;
    for (int m = 0; m < tiles; ++m) {
        int w = U[m] ? max(1, (int)((long long)grid * U[m] / all)) : 0;
        if (m == 0) w -= max(0, used - grid);
        if (m == m_wanted) first = at;
        if (cta >= at && cta < at + w) { *m_of = m; first = at; m_wanted = m; }
        at += w;
    }
    return first;
}
__device__ __forceinline__ int share_of(const int *U, int tiles, int grid, int m) {
    long long all = 0;
    int used = 0;
    for (int i = 0; i < tiles; ++i) all += U[i];
    for (int i = 0; i < tiles; ++i) used += U[i] ? max(1, (int)((long long)grid * U[i] / all)) : 0;
    const int w = U[m] ? max(1, (int)((long long)grid * U[m] / all)) : 0;
    return m == 0 ? w - max(0, used - grid) : w;
}
__device__ __forceinline__ int cut(int U, int W, int w) { return (int)((long long)U * w / W); }

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
tree_attn_kernel(const __grid_constant__ CUtensorMap kmap, const __grid_constant__ CUtensorMap vmap, const __grid_constant__ Params P) {
    using C = Cfg<FP8, HD>;
    constexpr int H = C::kHalves;
    constexpr int kThreads = C::kThreads;
    constexpr int kBox = FP8 ? 16 : 8;                       // tokens of a TMA box
    extern __shared__ unsigned char smem_dyn[];
    unsigned char *const smem = smem_dyn + ((1024u - (s32(smem_dyn) & 1023u)) & 1023u);
    unsigned char *const smQ = smem, *const ring = smQ + C::kQBytes, *const rawring = ring + C::kStages * kStageBytes;
    Shared &S = *reinterpret_cast<Shared *>(rawring + C::kRaw * kRawBytes);
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    unsigned *const status = &g_tree_status;

    if (tid == 0) {
        for (int i = 0; i < C::kStages; ++i) { mbar_init(s32(&S.full[i]), FP8 ? kConvWarps : 1); mbar_init(s32(&S.empty[i]), 1); }
        for (int i = 0; i < C::kRaw; ++i) { mbar_init(s32(&S.raw_full[i]), 1); mbar_init(s32(&S.raw_empty[i]), kConvWarps); }
        for (int i = 0; i < 2; ++i) { mbar_init(s32(&S.s_full[i]), 1); mbar_init(s32(&S.p_ready[i]), 4); mbar_init(s32(&S.v_here[i]), 1); mbar_init(s32(&S.pv_done[i]), 1); }
        mbar_init(s32(&S.q_full), 2); mbar_init(s32(&S.q_empty), 1);
        mbar_init(s32(&S.o_free), 4); mbar_init(s32(&S.drain), 1);
        S.nonfinite = 0;
        asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        fence_async();
    }
    if (tid < kMaxTiles) S.total[tid] = 0;
    if (warp == 1) tmem_alloc(s32(&S.tmem_base), 512);
    fence_before_sync();
    __syncthreads();
    fence_after_sync();
    const uint32_t tmem = S.tmem_base;
    asm volatile("griddepcontrol.wait;" ::: "memory");       // lengths, queries, cache rows of the kernels before
    asm volatile("griddepcontrol.launch_dependents;");

    // ---- this CTA's piece of the line
    for (int b0 = 0; b0 < P.batch; b0 += kThreads) {
        const int b = b0 + tid;
        int rows = 0, count = 0;
        if (b < P.batch) { const Seq s = seq_of(P, b); rows = s.rows; count = s.blocks * P.kvh; }
        for (int m = 0; m < P.tiles; ++m) {
            const int sum = __reduce_add_sync(0xffffffffu, rows > kM * m ? count : 0);
            if (lane == 0 && sum) atomicAdd(&S.total[m], sum);
        }
    }
    __syncthreads();
    int m;
    const int cta0 = share_out(S.total, P.tiles, gridDim.x, -1, &m, blockIdx.x);
    int u0 = 0, u1 = 0, w = 0;
    if (m >= 0) {
        w = blockIdx.x - cta0;
        const int W = share_of(S.total, P.tiles, gridDim.x, m);
        u0 = cut(S.total[m], W, w);
        u1 = cut(S.total[m], W, w + 1);
        if (w == 0 && tid == 0) { P.plan[m] = W; P.plan[kMaxTiles + m] = S.total[m]; }
    }
    if (blockIdx.x == 0 && tid < P.tiles && S.total[tid] == 0) { P.plan[tid] = 0; P.plan[kMaxTiles + tid] = 0; }
    if (m >= 0 && (u1 > u0 || w == 0)) {
        int carry = 0;
        for (int b0 = 0; b0 < P.batch; b0 += kThreads) {
            const int b = b0 + tid;
            int v = 0;
            if (b < P.batch) { const Seq s = seq_of(P, b); v = s.rows > kM * m ? s.blocks * P.kvh : 0; }
            int x = v;
#pragma unroll
            for (int o = 1; o < 32; o <<= 1) {
                const int y = __shfl_up_sync(0xffffffffu, x, o);
                if (lane >= o) x += y;
            }
            __syncthreads();
            if (lane == 31) S.sums[warp] = x;
            __syncthreads();
            int before = carry, all = 0;
            for (int i = 0; i < kThreads / 32; ++i) { if (i < warp) before += S.sums[i]; all += S.sums[i]; }
            const int excl = before + x - v;
            if (v && u0 >= excl && u0 < excl + v) { S.first_seq = b; S.first_off = u0 - excl; }
            if (w == 0) {
                int *const prefix = P.plan + 2 * kMaxTiles + (size_t)m * (P.batch + 1);
                if (b < P.batch) prefix[b] = excl;
                if (b == P.batch - 1) prefix[P.batch] = excl + v;
            }
            carry += all;
        }
    }
    __syncthreads();

    if (u1 > u0) {
        Walk wk(P, m, S.first_seq, S.first_off, u1 - u0);
        if (warp == 0) {
            // ---------------- producer: lane g fetches boxes of eight tokens (e4m3: sixteen)
            constexpr int kBoxes = kTok / kBox;
            constexpr int kSlots = FP8 ? C::kRaw : C::kStages;
            constexpr uint32_t kBytes = FP8 ? kRawBytes : kStageBytes;
            uint64_t *const full = FP8 ? S.raw_full : S.full, *const empty = FP8 ? S.raw_empty : S.empty;
            unsigned char *const slots = FP8 ? rawring : ring;
            Cursor rc(0, kSlots);
            int filled = 0;
            bool ok = true;
            const auto page_of = [&](int tok0) {           // this lane's page, or one outside the pool
                const int t = tok0 + (lane % kBoxes) * kBox;
                if (t >= wk.s.len) return P.num_pages;
                const int page = __ldg(P.block_table + (size_t)wk.b * P.bt_stride + t / P.page_size);
                return page >= 0 && page < P.num_pages ? page : P.num_pages;
            };
            const auto fetch = [&](const CUtensorMap *map, int tok0, int page) {
                for (int h = 0; h < H && ok; ++h, rc.advance(1), ++filled) {
                    if (lane == 0 && rc.wrapped) ok = mbar_wait(s32(&empty[rc.idx]), rc.phase ^ 1u, status, 20);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const uint32_t bar = s32(&full[rc.idx]);
                    if (lane == 0) mbar_expect_tx(bar, kBytes);
                    __syncwarp();
                    if (lane < kBoxes) {
                        const uint32_t dst = s32(slots + (size_t)rc.idx * kBytes) + lane * (kBytes / kBoxes);
                        const int at = (tok0 + lane * kBox) % P.page_size;
                        if constexpr (FP8) tma_4d(dst, map, h * kDims, at, wk.hk, page, bar);
                        else tma_5d(dst, map, 0, at, 2 * h, wk.hk, page, bar);
                    }
                }
            };
            while (ok && wk.next()) {
                const int t0 = wk.blk * kTok;
                int page = page_of(t0);
                fetch(&kmap, t0, page);
                for (int i = 0; i < wk.nb && ok; ++i) {
                    const int tok0 = t0 + i * kTok, ahead = i + 1 < wk.nb ? page_of(tok0 + kTok) : P.num_pages;
                    if (i + 1 < wk.nb) fetch(&kmap, tok0 + kTok, ahead);
                    fetch(&vmap, tok0, page);
                    page = ahead;
                }
            }
            // every copy issued has landed before the CTA goes (they have, unless a wait ran out)
            if (lane == 0)
                for (int f = max(0, filled - kSlots); f < filled; ++f) mbar_wait(s32(&full[f % kSlots]), (f / kSlots) & 1, status, 20);
        } else if (warp == 1) {
            // ---------------- the MMAs
            if (lane == 0) {
                constexpr uint32_t kType = __is_same(T, __half) ? 0u : (1u << 7 | 1u << 10);
                const uint32_t id_qk = umma_idesc_f16(kM, kTok) | kType, id_pv = umma_idesc_f16(kM, kDims) | kType | 1u << 16;
                Cursor rc(0, C::kStages);
                bool ok = true;
                int cnt = 0;                                   // blocks whose probabilities were used
                const auto scores = [&](int n) {               // S(n) = Q K^T
                    const uint32_t d = tmem + HD + (n & 1) * kTok;
                    for (int h = 0; h < H && ok; ++h, rc.advance(1)) {
                        ok = mbar_wait(s32(&S.full[rc.idx]), rc.phase, status);
                        if (!ok) return;
                        fence_after_sync();
                        const uint32_t kb = s32(ring + (size_t)rc.idx * kStageBytes);
#pragma unroll
                        for (int k = 0; k < kDims / 16; ++k)
                            umma_f16_ss(d, desc_sw128(s32(smQ) + (2 * h + k / 4) * (kM * 128) + (k % 4) * 32, 16, 1024),
                                        desc_sw128(kb + (k / 4) * 1024 + (k % 4) * 32, 16, 2048), id_qk, h || k);
                        umma_commit(s32(&S.empty[rc.idx]));
                    }
                    umma_commit(s32(&S.s_full[n & 1]));
                };
                while (ok && wk.next()) {
                    ok = mbar_wait(s32(&S.q_full), wk.index & 1, status);
                    if (!ok) break;
                    fence_after_sync();
                    scores(cnt);
                    if (wk.nb == 1) umma_commit(s32(&S.q_empty));
                    for (int i = 0; i < wk.nb && ok; ++i, ++cnt) {
                        if (i + 1 < wk.nb) {
                            scores(cnt + 1);
                            if (i + 2 == wk.nb) umma_commit(s32(&S.q_empty));
                        }
                        Cursor vc = rc;
                        for (int h = 0; h < H && ok; ++h, vc.advance(1)) ok = mbar_wait(s32(&S.full[vc.idx]), vc.phase, status);
                        if (ok) mbar_arrive(s32(&S.v_here[cnt & 1]));
                        if (ok) ok = mbar_wait(s32(&S.p_ready[cnt & 1]), (cnt >> 1) & 1, status);
                        if (ok && i == 0 && wk.index) ok = mbar_wait(s32(&S.o_free), (wk.index - 1) & 1, status);
                        if (!ok) break;
                        fence_after_sync();
                        for (int h = 0; h < H; ++h, rc.advance(1)) {
                            const uint32_t vb = s32(ring + (size_t)rc.idx * kStageBytes);
                            const uint32_t p = tmem + HD + (cnt & 1) * kTok;
#pragma unroll
                            for (int k = 0; k < kTok / 16; ++k)
                                umma_f16_ts(tmem + h * kDims, p + 8 * k, desc_sw128(vb + k * 4096, 1024, 2048), id_pv, i || k);
                            umma_commit(s32(&S.empty[rc.idx]));
                        }
                        umma_commit(s32(&S.pv_done[cnt & 1]));
                    }
                }
                umma_commit(s32(&S.drain));
                mbar_wait(s32(&S.drain), 0, status);
            }
        } else if (warp < 4) {
            // ---------------- query rows into shared memory (swizzled, K-major), rows behind the last one zero
            bool ok = true;
            constexpr int kUnits = HD / 8;                     // 16-byte units of a row
            while (ok && wk.next()) {
                if (wk.index) {
                    ok = mbar_wait(s32(&S.q_empty), (wk.index - 1) & 1, status, 20);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                }
                const int rows = wk.rows();
                const uint32_t flip = P.negate ? 0x80008000u : 0u;
                for (int e = (warp - 2) * 32 + lane; e < kM * kUnits; e += 64) {
                    const int r = e / kUnits, u = e - r * kUnits, c = u >> 3;
                    uint4 x = make_uint4(0, 0, 0, 0);
                    if (r < rows) {
                        const int R = kM * m + r, i = R / P.G, g = R - i * P.G;
                        x = *reinterpret_cast<const uint4 *>(static_cast<const T *>(P.q) + (size_t)(wk.s.first + i) * P.q_stride +
                                                             (size_t)(wk.hk * P.G + g) * HD + 8 * u);
                        x.x ^= flip; x.y ^= flip; x.z ^= flip; x.w ^= flip;
                    }
                    *reinterpret_cast<uint4 *>(smQ + c * (kM * 128) + r * 128 + (((u & 7) ^ (r & 7)) << 4)) = x;
                }
                fence_async();
                __syncwarp();
                if (lane == 0) mbar_arrive(s32(&S.q_full));
            }
        } else if (warp < 8) {
            // ---------------- softmax: thread = row = TMEM lane
            const int row = tid - 128;
            const uint32_t lane_base = (uint32_t)(32 * (warp & 3)) << 16;
            bool ok = true;
            int cnt = 0, pos = 0;                              // blocks done; ring position of the segment
            while (ok && wk.next()) {
                const int R = kM * m + row, draft = R / P.G;
                const bool live = row < wk.rows();
                const int ctx = wk.s.len - wk.s.n;             // first draft's token (negative: drafts that have none)
                unsigned long long bits = 0;
                if (live) bits = P.mask ? (unsigned long long)__ldg(P.mask + wk.s.first + draft) : (draft >= 63 ? ~0ull : (2ull << draft) - 1);
                float top = -INFINITY, sum = 0.f;
                const auto page_ok = [&](int tok0) {           // lanes 0..15: is the page of eight tokens in the pool?
                    const int t = tok0 + (lane & 15) * 8;
                    if (t >= wk.s.len) return true;
                    const int page = __ldg(P.block_table + (size_t)wk.b * P.bt_stride + t / P.page_size);
                    return page >= 0 && page < P.num_pages;
                };
                bool pages = page_ok(wk.blk * kTok);
                for (int i = 0; i < wk.nb && ok; ++i, ++cnt) {
                    const int tok0 = (wk.blk + i) * kTok;
                    const uint32_t groups = __ballot_sync(0xffffffffu, pages) & 0xFFFFu;
                    if (i + 1 < wk.nb) pages = page_ok(tok0 + kTok);
                    const bool masked = tok0 + kTok > ctx || groups != 0xFFFFu;        // uniform in the four warps
                    uint32_t vis[4] = {~0u, ~0u, ~0u, ~0u};
                    if (masked) {
#pragma unroll
                        for (int k = 0; k < 4; ++k) {
                            const int a = tok0 + 32 * k;
                            uint32_t v = 0;
                            // context tokens of these 32, then the drafts' bits shifted to their places
                            const int c = ctx - a, l = wk.s.len - a;
                            if (c >= 32) v = ~0u;
                            else if (c > 0) v = (1u << c) - 1 | (uint32_t)(bits << c);
                            else v = -c < 64 ? (uint32_t)(bits >> -c) : 0u;
                            if (l < 32) v &= l > 0 ? (1u << l) - 1 : 0u;
                            const uint32_t g4 = groups >> (4 * k) & 15u;
                            v &= (g4 & 1 ? 0xFFu : 0u) | (g4 & 2 ? 0xFF00u : 0u) | (g4 & 4 ? 0xFF0000u : 0u) | (g4 & 8 ? 0xFF000000u : 0u);
                            vis[k] = live ? v : 0u;
                        }
                    }
                    const uint32_t s_t = tmem + lane_base + HD + (cnt & 1) * kTok;
                    ok = __all_sync(0xffffffffu, mbar_wait(s32(&S.s_full[cnt & 1]), (cnt >> 1) & 1, status));
                    if (!ok) break;
                    fence_after_sync();
                    float mx = -INFINITY;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t x[32];
                        tmem_ld32(s_t + 32 * k, x);
                        if (masked) {
#pragma unroll
                            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, vis[k] >> e & 1 ? __uint_as_float(x[e]) : -INFINITY);
                        } else {
#pragma unroll
                            for (int e = 0; e < 32; ++e) mx = fmaxf(mx, __uint_as_float(x[e]));
                        }
                    }
                    mx = mx == -INFINITY ? mx : mx * P.scale_log2;
                    const bool raise = mx > top + kRaise || (top == -INFINITY && mx > top);
                    if (__any_sync(0xffffffffu, raise)) {
                        const float corr = raise ? ex2(top - mx) : 1.f;      // 0 when nothing was seen before
                        if (raise) { top = mx; sum *= corr; }
                        if (i > 0) {
                            ok = __all_sync(0xffffffffu, mbar_wait(s32(&S.pv_done[(cnt - 1) & 1]), ((cnt - 1) >> 1) & 1, status));
                            if (!ok) break;
                            fence_after_sync();
#pragma unroll
                            for (int c = 0; c < HD; c += 32) {
                                uint32_t o[32];
                                tmem_ld32(tmem + lane_base + c, o);
#pragma unroll
                                for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * corr);
                                tmem_st32(tmem + lane_base + c, o);
                            }
                        }
                    }
                    const float shift = top == -INFINITY ? 0.f : top;
#pragma unroll
                    for (int k = 0; k < 4; ++k) {
                        uint32_t x[32], p[16];
                        tmem_ld32(s_t + 32 * k, x);
#pragma unroll
                        for (int e = 0; e < 16; ++e) {
                            float a = ex2(fmaf(__uint_as_float(x[2 * e]), P.scale_log2, -shift));
                            float c = ex2(fmaf(__uint_as_float(x[2 * e + 1]), P.scale_log2, -shift));
                            if (masked) {
                                if (!(vis[k] >> (2 * e) & 1)) a = 0.f;
                                if (!(vis[k] >> (2 * e + 1) & 1)) c = 0.f;
                            }
                            sum += a + c;
                            p[e] = Type16<T>::pack(a, c);
                        }
                        tmem_st16(s_t + 16 * k, p);            // over scores that were read
                    }
                    if (tok0 + kTok > ctx) {
                        // rows of V behind the end become zeros, non-finite values of drafts too (see the top of the file)
                        const int from = max(0, ctx - tok0), have = min(kTok, wk.s.len - tok0), upto = min(kTok, (have + kBox - 1) & ~(kBox - 1));
                        const int vpos = pos + H + 2 * H * i + (i + 1 < wk.nb ? H : 0);
                        // (announced by the MMA thread, which looks at every stage in its turn: the stage's own barrier may
                        // still be a whole round behind, or ahead, of what this thread would wait for)
                        ok = __all_sync(0xffffffffu, mbar_wait(s32(&S.v_here[cnt & 1]), (cnt >> 1) & 1, status));
                        if (!ok) break;
                        for (int h = 0; h < H; ++h) {
                            const int st = (vpos + h) % C::kStages;
                            for (int e = row; e < (upto - from) * 16; e += 128) {
                                const int r = from + (e >> 4), u = e & 15;
                                uint4 *const at = reinterpret_cast<uint4 *>(ring + (size_t)st * kStageBytes + (r >> 3) * 2048 + (u >> 3) * 1024 +
                                                                            (r & 7) * 128 + (((u & 7) ^ (r & 7)) << 4));
                                if (r >= have) {
                                    *at = make_uint4(0, 0, 0, 0);
                                } else {
                                    uint4 x = *at, y;
                                    const bool a = nonfinite2<T>(x.x, y.x), b2 = nonfinite2<T>(x.y, y.y), c = nonfinite2<T>(x.z, y.z),
                                               d = nonfinite2<T>(x.w, y.w);
                                    if (a || b2 || c || d) { *at = y; S.nonfinite = 1; }
                                }
                            }
                        }
                        fence_async();
                    }
                    tmem_wait_st();
                    fence_before_sync();
                    __syncwarp();
                    if (lane == 0) mbar_arrive(s32(&S.p_ready[cnt & 1]));
                }
                if (!ok) break;
                // ---- the segment's result
                ok = __all_sync(0xffffffffu, mbar_wait(s32(&S.pv_done[(cnt - 1) & 1]), ((cnt - 1) >> 1) & 1, status));
                if (!ok) break;
                fence_after_sync();
                softmax_sync();
                const bool mend = S.nonfinite != 0;            // uniform: all have written it before the barrier
                const bool whole = wk.whole();
                const float inv = sum == 0.f ? 0.f : P.v_scale / sum;
                const int slot = 2 * blockIdx.x + (wk.index ? 1 : 0);
                T *const orow = static_cast<T *>(P.out) + (size_t)(wk.s.first + draft) * P.out_stride + (size_t)(wk.hk * P.G + R - draft * P.G) * HD;
                float *const prow = P.part_o + ((size_t)slot * P.rows_ws + row) * HD;
#pragma unroll 1
                for (int c = 0; c < HD; c += 32) {
                    uint32_t o[32];
                    tmem_ld32(tmem + lane_base + c, o);
                    if (mend && live) {
                        const int t_end = min(wk.s.len, (wk.blk + wk.nb) * kTok);
                        for (int t = max(max(0, ctx), wk.blk * kTok); t < t_end; ++t) {
                            if (t - ctx > 63 || !(bits >> (t - ctx) & 1)) continue;
                            const int page = __ldg(P.block_table + (size_t)wk.b * P.bt_stride + t / P.page_size);
                            if (page < 0 || page >= P.num_pages) continue;
                            const size_t at = (size_t)page * P.page_stride + (size_t)wk.hk * P.head_stride + (size_t)(t % P.page_size) * P.tok_stride + c;
#pragma unroll
                            for (int e = 0; e < 32; ++e) {
                                float x;
                                if constexpr (FP8) x = (float)static_cast<const __nv_fp8_e4m3 *>(P.v)[at + e];
                                else x = (float)static_cast<const T *>(P.v)[at + e];
                                if (!isfinite(x)) o[e] = __float_as_uint(__uint_as_float(o[e]) + x);
                            }
                        }
                    }
                    if (live && whole) {
#pragma unroll
                        for (int e = 0; e < 32; e += 8) {
                            uint4 r;
                            r.x = Type16<T>::pack(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv);
                            r.y = Type16<T>::pack(__uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
                            r.z = Type16<T>::pack(__uint_as_float(o[e + 4]) * inv, __uint_as_float(o[e + 5]) * inv);
                            r.w = Type16<T>::pack(__uint_as_float(o[e + 6]) * inv, __uint_as_float(o[e + 7]) * inv);
                            *reinterpret_cast<uint4 *>(orow + c + e) = r;
                        }
                    } else if (live) {
#pragma unroll
                        for (int e = 0; e < 32; e += 4)
                            *reinterpret_cast<uint4 *>(prow + c + e) = make_uint4(o[e], o[e + 1], o[e + 2], o[e + 3]);
                    }
                    __syncwarp();
                }
                if (live && !whole) *reinterpret_cast<float2 *>(P.part_ml + ((size_t)slot * P.rows_ws + row) * 2) = make_float2(top, sum);
                fence_before_sync();
                softmax_sync();
                if (row == 0) S.nonfinite = 0;
                softmax_sync();
                if (lane == 0) mbar_arrive(s32(&S.o_free));
                pos += 2 * H * wk.nb;
            }
        } else if constexpr (FP8) {
            // ---------------- e4m3 stages -> 16-bit stages: sixteen bytes per thread and step, two units of the swizzled row
            const int ct = tid - 256;
            Cursor rc(0, C::kRaw), cc(0, C::kStages);
            bool ok = true;
            while (ok && wk.next()) {
                for (int i = 0; i < 2 * H * wk.nb && ok; ++i, rc.advance(1), cc.advance(1)) {
                    ok = mbar_wait(s32(&S.raw_full[rc.idx]), rc.phase, status, 20);
                    if (ok && cc.wrapped) ok = mbar_wait(s32(&S.empty[cc.idx]), cc.phase ^ 1u, status, 20);
                    ok = __all_sync(0xffffffffu, ok);
                    if (!ok) break;
                    const unsigned char *const src = rawring + (size_t)rc.idx * kRawBytes;
                    unsigned char *const dst = ring + (size_t)cc.idx * kStageBytes;
                    uint4 x[4];
#pragma unroll
                    for (int j = 0; j < 4; ++j) x[j] = *reinterpret_cast<const uint4 *>(src + 16 * (ct + 256 * j));
#pragma unroll
                    for (int j = 0; j < 4; ++j) {
                        const int e = ct + 256 * j, r = e >> 3, u = e & 7;
                        uint4 a, b;
                        widen4<T>(x[j].x, a.x, a.y);
                        widen4<T>(x[j].y, a.z, a.w);
                        widen4<T>(x[j].z, b.x, b.y);
                        widen4<T>(x[j].w, b.z, b.w);
                        unsigned char *const at = dst + (r >> 3) * 2048 + (u >> 2) * 1024 + (r & 7) * 128;
                        const int k = (u & 3) * 2;
                        // the two halves of a row's lanes start with different units: no bank conflicts
                        const bool swap = u & 4;
                        *reinterpret_cast<uint4 *>(at + (((k + (swap ? 1 : 0)) ^ (r & 7)) << 4)) = swap ? b : a;
                        *reinterpret_cast<uint4 *>(at + (((k + (swap ? 0 : 1)) ^ (r & 7)) << 4)) = swap ? a : b;
                    }
                    fence_async();
                    __syncwarp();
                    if (lane == 0) { mbar_arrive(s32(&S.raw_empty[rc.idx])); mbar_arrive(s32(&S.full[cc.idx])); }
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

// Joins the partial results: CTA (c, y) takes the pair whose blocks begin in CTA c's piece and end behind it, eight rows of
// its tile, one warp per row.
template <typename T, int HD>
__global__ void __launch_bounds__(256) tree_merge_kernel(const __grid_constant__ Params P) {
    constexpr int kVec = HD / 128;                             // float4 per lane
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int lane = threadIdx.x & 31, row = blockIdx.y * 8 + (threadIdx.x >> 5);
    int m = 0, cta0 = 0;
    while (m < P.tiles && (int)blockIdx.x >= cta0 + P.plan[m]) cta0 += P.plan[m++];
    if (m >= P.tiles) return;
    const int W = P.plan[m], U = P.plan[kMaxTiles + m], w = blockIdx.x - cta0;
    const int u0 = cut(U, W, w), u1 = cut(U, W, w + 1);
    if (u1 <= u0 || w + 1 >= W) return;
    const int *const prefix = P.plan + 2 * kMaxTiles + (size_t)m * (P.batch + 1);
    int lo = 0, hi = P.batch - 1;
    while (lo < hi) {                                          // last sequence that begins at or before the piece's last block
        const int mid = (lo + hi + 1) >> 1;
        if (prefix[mid] <= u1 - 1) lo = mid; else hi = mid - 1;
    }
    const int b = lo, base = prefix[b], nblk = (prefix[b + 1] - base) / P.kvh;
    if (nblk <= 0) return;
    const int hk = (u1 - 1 - base) / nblk, begin = base + hk * nblk, end = begin + nblk;
    if (begin < u0 || end <= u1) return;
    const Seq s = seq_of(P, b);
    if (row >= min(kM, s.rows - kM * m)) return;
    int last = w + 1;                                          // the CTAs w .. last hold parts of it
    while (last + 1 < W && cut(U, W, last + 1) < end) ++last;
    const auto slot = [&](int k) { return (size_t)(2 * (cta0 + k) + (k == w && begin != u0 ? 1 : 0)) * P.rows_ws + row; };
    float top = -INFINITY;
    for (int k = w + lane; k <= last; k += 32)
        if (cut(U, W, k) < cut(U, W, k + 1)) top = fmaxf(top, __ldcg(P.part_ml + 2 * slot(k)));
#pragma unroll
    for (int o = 16; o; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
    float4 acc[kVec];
#pragma unroll
    for (int v = 0; v < kVec; ++v) acc[v] = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
    for (int k0 = w; k0 <= last; k0 += 32) {
        float wt = 0.f, l = 0.f;
        bool has = false;
        if (k0 + lane <= last && cut(U, W, k0 + lane) < cut(U, W, k0 + lane + 1)) {
            const float2 ml = __ldcg(reinterpret_cast<const float2 *>(P.part_ml + 2 * slot(k0 + lane)));
            has = ml.x != -INFINITY || ml.y != 0.f;            // parts in which the row saw nothing are zeros (a NaN is not)
            wt = has ? exp2f(ml.x - top) : 0.f;
            l = has ? ml.y * wt : 0.f;
        }
#pragma unroll
        for (int o = 16; o; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        sum += l;
        const uint32_t any = __ballot_sync(0xffffffffu, has);
        const int count = min(32, last - k0 + 1);
#pragma unroll 4
        for (int j = 0; j < count; ++j) {
            const float f = __shfl_sync(0xffffffffu, wt, j);
            if (!(any >> j & 1)) continue;
            const float4 *const src = reinterpret_cast<const float4 *>(P.part_o + slot(k0 + j) * HD) + lane;
#pragma unroll
            for (int v = 0; v < kVec; ++v) {
                const float4 x = __ldcg(src + 32 * v);
                acc[v].x += x.x * f; acc[v].y += x.y * f; acc[v].z += x.z * f; acc[v].w += x.w * f;
            }
        }
    }
    const float inv = sum == 0.f ? 0.f : P.v_scale / sum;
    const int R = kM * m + row, i = R / P.G;
    T *const out = static_cast<T *>(P.out) + (size_t)(s.first + i) * P.out_stride + (size_t)(hk * P.G + R - i * P.G) * HD;
#pragma unroll
    for (int v = 0; v < kVec; ++v) {
        uint2 r;
        r.x = Type16<T>::pack(acc[v].x * inv, acc[v].y * inv);
        r.y = Type16<T>::pack(acc[v].z * inv, acc[v].w * inv);
        *reinterpret_cast<uint2 *>(out + 128 * v + 4 * lane) = r;
    }
}

// ---------------------------------------------------------------- host side
using EncodeTiledFn = CUresult (*)(CUtensorMap *, CUtensorMapDataType, cuuint32_t, void *, const cuuint64_t *,
                                   const cuuint64_t *, const cuuint32_t *, const cuuint32_t *, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);
static EncodeTiledFn encode_fn() {
    static EncodeTiledFn fn = nullptr;
    if (!fn) {
        void *p = nullptr;
        cudaDriverEntryPointQueryResult q;
        if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
            q == cudaDriverEntryPointSuccess)
            fn = reinterpret_cast<EncodeTiledFn>(p);
        else
            cudaGetLastError();
    }
    return fn;
}

// 16-bit pools: (64 values, token, 64-value chunk, head, page), boxes of 8 tokens x 2 chunks, 128-byte swizzle: a box is two
// 1 KB swizzle atoms.  e4m3 pools: (byte, token, head, page), boxes of 16 tokens x 128 bytes, as they lie.
static bool make_map(CUtensorMap *map, void *pool, const exl3_paged_cache &c) {
    const EncodeTiledFn fn = encode_fn();
    if (!fn) return false;
    const bool fp8 = c.dtype == EXL3_KV_E4M3;
    const cuuint64_t e = fp8 ? 1 : 2;
    const cuuint64_t hd = c.head_dim, page = c.page_size, heads = c.kv_heads, pages = c.num_pages;
    const cuuint64_t ts = c.token_stride * e, hs = c.head_stride * e, ps = c.page_stride * e;
    const cuuint32_t one[5] = {1, 1, 1, 1, 1};
    if (fp8) {
        const cuuint64_t dims[4] = {hd, page, heads, pages}, strides[3] = {ts, hs, ps};
        const cuuint32_t box[4] = {kDims, 16, 1, 1};
        return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 4, pool, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
                  CU_TENSOR_MAP_SWIZZLE_NONE, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
    }
    const cuuint64_t dims[5] = {64, page, hd / 64, heads, pages}, strides[4] = {ts, 128, hs, ps};
    const cuuint32_t box[5] = {64, 8, 2, 1, 1};
    return fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT16, 5, pool, dims, strides, box, one, CU_TENSOR_MAP_INTERLEAVE_NONE,
              CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

struct Sizes { int tiles, rows_ws; size_t plan, ml, total; };
static Sizes sizes_of(int batch, int G, int max_drafts, int hd) {
    Sizes z;
    const int rows = max_drafts * G;
    z.tiles = (rows + kM - 1) / kM;
    z.rows_ws = rows < kM ? rows : kM;
    z.plan = ((size_t)(2 * kMaxTiles + (size_t)z.tiles * (batch + 1)) * 4 + 255) & ~(size_t)255;
    z.ml = ((size_t)2 * kMaxGrid * z.rows_ws * 8 + 255) & ~(size_t)255;
    z.total = z.plan + z.ml + (size_t)2 * kMaxGrid * z.rows_ws * hd * 4;
    return z;
}

template <typename T, bool FP8, int HD>
static int launch(const CUtensorMap &kmap, const CUtensorMap &vmap, const Params &P, cudaStream_t st) {
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
    if (launch_pdl(kernel, dim3(kMaxGrid), dim3(C::kThreads), C::kSmem, st, kmap, vmap, P) != cudaSuccess) return EXL3_E_LAUNCH;
    if (launch_pdl(tree_merge_kernel<T, HD>, dim3(kMaxGrid, (P.rows_ws + 7) / 8), dim3(256), 0, st, P) != cudaSuccess)
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
    return exl3::tree::sizes_of(batch, q_heads / cache->kv_heads, max_drafts, cache->head_dim).total;
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
        (long long)batch * kvh * (((long long)table_width * cache->page_size + kTok - 1) / kTok + 1) > INT_MAX)
        return EXL3_E_SHAPE;
    if (q_heads / kvh > 64) return EXL3_E_UNSUPPORTED;
    if (!aligned(q, 16) || !aligned(out, 16) || !aligned(block_table, 4) || !aligned(seq_lens, 4) || !aligned(starts, 4) ||
        !aligned(mask, 8))
        return EXL3_E_ALIGN;
    if (batch == 0 || tokens == 0) return EXL3_OK;
    const Sizes z = sizes_of(batch, q_heads / kvh, max_drafts, hd);
    if (!workspace || workspace_bytes < z.total) return EXL3_E_WORKSPACE;
    if (!aligned(workspace, 16)) return EXL3_E_ALIGN;
    Params P = {};
    P.q = q; P.out = out; P.q_stride = q_stride; P.out_stride = out_stride;
    P.v = cache->v_pages;
    P.page_stride = cache->page_stride; P.head_stride = cache->head_stride; P.tok_stride = cache->token_stride;
    P.block_table = (const int *)block_table; P.seq_lens = (const int *)seq_lens; P.starts = (const int *)starts;
    P.mask = (const long long *)mask;
    P.bt_stride = table_stride; P.width = table_width; P.num_pages = cache->num_pages; P.page_size = cache->page_size;
    P.batch = batch; P.tokens = tokens; P.max_drafts = max_drafts; P.kvh = kvh; P.G = q_heads / kvh; P.tiles = z.tiles;
    const float s2 = scale * cache->k_scale * 1.4426950408889634f;
    P.negate = s2 < 0.f;
    P.scale_log2 = P.negate ? -s2 : s2;
    P.v_scale = cache->v_scale;
    P.rows_ws = z.rows_ws;
    P.plan = (int *)workspace;
    P.part_ml = (float *)((char *)workspace + z.plan);
    P.part_o = (float *)((char *)workspace + z.plan + z.ml);
    CUtensorMap kmap, vmap;
    if (!make_map(&kmap, cache->k_pages, *cache) || !make_map(&vmap, cache->v_pages, *cache)) return EXL3_E_LAUNCH;
    const bool fp8 = cache->dtype == EXL3_KV_E4M3;
    cudaStream_t st = (cudaStream_t)stream;
    if (hd == 256) {
        if (is_bf16) return fp8 ? launch<__nv_bfloat16, true, 256>(kmap, vmap, P, st) : launch<__nv_bfloat16, false, 256>(kmap, vmap, P, st);
        return fp8 ? launch<__half, true, 256>(kmap, vmap, P, st) : launch<__half, false, 256>(kmap, vmap, P, st);
    }
    if (is_bf16) return fp8 ? launch<__nv_bfloat16, true, 128>(kmap, vmap, P, st) : launch<__nv_bfloat16, false, 128>(kmap, vmap, P, st);
    return fp8 ? launch<__half, true, 128>(kmap, vmap, P, st) : launch<__half, false, 128>(kmap, vmap, P, st);
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
