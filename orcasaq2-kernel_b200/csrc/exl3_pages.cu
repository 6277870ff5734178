// Pages of a KV cache kept on the device: fork (share full pages, copy the partial one), reserve (pages and slots for
// new tokens), accept (the accepted path of a draft tree moved to the front of its place), free.  All in the order of
// a stream, nothing returns to the host, so a whole speculative step can be one CUDA graph.
//
// Bookkeeping: `free_list` is a stack of page numbers (counters[0] of them), `refs` counts the sequences that hold a
// page.  Every call takes or returns pages for all its sequences at once: what sequence i needs is known from its
// lengths, an exclusive prefix sum over the call gives its place in the stack, and so the result is the one that
// serving the sequences in the order of the call would give, whatever order the threads run in, with one exception: once
// the stack is too short for a sequence, none behind it takes pages, though fewer might do for it (its place in the
// stack lies behind the place of the one that got none).  For fork and reserve this is a few hundred bytes of work bound
// by latency: one CTA, one thread per sequence.  free passes four times over every entry of its sequences' rows of the
// table in that one CTA: 9 us for 64 pages in all, 62 us for 64 sequences of 256, 481 us for 64 of 2048.
// Data: rows (one token of one head) are moved with 16-byte accesses for all pools (K and V of every layer) in one
// launch; bound by HBM: the rows are written once per child and read once per parent (its children's CTAs find them in
// L2).  Sixteen parents' partial pages for 96 children, 482 MB written, 80 read: 125 us, what a plain fill of 482 MB takes.
//
// What cannot be served is not an error of the call (the host does not wait for it): a sequence for which no pages
// are left, or whose arguments do not fit its state, stays as it was and a bit of counters[1] is set.
#include <cuda_runtime.h>
#include <limits.h>
#include <stdint.h>

#include "exl3_common.cuh"
#include "exl3_paged.cuh"

namespace exl3 {

constexpr int kMaxCall = EXL3_PAGES_MAX_SEQS;    // sequences of one call: one thread each
constexpr int kBookThreads = 1024;
static_assert(kMaxCall == kBookThreads, "one thread per sequence");

struct Tables {
    int *block_table, *seq_lens, *held, *refs, *free_list, *counters;
    int bt_stride, width, max_seqs, num_pages, page_size;
};

// Exclusive prefix sum over the CTA; *total receives the sum.
__device__ __forceinline__ int block_scan(int v, int *warp_sums, int *total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    int x = v;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, x, o);
        if (lane >= o) x += y;
    }
    __syncthreads();                               // warp_sums may still be read from the scan before
    if (lane == 31) warp_sums[warp] = x;
    __syncthreads();
    if (warp == 0) {
        int s = warp_sums[lane];
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int y = __shfl_up_sync(0xffffffffu, s, o);
            if (lane >= o) s += y;
        }
        warp_sums[lane] = s;
    }
    __syncthreads();
    *total = warp_sums[31];
    return x - v + (warp ? warp_sums[warp - 1] : 0);
}

// The last sequence i of n whose exclusive prefix starts[i] is <= e (entries are numbered through all sequences).
__device__ __forceinline__ int owner_of(const int *starts, int n, int e) {
    int lo = 0, hi = n - 1;
    while (lo < hi) {
        const int mid = (lo + hi + 1) >> 1;
        if (starts[mid] <= e) lo = mid; else hi = mid - 1;
    }
    return lo;
}

// ---------------------------------------------------------------- fork
struct ForkPlan { int parent, child, full, rest, src, dst; };    // child < 0: nothing to do; dst < 0: no partial page

struct ForkParams {
    Tables t;
    const int *parents, *children;
    ForkPlan *plan;
    int n;
};

__global__ void __launch_bounds__(kBookThreads) fork_plan_kernel(const __grid_constant__ ForkParams P) {
    __shared__ int par_s[kMaxCall], kid_s[kMaxCall], sums[32];
    const Tables &T = P.t;
    const int i = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int left = min(max(T.counters[0], 0), T.num_pages);
    int p = -1, c = -1;
    if (i < P.n) { p = P.parents[i]; c = P.children[i]; }
    par_s[i] = p;
    kid_s[i] = c;
    __syncthreads();
    int len = 0, need = 0;
    bool ok = i < P.n && p >= 0 && p < T.max_seqs && c >= 0 && c < T.max_seqs;
    for (int j = 0; j < P.n && ok; ++j)            // a child twice, or a child that is a parent too: not served
        if ((j < i && kid_s[j] == c) || par_s[j] == c || kid_s[j] == p) ok = false;
    if (ok) {
        len = T.seq_lens[p];
        const int pages = len < 0 ? INT_MAX : (int)(((long long)len + T.page_size - 1) / T.page_size);
        ok = pages <= T.width && pages <= T.held[p] && T.held[c] == 0;
        need = ok && len % T.page_size ? 1 : 0;
    }
    int total;
    const int at = block_scan(need, sums, &total);
    const bool served = ok && (need == 0 || at + need <= left);
    int src = -1, dst = -1;
    const int full = ok ? len / T.page_size : 0;
    if (served && need) {
        src = T.block_table[(size_t)p * T.bt_stride + full];
        dst = T.free_list[left - 1 - at];
        if (src < 0 || src >= T.num_pages || dst < 0 || dst >= T.num_pages) { src = dst = -1; atomicOr(T.counters + 1, EXL3_PAGES_BAD); }
    }
    if (i < P.n) {
        P.plan[i] = ForkPlan{p, served ? c : -1, full, ok ? len - full * T.page_size : 0, src, dst};
        if (served) {
            T.seq_lens[c] = len;
            T.held[c] = full + need;
            if (need) T.block_table[(size_t)c * T.bt_stride + full] = dst;     // -1 from a broken stack or table: on no page
            if (dst >= 0) T.refs[dst] = 1;
        } else {
            atomicOr(T.counters + 1, ok ? EXL3_PAGES_EXHAUSTED : EXL3_PAGES_BAD);
        }
    }
    if (i == 0) T.counters[0] = left - min(total, left);
}

// Element e = (a, b, c) of an array [..][nb][nc], walked in steps of a fixed number of elements: two additions and carries
// a step (divisions were most of the copying kernels' instructions).
struct Walk3 {
    int a, b, c, da, db, dc, nb, nc;
    __device__ __forceinline__ Walk3(int e, int step, int nb_, int nc_) : nb(nb_), nc(nc_) {
        split(e, a, b, c);
        split(step, da, db, dc);
    }
    __device__ __forceinline__ void split(int e, int &x, int &y, int &z) const {
        const int r = e / nc;
        z = e - r * nc;
        x = r / nb;
        y = r - x * nb;
    }
    __device__ __forceinline__ void next() {
        c += dc; b += db; a += da;
        if (c >= nc) { c -= nc; ++b; }
        if (b >= nb) { b -= nb; ++a; }
    }
};

struct PoolList { void *pool[EXL3_PAGES_MAX_POOLS]; };
struct RowGeom { long long page_stride, head_stride, tok_stride; int heads, row_bytes; };    // strides in bytes

// grid (n, 1 + pools): y = 0 writes the shared part of the child's table row, the others copy the used rows of the
// partial page of one pool.
constexpr int kCopyThreads = 256;
__global__ void __launch_bounds__(kCopyThreads) fork_copy_kernel(const __grid_constant__ ForkParams P,
                                                                 const __grid_constant__ PoolList L,
                                                                 const __grid_constant__ RowGeom G) {
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const ForkPlan q = P.plan[blockIdx.x];
    if (q.child < 0) return;
    const Tables &T = P.t;
    if (blockIdx.y == 0) {
        for (int j = threadIdx.x; j < q.full; j += kCopyThreads) {
            const int page = T.block_table[(size_t)q.parent * T.bt_stride + j];
            T.block_table[(size_t)q.child * T.bt_stride + j] = page;
            if (page >= 0 && page < T.num_pages) atomicAdd(T.refs + page, 1);
            else atomicOr(T.counters + 1, EXL3_PAGES_BAD);
        }
        return;
    }
    if (q.dst < 0) return;
    char *const pool = static_cast<char *>(L.pool[blockIdx.y - 1]);
    const char *const src = pool + (long long)q.src * G.page_stride;
    char *const dst = pool + (long long)q.dst * G.page_stride;
    const int chunks = G.row_bytes >> 4;                              // 16-byte pieces of a row
    const int work = G.heads * q.rest * chunks;
    constexpr int kFly = 4;                                           // loads in flight per thread
    // rows in the order they lie in memory: by token when a token's heads are adjacent, else by head
    const bool by_token = G.head_stride < G.tok_stride;
    const long long outer = by_token ? G.tok_stride : G.head_stride, inner = by_token ? G.head_stride : G.tok_stride;
    Walk3 w(threadIdx.x, kCopyThreads, by_token ? G.heads : q.rest, chunks);
    for (int e0 = threadIdx.x; e0 < work; e0 += kFly * kCopyThreads) {
        uint4 v[kFly];
        long long off[kFly];
#pragma unroll
        for (int u = 0; u < kFly; ++u) {
            off[u] = w.a * outer + w.b * inner + (w.c << 4);
            if (e0 + u * kCopyThreads < work) v[u] = *reinterpret_cast<const uint4 *>(src + off[u]);
            w.next();
        }
#pragma unroll
        for (int u = 0; u < kFly; ++u)
            if (e0 + u * kCopyThreads < work) *reinterpret_cast<uint4 *>(dst + off[u]) = v[u];
    }
}

// ---------------------------------------------------------------- reserve
struct ReserveParams {
    Tables t;
    const int *seqs, *counts;
    long long *slots, *positions;
    int *starts, *base;
    int n, tokens;
};

__global__ void __launch_bounds__(kBookThreads) reserve_kernel(const __grid_constant__ ReserveParams P) {
    __shared__ int seq_s[kMaxCall], start_s[kMaxCall], page_s[kMaxCall], held_s[kMaxCall], len_s[kMaxCall], sums[32];
    const Tables &T = P.t;
    const int i = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int left = min(max(T.counters[0], 0), T.num_pages);
    int s = -1, cnt = 0;
    if (i < P.n) { s = P.seqs[i]; cnt = P.counts[i]; }
    seq_s[i] = s;
    __syncthreads();
    bool ok = i < P.n && s >= 0 && s < T.max_seqs && cnt >= 0;
    for (int j = 0; j < i && ok; ++j)
        if (seq_s[j] == s) ok = false;
    // the tokens of a sequence keep their place in the outputs, served or not
    const int keep = i < P.n ? min(max(cnt, 0), P.tokens) : 0;         // 1024 of at most 2^20: the sum fits
    int ntok, npage;
    const int t0 = block_scan(keep, sums, &ntok);
    int len = 0, held = 0, want = 0;
    if (ok) {
        len = T.seq_lens[s];
        held = T.held[s];
        const long long pages = ((long long)len + cnt + T.page_size - 1) / T.page_size;
        ok = len >= 0 && held >= 0 && held <= T.width && pages <= T.width && t0 + (long long)cnt <= P.tokens;
        // tokens that go to pages held already: nobody else may hold those (a sequence can be cut back into pages it shares)
        for (int j = len / T.page_size; ok && cnt && j < min(held, (int)pages); ++j) {
            const int page = T.block_table[(size_t)s * T.bt_stride + j];
            ok = page >= 0 && page < T.num_pages && T.refs[page] == 1;
        }
        want = ok && pages > held ? min((int)pages - held, left + 1) : 0;
    }
    const int p0 = block_scan(want, sums, &npage);
    const bool served = ok && (want == 0 || p0 + want <= left);
    start_s[i] = t0;
    page_s[i] = p0;
    held_s[i] = served ? held : -1;                                    // -1: not served
    len_s[i] = len;
    if (i < P.n) {
        P.starts[i] = min(t0, P.tokens);
        P.base[i] = len;
        if (i == 0) P.starts[P.n] = min(ntok, P.tokens);
        if (served) {
            T.seq_lens[s] = len + cnt;
            T.held[s] = held + want;
        } else {
            atomicOr(T.counters + 1, ok && p0 + want > left ? EXL3_PAGES_EXHAUSTED : EXL3_PAGES_BAD);
        }
    }
    // Pages taken: when the list ends before a sequence has all its pages, no sequence behind it takes any either
    // (their places lie behind the end of the list too), so those taken are the first of the scan.
    int last = served && want ? p0 + want : 0;
#pragma unroll
    for (int o = 16; o; o >>= 1) last = max(last, __shfl_xor_sync(0xffffffffu, last, o));
    __syncthreads();
    if ((i & 31) == 0) sums[i >> 5] = last;
    __syncthreads();
    int taken = 0;
    for (int w = 0; w < 32; ++w) taken = max(taken, sums[w]);
    if (i == 0) T.counters[0] = left - taken;
    for (int e = i; e < taken; e += kBookThreads) {
        const int o = owner_of(page_s, P.n, e);
        const int page = T.free_list[left - 1 - e];
        const bool there = page >= 0 && page < T.num_pages;
        if (!there) atomicOr(T.counters + 1, EXL3_PAGES_BAD);
        if (held_s[o] < 0) continue;
        T.block_table[(size_t)seq_s[o] * T.bt_stride + held_s[o] + (e - page_s[o])] = there ? page : -1;
        if (there) T.refs[page] = 1;
    }
    for (int t = i; t < P.tokens; t += kBookThreads) {
        long long slot = -1, pos = 0;
        if (t < ntok) {
            const int o = owner_of(start_s, P.n, t);
            pos = (long long)len_s[o] + (t - start_s[o]);
            if (held_s[o] >= 0) {
                const int idx = (int)(pos / T.page_size);
                const int page = idx < held_s[o] ? T.block_table[(size_t)seq_s[o] * T.bt_stride + idx]
                                                 : T.free_list[left - 1 - (page_s[o] + idx - held_s[o])];
                if (page >= 0 && page < T.num_pages) slot = (long long)page * T.page_size + pos % T.page_size;
            }
        }
        P.slots[t] = slot;
        P.positions[t] = pos;
    }
}

// ---------------------------------------------------------------- free
struct FreeParams {
    Tables t;
    const int *seqs;
    int n;
};

__global__ void __launch_bounds__(kBookThreads) free_kernel(const __grid_constant__ FreeParams P) {
    __shared__ int seq_s[kMaxCall], start_s[kMaxCall], sums[32];
    const Tables &T = P.t;
    const int i = threadIdx.x;
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const int left = min(max(T.counters[0], 0), T.num_pages);
    const int s = i < P.n ? P.seqs[i] : -1;
    seq_s[i] = s;
    __syncthreads();
    bool ok = i < P.n && s >= 0 && s < T.max_seqs;
    for (int j = 0; j < i && ok; ++j)
        if (seq_s[j] == s) ok = false;                                 // the same sequence twice: freed once
    int held = ok ? T.held[s] : 0;
    if (held < 0 || held > T.width) { held = 0; ok = false; }
    if (i < P.n && !ok) atomicOr(T.counters + 1, EXL3_PAGES_BAD);
    int total;
    start_s[i] = block_scan(held, sums, &total);
    __syncthreads();
    // entry e = page number (e - start) of sequence o; the page comes with it
    const auto page_at = [&](int e) {
        const int o = owner_of(start_s, P.n, e);
        const int page = T.block_table[(size_t)seq_s[o] * T.bt_stride + (e - start_s[o])];
        return page >= 0 && page < T.num_pages ? page : -1;
    };
    for (int e = i; e < total; e += kBookThreads) {
        const int page = page_at(e);
        if (page >= 0) atomicSub(T.refs + page, 1);
        else atomicOr(T.counters + 1, EXL3_PAGES_BAD);
    }
    __threadfence_block();
    __syncthreads();
    // A page that nobody holds any more is given back once, by the last entry of the call that held it: the count,
    // no longer needed, takes the smallest of marks that fall with the entry.
    const auto mark = [&](int e) { return INT_MIN + (total - 1 - e); };
    for (int e = i; e < total; e += kBookThreads) {
        const int page = page_at(e);
        if (page >= 0 && *(volatile int *)(T.refs + page) <= 0) atomicMin(T.refs + page, mark(e));
    }
    __threadfence_block();
    __syncthreads();
    int mine = 0;
    for (int e = i; e < total; e += kBookThreads) {
        const int page = page_at(e);
        mine += page >= 0 && *(volatile int *)(T.refs + page) == mark(e);
    }
    int given;
    block_scan(mine, sums, &given);
    // first entry to the top of the stack: what fork and reserve took in order goes back as it lay
    int above = left + given;
    for (int e0 = 0; e0 < total; e0 += kBookThreads) {
        const int e = e0 + i;
        const int page = e < total ? page_at(e) : -1;
        const bool out = page >= 0 && *(volatile int *)(T.refs + page) == mark(e);
        int got;
        const int rank = block_scan(out ? 1 : 0, sums, &got);
        if (out) {
            const int at = above - 1 - rank;
            if (at >= 0 && at < T.num_pages) T.free_list[at] = page;
            else atomicOr(T.counters + 1, EXL3_PAGES_BAD);
            T.refs[page] = 0;
        }
        above -= got;
    }
    if (ok) { T.held[s] = 0; T.seq_lens[s] = 0; }
    if (i == 0) T.counters[0] = min(left + given, T.num_pages);
}

// ---------------------------------------------------------------- accept
struct AcceptParams {
    Tables t;
    const int *seqs, *base, *drafts, *path, *taken;
    int n, path_stride, most, heads, pools, per;    // heads, per (pools): of one CTA; pools: in all
};

// grid (n, pool groups, head groups): one CTA moves the accepted rows of one sequence in some heads of some pools, through
// shared memory, so that a path in any order is moved as if all rows were read before the first is written.  Finding the
// rows is a chain of four dependent loads, so a CTA does it once for several pools, and reads the next pool's rows while
// it writes one's (64 sequences in 64 layers: 30 us, 4.8 TB/s; a CTA per pool took 40 us).
constexpr int kAcceptThreads = 128;
constexpr int kMaxRowBytes = 1024;
__global__ void __launch_bounds__(kAcceptThreads) accept_kernel(const __grid_constant__ AcceptParams P,
                                                                const __grid_constant__ PoolList L,
                                                                const __grid_constant__ RowGeom G) {
    extern __shared__ __align__(16) unsigned char rows_s[];
    __shared__ long long from_s[EXL3_TREE_MAX_DRAFTS], to_s[EXL3_TREE_MAX_DRAFTS];
    asm volatile("griddepcontrol.wait;" ::: "memory");
    asm volatile("griddepcontrol.launch_dependents;");
    const Tables &T = P.t;
    const int b = blockIdx.x, tid = threadIdx.x;
    const int s = P.seqs[b], base = P.base[b], drafts = P.drafts[b], taken = P.taken[b];
    bool bad = s < 0 || s >= T.max_seqs || base < 0 || drafts < 0 || taken < 0 || taken > P.most || taken > drafts;
    if (!bad) {
        const int held = T.held[s];
        // never longer than it is: behind its end lies nothing when the reserve before was refused.  (The CTA that writes the new
        // length, base + taken, may have done so already: that passes too, and where it does not pass nobody writes.)
        const int len = *(volatile const int *)(T.seq_lens + s);
        bad = held > T.width || (long long)base + drafts > (long long)held * T.page_size || (long long)base + taken > len;
        for (int j = tid; j < b; j += kAcceptThreads) bad |= P.seqs[j] == s;    // the same sequence twice: the first counts
        if (!bad && tid < taken) {
            const int from = P.path[(size_t)b * P.path_stride + tid];
            if (from < 0 || from >= drafts) {
                bad = true;
            } else {
                const int a = base + from, c = base + tid;
                const int pa = T.block_table[(size_t)s * T.bt_stride + a / T.page_size];
                const int pc = T.block_table[(size_t)s * T.bt_stride + c / T.page_size];
                bad = pa < 0 || pa >= T.num_pages || pc < 0 || pc >= T.num_pages || (from != tid && T.refs[pc] != 1);
                from_s[tid] = from == tid ? -1 : pa * G.page_stride + (a % T.page_size) * G.tok_stride;
                to_s[tid] = pc * G.page_stride + (c % T.page_size) * G.tok_stride;
            }
        }
    }
    if (__syncthreads_or(bad)) {                   // stays as it was
        if (tid == 0 && blockIdx.y == 0 && blockIdx.z == 0) atomicOr(T.counters + 1, EXL3_PAGES_BAD);
        return;
    }
    if (tid == 0 && blockIdx.y == 0 && blockIdx.z == 0) T.seq_lens[s] = base + taken;
    const int h0 = blockIdx.z * P.heads, nh = min(P.heads, G.heads - h0);
    const int chunks = G.row_bytes >> 4, work = taken * nh * chunks;
    const int p0 = blockIdx.y * P.per, p1 = min(P.pools, p0 + P.per);
    const uint32_t stage = static_cast<uint32_t>(__cvta_generic_to_shared(rows_s));
    const int buffer = P.most * P.heads * G.row_bytes;
    const Walk3 w0(tid, kAcceptThreads, nh, chunks);
    const auto read = [&](int p) {
        const char *const pool = static_cast<const char *>(L.pool[p]) + h0 * G.head_stride;
        Walk3 w = w0;
        for (int e = tid; e < work; e += kAcceptThreads, w.next())
            if (from_s[w.a] >= 0)
                asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(stage + (p & 1) * buffer + 16 * e),
                             "l"(pool + from_s[w.a] + w.b * G.head_stride + 16 * w.c) : "memory");
        asm volatile("cp.async.commit_group;" ::: "memory");
    };
    read(p0);
    for (int p = p0; p < p1; ++p) {
        if (p + 1 < p1) {
            read(p + 1);
            asm volatile("cp.async.wait_group 1;" ::: "memory");
        } else {
            asm volatile("cp.async.wait_group 0;" ::: "memory");
        }
        __syncthreads();
        char *const pool = static_cast<char *>(L.pool[p]) + h0 * G.head_stride;
        Walk3 w = w0;
        for (int e = tid; e < work; e += kAcceptThreads, w.next())
            if (from_s[w.a] >= 0)
                *reinterpret_cast<uint4 *>(pool + to_s[w.a] + w.b * G.head_stride + 16 * w.c) =
                    *reinterpret_cast<const uint4 *>(rows_s + (p & 1) * buffer + 16 * e);
        // (a thread writes what it read itself, and reads into the other buffer next: no barrier)
    }
}

// ---------------------------------------------------------------- host side
static int read_tables(const exl3_page_tables *in, Tables &t) {
    if (!in || !in->block_table || !in->seq_lens || !in->held || !in->refs || !in->free_list || !in->counters) return EXL3_E_NULL;
    if (in->max_seqs <= 0 || in->table_width <= 0 || in->table_stride < in->table_width || in->num_pages <= 0 ||
        in->page_size <= 0 || (long long)in->table_width * in->page_size > INT_MAX || in->num_pages > (1 << 20) ||
        in->table_width > (1 << 20))
        return EXL3_E_SHAPE;
    if (!aligned(in->block_table, 4) || !aligned(in->seq_lens, 4) || !aligned(in->held, 4) || !aligned(in->refs, 4) ||
        !aligned(in->free_list, 4) || !aligned(in->counters, 4))
        return EXL3_E_ALIGN;
    t = Tables{(int *)in->block_table, (int *)in->seq_lens, (int *)in->held, (int *)in->refs, (int *)in->free_list,
               (int *)in->counters, in->table_stride, in->table_width, in->max_seqs, in->num_pages, in->page_size};
    return EXL3_OK;
}

// The most shared memory that a call of accept_kernel can ask for, allowed once per device whatever the call's own size: beside
// the kernel's 1 KB of static shared memory a launch is refused from 47 KB on, and a limit set call by call could be lowered by
// another thread between this one's setting and its launch.
static bool allow_accept_rows() {
    static bool ready[64] = {};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev >= 0 && dev < 64 && ready[dev]) return true;
    if (cudaFuncSetAttribute(accept_kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, 2 * EXL3_TREE_MAX_DRAFTS * kMaxRowBytes) !=
        cudaSuccess) {
        cudaGetLastError();
        return false;
    }
    if (dev >= 0 && dev < 64) ready[dev] = true;
    return true;
}

static int read_pools(const exl3_page_pools *in, PoolList &l, RowGeom &g) {
    if (!in || !in->pools) return EXL3_E_NULL;
    if (in->num_pools <= 0 || in->num_pools > EXL3_PAGES_MAX_POOLS || in->heads <= 0 || in->row_bytes <= 0 || (in->row_bytes & 15) ||
        in->row_bytes > kMaxRowBytes || in->heads > 65535 || in->page_stride <= 0 || in->head_stride < in->row_bytes ||
        in->token_stride < in->row_bytes || (in->page_stride & 15) || (in->head_stride & 15) || (in->token_stride & 15))
        return EXL3_E_SHAPE;
    if (in->pool_stride < 0 || (in->pool_stride & 15)) return EXL3_E_SHAPE;
    for (int i = 0; i < in->num_pools; ++i) {
        void *const p = in->pool_stride ? (in->pools[0] ? (char *)in->pools[0] + i * in->pool_stride : nullptr) : in->pools[i];
        if (!p) return EXL3_E_NULL;
        if (!aligned(p, 16)) return EXL3_E_ALIGN;
        l.pool[i] = p;
    }
    g = RowGeom{in->page_stride, in->head_stride, in->token_stride, in->heads, in->row_bytes};
    return EXL3_OK;
}

}  // namespace exl3

extern "C" size_t exl3_cache_fork_workspace_bytes(int n) {
    return n > 0 && n <= EXL3_PAGES_MAX_SEQS ? (size_t)n * sizeof(exl3::ForkPlan) : 0;
}

extern "C" int exl3_cache_fork(const exl3_page_pools *pools, const exl3_page_tables *tables, const void *parents,
                               const void *children, int n, void *workspace, size_t workspace_bytes, void *stream) {
    using namespace exl3;
    ForkParams P = {};
    PoolList L = {};
    RowGeom G = {};
    int rc = read_tables(tables, P.t);
    if (rc == EXL3_OK) rc = read_pools(pools, L, G);
    if (rc != EXL3_OK) return rc;
    if (!parents || !children) return EXL3_E_NULL;
    if (n < 0 || n > kMaxCall || (long long)G.heads * P.t.page_size * (G.row_bytes >> 4) > INT_MAX - (1 << 16))    // pieces of a page
        return EXL3_E_SHAPE;
    if (!aligned(parents, 4) || !aligned(children, 4)) return EXL3_E_ALIGN;
    if (n == 0) return EXL3_OK;
    if (!workspace || workspace_bytes < exl3_cache_fork_workspace_bytes(n)) return EXL3_E_WORKSPACE;
    if (!aligned(workspace, 16)) return EXL3_E_ALIGN;
    P.parents = (const int *)parents; P.children = (const int *)children; P.n = n; P.plan = (ForkPlan *)workspace;
    cudaStream_t st = (cudaStream_t)stream;
    if (launch_pdl(fork_plan_kernel, dim3(1), dim3(kBookThreads), 0, st, P) != cudaSuccess) return EXL3_E_LAUNCH;
    if (launch_pdl(fork_copy_kernel, dim3(n, 1 + pools->num_pools), dim3(kCopyThreads), 0, st, P, L, G) != cudaSuccess)
        return EXL3_E_LAUNCH;
    return launch_status();
}

extern "C" int exl3_cache_reserve(const exl3_page_tables *tables, const void *seqs, const void *counts, int n, void *slots,
                                  void *positions, int tokens, void *starts, void *base, void *stream) {
    using namespace exl3;
    ReserveParams P = {};
    const int rc = read_tables(tables, P.t);
    if (rc != EXL3_OK) return rc;
    if (!seqs || !counts || !starts || !base || (tokens > 0 && (!slots || !positions))) return EXL3_E_NULL;
    if (n < 0 || n > kMaxCall || tokens < 0 || tokens > (1 << 20)) return EXL3_E_SHAPE;
    if (!aligned(seqs, 4) || !aligned(counts, 4) || !aligned(starts, 4) || !aligned(base, 4) || !aligned(slots, 8) ||
        !aligned(positions, 8))
        return EXL3_E_ALIGN;
    if (n == 0) return EXL3_E_SHAPE;
    P.seqs = (const int *)seqs; P.counts = (const int *)counts; P.n = n; P.tokens = tokens;
    P.slots = (long long *)slots; P.positions = (long long *)positions; P.starts = (int *)starts; P.base = (int *)base;
    if (launch_pdl(reserve_kernel, dim3(1), dim3(kBookThreads), 0, (cudaStream_t)stream, P) != cudaSuccess) return EXL3_E_LAUNCH;
    return launch_status();
}

extern "C" int exl3_cache_free(const exl3_page_tables *tables, const void *seqs, int n, void *stream) {
    using namespace exl3;
    FreeParams P = {};
    const int rc = read_tables(tables, P.t);
    if (rc != EXL3_OK) return rc;
    if (!seqs) return EXL3_E_NULL;
    if (n < 0 || n > kMaxCall) return EXL3_E_SHAPE;
    if (!aligned(seqs, 4)) return EXL3_E_ALIGN;
    if (n == 0) return EXL3_OK;
    P.seqs = (const int *)seqs; P.n = n;
    if (launch_pdl(free_kernel, dim3(1), dim3(kBookThreads), 0, (cudaStream_t)stream, P) != cudaSuccess) return EXL3_E_LAUNCH;
    return launch_status();
}

extern "C" int exl3_cache_accept(const exl3_page_pools *pools, const exl3_page_tables *tables, const void *seqs,
                                 const void *base, const void *drafts, const void *path, int path_stride, int most,
                                 const void *taken, int n, void *stream) {
    using namespace exl3;
    AcceptParams P = {};
    PoolList L = {};
    RowGeom G = {};
    int rc = read_tables(tables, P.t);
    if (rc == EXL3_OK) rc = read_pools(pools, L, G);
    if (rc != EXL3_OK) return rc;
    if (!seqs || !base || !drafts || (!path && most) || !taken) return EXL3_E_NULL;
    if (n < 0 || n > kMaxCall || most < 0 || most > EXL3_TREE_MAX_DRAFTS || path_stride < most) return EXL3_E_SHAPE;
    if (!aligned(seqs, 4) || !aligned(base, 4) || !aligned(drafts, 4) || !aligned(path, 4) || !aligned(taken, 4)) return EXL3_E_ALIGN;
    if (n == 0) return EXL3_OK;
    P.seqs = (const int *)seqs; P.base = (const int *)base; P.drafts = (const int *)drafts; P.path = (const int *)path;
    P.taken = (const int *)taken; P.n = n; P.path_stride = path_stride; P.most = most;
    // heads per CTA: up to 16 KB of rows, twice, which leaves room for seven CTAs on an SM; pools per CTA: two such rounds of CTAs
    const int per_head = most * G.row_bytes;
    P.heads = per_head ? (16 * 1024) / per_head : G.heads;
    if (P.heads < 1) P.heads = 1;
    if (P.heads > G.heads) P.heads = G.heads;
    const int smem = 2 * P.heads * per_head;
    if (!allow_accept_rows()) return EXL3_E_LAUNCH;
    const int groups = (G.heads + P.heads - 1) / P.heads;
    P.pools = pools->num_pools;
    P.per = (int)((long long)n * P.pools * groups / (2 * 7 * 148));
    P.per = P.per < 1 ? 1 : P.per > 32 ? 32 : P.per;
    const dim3 grid(n, (P.pools + P.per - 1) / P.per, groups);
    if (launch_pdl(accept_kernel, grid, dim3(kAcceptThreads), smem, (cudaStream_t)stream, P, L, G) != cudaSuccess)
        return EXL3_E_LAUNCH;
    return launch_status();
}
