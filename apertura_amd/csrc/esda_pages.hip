// esda_pages.hip -- the upkeep of caches in pages for MI355X (gfx950): pages taken and given up,
// sequences forked and cut, the pages in use moved together, rows copied in and out, and the accepted
// rows of a step of drafted tokens moved behind the committed ones.  The C ABI is include/esda_pages.h
// and, for the last, include/esda_tree.h.
//
// What to do is decided on the device, from the table and the references, so that a serving loop never
// waits for it on the host: small kernels of a workgroup per list entry, or of one workgroup where
// entries compete for free pages, write a list of moves, and a grid of waves carries it out.  The copies
// are bound by memory (a copy of 1 GiB moves 5.1 TB/s here).  Calls among others, on inputs that change: 4,095
// rows of 16 heads x 256, K and V, into 32-row pages, 134 MB in 22 us (6.1 TB/s: the rows come partly out of
// the Infinity Cache); 32,767 rows of 4 x 512 out of 16-row pages, 268 MB in 56; 473 MB of moving pages in 94 ..
// 99.  Calls of few bytes are bound by their launches; kernels by themselves, on the same inputs each time,
// take 2.4 .. 8 us: reserve_kernel 2.5 for 4 entries and 3.6 for 32, which wait for their slots' lengths, tables
// and free pages one after the other, the commit of 32 sequences' paths on 48 planes (20 MB) 8.0.  Of such
// kernels the code's own fetches are a part: loads that are under way together and little code count, unrolled
// loops do not pay.

#include <hip/hip_runtime.h>

#include <algorithm>
#include <climits>
#include <cstdint>
#include <string>

#include "esda.h"
#include "esda_device.h"
#include "esda_internal.h"
#include "esda_page_view.h"
#include "esda_pages.h"
#include "esda_tree.h"

namespace {

using namespace esda_page_view;

constexpr int kPieceBytes = 16384;  // what a wave copies at a time
constexpr int kCopyGroups = 2048;   // most workgroups of a copy: 8 a CU
constexpr int kOneGroup = 1024;     // threads of the kernels that are one workgroup

struct Pool {
    uint16_t *data;
    int planes, heads, D, pieces;  // pieces of at most kPieceBytes in a page of one head
    long long plane_stride, page_stride, head_stride;
    __host__ __device__ int rows_per_piece() const { return kPieceBytes / 2 / D; }
};

// (src page, dst page, rows, 0)
typedef int Move __attribute__((ext_vector_type(4)));

enum EntryState { kLeftOut = 0, kShared = 1, kNeedsPage = 2, kFailed = 3 };

struct Entry {
    int state, dst, rows;
    int tail;  // the page to copy from; ~page where it was the entry's own
};

struct Header {
    int left_out, moves, live;  // 256 bytes, then a ticket of each slot
};

struct Params {
    int N, R, shift, S, P;
    long long table_stride;
    int *table, *refs, *length;
    int num_pools;
    unsigned pieces;     // of one move, over all pools
    unsigned last_move;  // moves' room - 1
    Header *head;
    Entry *entries;
    Move *moves;
    int *ids;   // [N]: free pages in order, or where each page goes
    int *rows;  // [min(S, ESDA_MAX_ENTRIES)][P]: the new rows of a fork's table
    Pool pools[ESDA_MAX_POOLS];
};

__device__ __forceinline__ bool is_page(int id, int N) { return (unsigned) id < (unsigned) N; }

__device__ __forceinline__ void add(int *at, int by) { __hip_atomic_fetch_add(at, by, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

// W threads that work on an entry: a wave, or a workgroup of 256.
template <int W>
__device__ __forceinline__ bool any_of(bool x) {
    if constexpr (W == 64) return __builtin_amdgcn_ballot_w64(x) != 0ull;
    else return __syncthreads_or(x);
}
// Whether list[i] stands in list before i; every one of the W threads, numbers t, calls it.
template <int W>
__device__ __forceinline__ bool named_before(const int *list, int i, int t) {
    const int x = list[i];
    bool found = false;
    for (int j = t; j < i; j += W) found = found || list[j] == x;
    return any_of<W>(found);
}

// `chunks` 16-byte pieces by the lanes of a wave, eight loads in flight each.  LOADED / STORED: past the
// caches.  Pages are written so: nothing reads them soon, and they push out what is (calls as above: a prompt's
// 134 MB 22 us, with plain stores 30.5).  Rows that are read out are used next, and written plainly (268 MB: 56
// us, and 53 past the caches; 65 and 73 where the GPU is waited for after each call).  Pages that move are not
// read again (473 MB: 94 .. 99 us, 99 .. 100 with such stores alone, 104 .. 105 with neither); those that are
// forked are, by the next child.
template <bool LOADED, bool STORED>
__device__ __forceinline__ void wave_copy(uint16_t *dst, const uint16_t *src, int chunks, int lane) {
    constexpr int U = 8;
    const u32x4 *s = reinterpret_cast<const u32x4 *>(src);
    u32x4 *d = reinterpret_cast<u32x4 *>(dst);
    for (int c = lane; c < chunks; c += 64 * U) {
        u32x4 v[U];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c + 64 * u < chunks) v[u] = LOADED ? __builtin_nontemporal_load(s + c + 64 * u) : s[c + 64 * u];
#pragma unroll
        for (int u = 0; u < U; ++u)
            if (c + 64 * u < chunks) {
                if constexpr (STORED) __builtin_nontemporal_store(v[u], d + c + 64 * u);
                else d[c + 64 * u] = v[u];
            }
    }
}

// Piece i of a move's: its pool, its place in a page of the pool and its first row.
struct Piece {
    const Pool *pool;
    long long at;  // elements from the page's start
    int row;
};
__device__ __forceinline__ Piece piece_of(const Params &p, unsigned i) {
    int k = 0;
    for (; k + 1 < p.num_pools; ++k) {
        const unsigned n = (unsigned) p.pools[k].planes * p.pools[k].heads * p.pools[k].pieces;
        if (i < n) break;
        i -= n;
    }
    const Pool &o = p.pools[k];
    const unsigned part = i % (unsigned) o.pieces, block = i / (unsigned) o.pieces;
    const int row = (int) part * o.rows_per_piece();
    return {&o, (long long) (block / (unsigned) o.heads) * o.plane_stride + (long long) (block % (unsigned) o.heads) * o.head_stride +
                    (long long) row * o.D, row};
}

// The listed moves, a wave to a piece.  (The first is read beside their number; moves has room for it.)
template <bool LOADED>
__device__ __forceinline__ void carry_out(const Params &p) {
    if (p.num_pools == 0) return;
    const int lane = threadIdx.x & 63;
    const unsigned waves = gridDim.x * (blockDim.x / 64), u = blockIdx.x * (blockDim.x / 64) + (unsigned) uniform(threadIdx.x >> 6);
    unsigned m = u / p.pieces, i = u % p.pieces;
    const unsigned step = waves / p.pieces, over = waves % p.pieces;
    Move mv = p.moves[min(m, p.last_move)];
    const unsigned moves = (unsigned) p.head->moves;
    while (m < moves) {
        const Piece x = piece_of(p, i);
        const int rows = min(mv[2] - x.row, min(p.R, x.pool->rows_per_piece()));
        uint16_t *const base = x.pool->data + x.at;
        if (rows > 0)
            wave_copy<LOADED, true>(base + (long long) mv[1] * x.pool->page_stride, base + (long long) mv[0] * x.pool->page_stride,
                                    rows * x.pool->D / 8, lane);
        m += step;
        i += over;
        if (i >= p.pieces) {
            i -= p.pieces;
            ++m;
        }
        mv = p.moves[min(m, p.last_move)];
    }
}

// Exclusive sum over the threads of a workgroup of kOneGroup, and the total.  (These kernels are one
// workgroup, whose time is the latency of its steps and of its code's fetches.)
struct Scan {
    int before, total;
};
__device__ __forceinline__ Scan scan(int x) {
    constexpr int W = kOneGroup / 64;
    static_assert(W == 16, "a wave's sums: a lane of a row each");
    __shared__ int of[W];
    const int lane = threadIdx.x & 63, wave = uniform(threadIdx.x >> 6);
    const int in = wave_sums(x);
    __syncthreads();  // (the last call's sums are read)
    if (lane == 63) of[wave] = in;
    __syncthreads();
    const int upto = row_sums(of[lane & 15]);
    const int before = wave ? __builtin_amdgcn_readlane(upto, wave - 1) : 0;
    return {before + in - x, __builtin_amdgcn_readlane(upto, W - 1)};
}

// A page's references as the atomics have left them, past the caches of this CU.
__device__ __forceinline__ int references(const Params &p, int id) {
    return __hip_atomic_load(p.refs + id, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

// The lowest `need` free pages in order, put(rank, page) for each; how many there are (at most need).
template <class Put>
__device__ __forceinline__ int lowest_free(const Params &p, int need, Put &&put) {
    int got = 0;
    for (int base = 0; base < p.N && got < need; base += 4 * kOneGroup) {
        const int id0 = base + 4 * (int) threadIdx.x;
        int of[4], n = 0;
        bool free[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) of[e] = references(p, min(id0 + e, p.N - 1));  // (no branch: all under way at once)
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            free[e] = id0 + e < p.N && of[e] == 0;
            n += free[e];
        }
        const Scan s = scan(n);
        int rank = got + s.before;
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (free[e]) {
                if (rank < need) put(rank, id0 + e);
                ++rank;
            }
        got += s.total;
    }
    return min(got, need);
}

// ------------------------------------------------------------------------ kernels

// A workgroup per entry.
__global__ __launch_bounds__(256) void free_kernel(Params p, const int *slots) {
    const int i = blockIdx.x, s = slots[i];
    const bool twice = named_before<256>(slots, i, threadIdx.x);
    if (twice || (unsigned) s >= (unsigned) p.S) {
        if (threadIdx.x == 0) add(&p.head->left_out, 1);
        return;
    }
    int *const row = p.table + (long long) s * p.table_stride;
    for (int k = threadIdx.x; k < p.P; k += 256) {
        const int id = row[k];
        if (is_page(id, p.N)) add(p.refs + id, -1);
        row[k] = -1;
    }
    if (threadIdx.x == 0) p.length[s] = 0;
}

// One workgroup: what each entry lacks, which pages are free, who gets them.  (One: entries compete for
// the lowest pages.  A scan takes 4,096 pages' references a step and ends with the last page that is needed.)
__global__ __launch_bounds__(kOneGroup) void reserve_kernel(Params p, const int *slots, const int *rows, int n) {
    __shared__ int slot[ESDA_MAX_ENTRIES], first[ESDA_MAX_ENTRIES], last[ESDA_MAX_ENTRIES], lack[ESDA_MAX_ENTRIES], from[ESDA_MAX_ENTRIES];
    const int t = threadIdx.x, lane = t & 63, wave = uniform(t >> 6);
    if (t < n) {
        const int s = slots[t], r = rows[t];
        const bool there = (unsigned) s < (unsigned) p.S;
        const int len = p.length[there ? s : 0];
        const bool ok = there && r >= 0 && r <= (long long) p.P * p.R && len >= 0;
        slot[t] = s;
        first[t] = ok ? len >> p.shift : 0;
        last[t] = ok ? (int) (((long long) r + p.R - 1) >> p.shift) : -1;  // (-1: left out)
    }
    __syncthreads();
    for (int i = wave; i < n; i += kOneGroup / 64) {
        const int s = slot[i];
        bool twice = false;
        for (int j = lane; j < i; j += 64) twice = twice || slot[j] == s;
        int to = last[i], sum = 0;
        if (to < 0 || any_of<64>(twice)) {
            if (lane == 0) add(&p.head->left_out, 1);
            to = 0;
        }
        const int *const row = p.table + (long long) s * p.table_stride;
        for (int k = first[i]; k < to; k += 64)
            sum += __popcll(__builtin_amdgcn_ballot_w64(k + lane < to && !is_page(row[k + lane], p.N)));
        if (lane == 0) lack[i] = sum;
    }
    __syncthreads();
    const Scan s = scan(t < n ? lack[t] : 0);  // (1024 entries of at most 2^20)
    if (t < n) from[t] = s.before;
    const int got = lowest_free(p, min(s.total, p.N), [&](int rank, int id) { p.ids[rank] = id; });
    __syncthreads();
    for (int i = wave; i < n; i += kOneGroup / 64) {
        int at = from[i];
        if (lack[i] == 0) continue;
        if (at > got - lack[i]) {
            if (lane == 0) add(&p.head->left_out, 1);
            continue;
        }
        int *const row = p.table + (long long) slot[i] * p.table_stride;
        for (int k = first[i]; k < last[i]; k += 64) {
            const bool needs = k + lane < last[i] && !is_page(row[k + lane], p.N);
            const unsigned long long who = __builtin_amdgcn_ballot_w64(needs);
            if (needs) {
                const int id = p.ids[at + __popcll(who & ((1ull << lane) - 1))];
                row[k + lane] = id;
                p.refs[id] = 1;
            }
            at += __popcll(who);
        }
    }
}

// An entry of a fork, by W threads: references of what it shares and gives up, the new row of its table
// (dst's may be another's source), and what is left to copy.  The page to copy from holds a reference more
// until the free pages are given out, so that it is none of them.
template <int W>
__device__ Entry fork_entry(const Params &p, const int *src, const int *dst, const int *rows, int i, int t) {
    const int s = src[i], d = dst[i], most = rows ? rows[i] : INT_MAX;
    bool ok = (unsigned) s < (unsigned) p.S && (unsigned) d < (unsigned) p.S;
    const int len = p.length[ok ? s : 0], r = min(most, len);
    ok = ok && r >= 0 && len <= (long long) p.P * p.R && !named_before<W>(dst, i, t);
    const int full = r >> p.shift, part = r & (p.R - 1);
    const int *const from = p.table + (long long) (ok ? s : 0) * p.table_stride;
    bool there = true;
    if (ok)
        for (int k = t; k < full + (part > 0); k += W) there = there && is_page(from[k], p.N);
    if (any_of<W>(!there) || !ok) {
        if (t == 0) add(&p.head->left_out, 1);
        return Entry{kLeftOut, 0, 0, 0};
    }
    // a cut within the page of the sequence's own last rows keeps that page
    const bool keep = s == d && part > 0 && full == len >> p.shift;
    const int *const old = p.table + (long long) d * p.table_stride;
    int *const row = p.rows + (long long) i * p.P;
    for (int k = t; k < p.P; k += W) {
        const int was = old[k];
        int is = -1;
        if (k < full || (keep && k == full)) {
            is = from[k];
            if (s != d) add(p.refs + is, 1);
        }
        if (is_page(was, p.N) && !(s == d && is >= 0)) add(p.refs + was, -1);
        row[k] = is;
    }
    const bool copies = part > 0 && !keep;
    const int tail = copies ? from[full] : 0;
    if (copies && t == 0) add(p.refs + tail, 1);
    return Entry{copies ? kNeedsPage : kShared, d, r, copies && s == d ? ~tail : tail};
}

// A free page for every entry that copies, by a workgroup of kOneGroup; the entries as the copy takes them.
__device__ void fork_pages(const Params &p, const Entry *entries, int n) {
    __shared__ int ids[ESDA_MAX_ENTRIES];
    const int t = threadIdx.x;
    Entry e = t < n ? entries[t] : Entry{kLeftOut, 0, 0, 0};
    const int tail = e.tail < 0 ? ~e.tail : e.tail, full = e.rows >> p.shift;
    int *const row = p.rows + (long long) t * p.P;
    bool needs = e.state == kNeedsPage;
    if (needs && e.tail < 0 && references(p, tail) == 1) {  // a sequence cut within a page that nobody else holds or copies
        row[full] = tail;
        needs = false;
    }
    const Scan s = scan(needs);
    const int got = lowest_free(p, s.total, [&](int rank, int id) { ids[rank] = id; });
    __syncthreads();
    if (needs) {
        add(p.refs + tail, -1);
        if (s.before < got) {
            const int id = ids[s.before];
            row[full] = id;
            p.refs[id] = 1;
            p.moves[s.before] = Move{tail, id, e.rows & (p.R - 1), 0};
        } else {  // rare: no page left
            add(&p.head->left_out, 1);
            for (int k = 0; k < full; ++k) {
                add(p.refs + row[k], -1);
                row[k] = -1;
            }
            e.state = kFailed;
        }
    }
    if (t < n) p.entries[t] = e;
    if (t == 0) p.head->moves = got;
}

// A fork's decisions: of a small one in one launch, a wave to an entry; else in two, a workgroup to an
// entry and then one for the free pages.  (4 children of 32 pages, and their next page: 13.7 us in two, 11.3
// in one; 32 children of 79, two to a wave: 17.1 and 19.2.  As the work of the last workgroup of the first of
// two, behind fences for what the others wrote, the free pages took 5 and 10 us more.)
constexpr int kSmallFork = kOneGroup / 64, kSmallForkTable = 256;  // entries, pages of each
__global__ __launch_bounds__(kOneGroup) void fork_small_kernel(Params p, const int *src, const int *dst, const int *rows, int n) {
    __shared__ Entry entries[kSmallFork];
    const int lane = threadIdx.x & 63;
    for (int i = uniform(threadIdx.x >> 6); i < n; i += kOneGroup / 64) {
        const Entry e = fork_entry<64>(p, src, dst, rows, i, lane);
        if (lane == 0) entries[i] = e;
    }
    ESDA_WAIT_VM(0);  // references and rows are written
    __syncthreads();
    fork_pages(p, entries, n);
}
__global__ __launch_bounds__(256) void fork_kernel(Params p, const int *src, const int *dst, const int *rows) {
    const Entry e = fork_entry<256>(p, src, dst, rows, blockIdx.x, threadIdx.x);
    if (threadIdx.x == 0) p.entries[blockIdx.x] = e;
}
__global__ __launch_bounds__(kOneGroup) void fork_pages_kernel(Params p, int n) { fork_pages(p, p.entries, n); }

// .. and what follows from them: the tables, by the last n workgroups, and the rows of the last pages.
__global__ __launch_bounds__(256) void fork_copy_kernel(Params p, int n) {
    const int i = (int) (blockIdx.x + n - gridDim.x);
    if (i >= 0) {
        const Entry e = p.entries[i];
        if (e.state != kLeftOut) {
            int *const to = p.table + (long long) e.dst * p.table_stride;
            const int *const row = p.rows + (long long) i * p.P;
            for (int k = threadIdx.x; k < p.P; k += 256) to[k] = row[k];
            if (threadIdx.x == 0) p.length[e.dst] = e.state == kFailed ? 0 : e.rows;
        }
    }
    carry_out<false>(p);
}

// Compaction, first launch, one workgroup: the pages in use at or above their number, and the free ones
// below it, both in order; references and the way of each page that moves.
__global__ __launch_bounds__(kOneGroup) void compact_kernel(Params p) {
    const int t = threadIdx.x;
    // references of pages id0 .. id0 + 3 (past the last: of that; no branch: all under way at once)
    auto four = [&](int id0, int (&of)[4]) {
#pragma unroll
        for (int e = 0; e < 4; ++e) of[e] = p.refs[min(id0 + e, p.N - 1)];
    };
    int n = 0, of[4];
    for (int id0 = 4 * t; id0 < p.N; id0 += 4 * kOneGroup) {
        four(id0, of);
#pragma unroll
        for (int e = 0; e < 4; ++e) n += id0 + e < p.N && of[e] != 0;
    }
    const int live = scan(n).total;
    int moves = 0, holes = 0;
    for (int base = 0; base < p.N; base += 4 * kOneGroup) {
        bool mover[4], hole[4];
        int m = 0, h = 0;
        four(base + 4 * t, of);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int id = base + 4 * t + e;
            const bool used = id < p.N && of[e] != 0;
            mover[e] = used && id >= live;
            hole[e] = !used && id < live;
            m += mover[e];
            h += hole[e];
        }
        const Scan s = scan(m << 16 | h);  // (4096 of them at most)
        int mr = moves + (s.before >> 16), hr = holes + (s.before & 0xffff);
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const int id = base + 4 * t + e;
            if (mover[e]) reinterpret_cast<int *>(p.moves + mr++)[0] = id;
            else if (id >= live && id < p.N) p.ids[id] = id;  // (nobody's)
            if (hole[e]) reinterpret_cast<int *>(p.moves + hr++)[1] = id;
        }
        moves += s.total >> 16;
        holes += s.total & 0xffff;
    }
    __syncthreads();
    for (int i = t; i < moves; i += kOneGroup) {
        const int from = p.moves[i][0], to = p.moves[i][1];
        reinterpret_cast<int *>(p.moves + i)[2] = p.R;
        p.ids[from] = to;
        p.refs[to] = p.refs[from];
        p.refs[from] = 0;
    }
    if (t == 0) {
        p.head->moves = moves;
        p.head->live = live;
    }
}

__global__ __launch_bounds__(256) void compact_copy_kernel(Params p) {
    const int live = p.head->live;
    if (p.head->moves == 0) return;
    for (long long x = blockIdx.x * 256LL + threadIdx.x; x < (long long) p.S * p.P; x += 256LL * gridDim.x) {
        int *const at = p.table + x / p.P * p.table_stride + x % p.P;
        const int id = *at;
        if (id >= live && id < p.N) *at = p.ids[id];
    }
    carry_out<true>(p);
}

// ---- rows in and out

struct RowsParams {
    Pool pool;
    int N, R, shift, P, batch, rows;
    unsigned pieces;  // of a sequence's rows, more than they can touch
    long long table_stride, plane_stride, seq_stride, head_stride;  // of the table, of the linear rows
    const int *table, *row0;
    uint16_t *linear;
};

// A wave to a piece: rows of one page, one head, one plane.
template <bool WRITE>
__global__ __launch_bounds__(256) void rows_kernel(RowsParams p) {
    const int lane = threadIdx.x & 63;
    const int per = min(p.R, p.pool.rows_per_piece());
    const unsigned waves = gridDim.x * 4u;
    const unsigned long long all = (unsigned long long) p.pool.planes * p.pool.heads * p.batch * p.pieces;
    for (unsigned long long u = blockIdx.x * 4u + (unsigned) uniform(threadIdx.x >> 6); u < all; u += waves) {
        const unsigned long long of = u / p.pieces;
        const int piece = (int) (u - of * p.pieces);
        const int b = (int) (of % (unsigned) p.batch);
        const unsigned block = (unsigned) (of / (unsigned) p.batch);
        const int head = (int) (block % (unsigned) p.pool.heads), plane = (int) (block / (unsigned) p.pool.heads);
        const long long first = p.row0[b], start = (first & -(long long) per) + (long long) piece * per;
        const long long i = max(first, start), j = min(first + p.rows, start + per);
        if (i >= j) continue;
        const long long k = start >> p.shift;  // (a piece lies in one page, or before row 0)
        const int id = k >= 0 && k < p.P ? p.table[b * p.table_stride + k] : -1;
        if (!is_page(id, p.N)) {
            if constexpr (!WRITE) {
                u32x4 *const to = reinterpret_cast<u32x4 *>(p.linear + plane * p.plane_stride + b * p.seq_stride +
                                                            head * p.head_stride + (i - first) * p.pool.D);
                for (int c = lane; c < (int) (j - i) * p.pool.D / 8; c += 64) to[c] = u32x4{0u, 0u, 0u, 0u};
            }
            continue;
        }
        uint16_t *const page = p.pool.data + plane * p.pool.plane_stride + (long long) id * p.pool.page_stride +
                               head * p.pool.head_stride + (i & (p.R - 1)) * p.pool.D;
        uint16_t *const rows = p.linear + plane * p.plane_stride + b * p.seq_stride + head * p.head_stride + (i - first) * p.pool.D;
        wave_copy<false, WRITE>(WRITE ? page : rows, WRITE ? rows : page, (int) (j - i) * p.pool.D / 8, lane);
    }
}

// ---- accepted rows

constexpr int kCommitParts = 2;  // times 256 lanes of rows a workgroup
__host__ __device__ inline unsigned commit_groups(const Pool &o) {
    return (unsigned) (((long long) o.planes * o.heads * (o.D / 8) + 256 * kCommitParts - 1) / (256 * kCommitParts));
}

struct CommitParams {
    int N, shift, S, P, cap, linear;  // linear: slot s in page s, rows below cap
    long long table_stride, accept_stride;
    const int *table, *accept, *count;
    int *length;
    int max_accept, num_pools;
    unsigned groups;  // workgroups of a slot, over all pools
    Header *head;
    Pool pools[ESDA_MAX_POOLS];
};

// Slot s's list, as a wave: lane i has the place of the row to take (page, row) and of the one it becomes.
// False where the slot is left as it was.
__device__ __forceinline__ bool accepted(const CommitParams &p, int s, int lane, int &n, int &take, int &c, int2 &from, int2 &to) {
    // (every lane loads, within the list and the table: a branch would wait for each load)
    n = p.length[s];
    c = p.count[s];
    take = p.accept[s * p.accept_stride + min(lane, p.max_accept - 1)];
    const int before = __shfl_up(take, 1);
    const bool listed = n >= 0 && c >= 0 && c <= p.max_accept, mine = listed && lane < c;
    bool ok = take >= 0 && take < 64 && (lane == 0 || take > before);
    const unsigned a = (unsigned) max(n, 0) + (take & 63), b = (unsigned) max(n, 0) + lane;
    if (p.linear) {
        from = int2{s, (int) a};
        to = int2{s, (int) b};
        ok = ok && max(a, b) < (unsigned) p.cap;
    } else {
        const int *const row = p.table + s * p.table_stride;
        const unsigned ka = a >> p.shift, kb = b >> p.shift, within = (1u << p.shift) - 1;
        from = int2{row[min(ka, p.P - 1u)], (int) (a & within)};
        to = int2{row[min(kb, p.P - 1u)], (int) (b & within)};
        ok = ok && max(ka, kb) < (unsigned) p.P && is_page(from.x, p.N) && is_page(to.x, p.N);
    }
    return listed && __builtin_amdgcn_ballot_w64(mine && !ok) == 0ull;
}

// Groups of D / 8 lanes, each a (plane, kv head) of one slot: they take the moved rows in order, eight
// at a time.  The rows rise, so that a row is written after it was read: row i becomes accept[i] >= i,
// and what is read later lies above accept[i].  Of a slot's workgroups the last to have read its list
// moves its length on.  Bound by the latency of the list, its pages and the rows.
__global__ __launch_bounds__(256) void commit_kernel(CommitParams p) {
    __shared__ int2 from[64], to[64];
    __shared__ int moved;
    const int s = (int) (blockIdx.x / p.groups), lane = threadIdx.x & 63;
    int n = 0, c = 0;
    bool ok = false;
    if (threadIdx.x < 64) {
        int take;
        int2 a{0, 0}, b{0, 0};
        ok = accepted(p, s, lane, n, take, c, a, b);
        const bool moves = ok && lane < c && take != lane;
        const unsigned long long who = __builtin_amdgcn_ballot_w64(moves);
        if (moves) {
            const int at = __popcll(who & ((1ull << lane) - 1));
            from[at] = a;
            to[at] = b;
        }
        if (lane == 0) moved = __popcll(who);
    }
    __syncthreads();  // the list was read
    if (threadIdx.x == 0) {
        int *const ticket = reinterpret_cast<int *>(p.head) + 64 + s;
        if (__hip_atomic_fetch_add(ticket, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == (int) p.groups - 1) {
            *ticket = 0;
            if (ok) p.length[s] = n + c;
            else add(&p.head->left_out, 1);
        }
    }
    if (p.num_pools == 0) return;  // (lengths alone)
    unsigned g = blockIdx.x % p.groups;
    int k = 0;
    for (; k + 1 < p.num_pools; ++k) {
        const unsigned of = commit_groups(p.pools[k]);
        if (g < of) break;
        g -= of;
    }
    const Pool &o = p.pools[k];
    const unsigned lanes = (unsigned) o.D / 8;
    for (int part = 0; part < kCommitParts; ++part) {
        const unsigned block = ((g * kCommitParts + part) * 256 + threadIdx.x) / lanes;
        if (moved == 0 || block >= (unsigned) (o.planes * o.heads)) break;
        constexpr int U = 8;
        uint16_t *const base = o.data + (long long) (block / (unsigned) o.heads) * o.plane_stride +
                               (long long) (block % (unsigned) o.heads) * o.head_stride + 8 * (threadIdx.x % lanes);
        auto at = [&](const int2 &x) { return reinterpret_cast<u32x4 *>(base + x.x * o.page_stride + (long long) x.y * o.D); };
        for (int i = 0; i < moved; i += U) {
            u32x4 v[U];
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u < moved) v[u] = *at(from[i + u]);
#pragma unroll
            for (int u = 0; u < U; ++u)
                if (i + u < moved) *at(to[i + u]) = v[u];
        }
    }
}

// ------------------------------------------------------------------------ host side

int fail(int code, const std::string &msg) {
    esda_detail::set_error(msg);
    return code;
}

int refuse(const char *call, const char *why) { return fail(ESDA_ERR_INVALID_ARGUMENT, std::string(call) + ": " + why); }

int launched(const char *call) {
    const hipError_t e = hipGetLastError();
    return e == hipSuccess ? ESDA_OK : fail(ESDA_ERR_HIP, std::string(call) + " launch: " + hipGetErrorString(e));
}

bool aligned(const void *p, unsigned n) { return (reinterpret_cast<uintptr_t>(p) & (n - 1)) == 0; }

struct Layout {
    size_t entries, moves, ids, rows, bytes;
};

// The status word and the tickets, zeroed once: each call leaves the tickets as it finds them.
size_t zeroed(int slots) { return 256 + (sizeof(int) * (size_t) slots + 255) / 256 * 256; }

size_t most_moves(int num_pages) { return std::max<size_t>(ESDA_MAX_ENTRIES, num_pages / 2 + 1); }

Layout layout(int num_pages, int slots, int max_pages) {
    auto up = [](size_t n) { return (n + 255) / 256 * 256; };
    Layout l;
    l.entries = zeroed(slots);
    l.moves = l.entries + sizeof(Entry) * ESDA_MAX_ENTRIES;
    l.ids = l.moves + sizeof(Move) * most_moves(num_pages);
    l.rows = l.ids + up(sizeof(int) * (size_t) num_pages);
    l.bytes = l.rows + sizeof(int) * (size_t) std::min(slots, ESDA_MAX_ENTRIES) * max_pages;
    return l;
}

Pool pool_params(const esda_pool &x, int page_rows) {
    Pool o{static_cast<uint16_t *>(x.data), x.planes, x.num_kv_heads, x.head_dim, 0, x.plane_stride, x.page_stride, x.head_stride};
    o.pieces = (page_rows + o.rows_per_piece() - 1) / o.rows_per_piece();
    return o;
}

const char *check_pools(const esda_pages *c, int page_rows) {
    if (c->num_pools < 0 || c->num_pools > ESDA_MAX_POOLS) return "at most 8 pools";
    for (int i = 0; i < c->num_pools; ++i) {
        if (const char *why = check_pool(c->pools[i], c->num_pages, page_rows)) return why;
        for (int j = 0; j < i; ++j)
            if (!apart(blocks_of(c->pools[i], c->num_pages, page_rows), blocks_of(c->pools[j], c->num_pages, page_rows)))
                return "two pools overlap, or lie between one another with strides that do not show otherwise";
    }
    return nullptr;
}

// .. with a workspace of which a call uses `bytes`, beside checked pools.  (Lists: in ints.)
const char *check_workspace(const esda_pages *c, size_t bytes) {
    auto holds = [&](const void *list, long long ints) { return list && meet(c->workspace, (long long) bytes / 2, list, 2 * ints); };
    if (holds(c->table, (c->slots - 1) * c->table_stride + c->max_pages) || holds(c->refs, c->num_pages) || holds(c->length, c->slots))
        return "the workspace must not overlap table, refs or length";
    for (int i = 0; i < c->num_pools; ++i)
        if (!apart(bytes_at(c->workspace, bytes), blocks_of(c->pools[i], c->num_pages, c->page_rows))) return "the workspace must not overlap a pool";
    return nullptr;
}

// Fills the kernels' parameters; an error code where the cache is none.
int page_params(const char *call, const esda_pages *c, Params *p) {
    if (!c) return refuse(call, "null cache");
    if (const char *why = check_table(c->num_pages, c->page_rows, c->slots, c->max_pages, c->table_stride)) return refuse(call, why);
    if (!c->table || !c->refs || !c->length || !aligned(c->table, 4) || !aligned(c->refs, 4) || !aligned(c->length, 4))
        return refuse(call, "table, refs and length must be 4-byte aligned device memory");
    if (const char *why = check_pools(c, c->page_rows)) return refuse(call, why);
    const Layout l = layout(c->num_pages, c->slots, c->max_pages);
    if (!c->workspace || c->workspace_bytes < l.bytes || !aligned(c->workspace, 16))
        return fail(ESDA_ERR_WORKSPACE, std::string(call) + ": workspace missing or smaller than esda_pages_workspace_size");
    if (const char *why = check_workspace(c, l.bytes)) return refuse(call, why);
    char *const ws = static_cast<char *>(c->workspace);
    *p = Params{};
    p->N = c->num_pages;
    p->R = c->page_rows;
    p->shift = __builtin_ctz((unsigned) c->page_rows);
    p->S = c->slots;
    p->P = c->max_pages;
    p->table_stride = c->table_stride;
    p->table = c->table;
    p->refs = c->refs;
    p->length = c->length;
    p->num_pools = c->num_pools;
    p->last_move = (unsigned) most_moves(c->num_pages) - 1;
    p->head = reinterpret_cast<Header *>(ws);
    p->entries = reinterpret_cast<Entry *>(ws + l.entries);
    p->moves = reinterpret_cast<Move *>(ws + l.moves);
    p->ids = reinterpret_cast<int *>(ws + l.ids);
    p->rows = reinterpret_cast<int *>(ws + l.rows);
    long long pieces = 0;
    for (int i = 0; i < c->num_pools; ++i) {
        p->pools[i] = pool_params(c->pools[i], c->page_rows);
        pieces += (long long) p->pools[i].planes * p->pools[i].heads * p->pools[i].pieces;
    }
    if (pieces >= 1LL << 31) return refuse(call, "too many planes and heads");
    p->pieces = (unsigned) std::max(1LL, pieces);
    return ESDA_OK;
}

const char *check_list(const void *list, int n) {
    if (n < 0 || n > ESDA_MAX_ENTRIES) return "a call names at most 1024 slots";
    if (n > 0 && (!list || !aligned(list, 4))) return "lists must be 4-byte aligned device memory";
    return nullptr;
}

// Workgroups of four waves for at most `moves` moves.
unsigned copy_groups(const Params &p, long long moves) {
    return (unsigned) std::max(1LL, std::min<long long>(kCopyGroups, (moves * p.pieces + 3) / 4));
}

int rows_call(const char *call, bool write, const esda_page_rows_desc *d, const int32_t *table, const int32_t *row0, void *linear,
              hipStream_t st) {
    if (!d) return refuse(call, "null description");
    if (const char *why = check_table(d->num_pages, d->page_rows, d->batch, d->max_pages, d->table_stride)) return refuse(call, why);
    if (const char *why = check_pool(d->pool, d->num_pages, d->page_rows)) return refuse(call, why);
    if (d->rows < 0 || d->rows > 1 << 30) return refuse(call, "rows must be 0 .. 2^30");
    if (!whole16(d->linear_plane_stride) || !whole16(d->linear_seq_stride) || !whole16(d->linear_head_stride))
        return refuse(call, "strides must be non-negative multiples of 8");
    if (!table || !row0 || !aligned(table, 4) || !aligned(row0, 4)) return refuse(call, "table and row0 must be 4-byte aligned device memory");
    if (!linear || !aligned(linear, 16)) return refuse(call, "linear rows must be 16-byte aligned device memory");
    if (!write && !blocks_apart({d->pool.planes, d->batch, d->pool.num_kv_heads},
                                {d->linear_plane_stride, d->linear_seq_stride, d->linear_head_stride}, (long long) d->rows * d->pool.head_dim))
        return refuse(call, "the linear rows overlap");
    const __int128 reach = (__int128) (d->pool.planes - 1) * d->linear_plane_stride + (__int128) (d->batch - 1) * d->linear_seq_stride +
                           (__int128) (d->pool.num_kv_heads - 1) * d->linear_head_stride + (__int128) d->rows * d->pool.head_dim;
    if (reach > (__int128) 1 << 60) return refuse(call, "the linear rows reach too far");
    if (d->rows > 0 && meet(linear, (long long) reach, d->pool.data,
                            (d->pool.planes - 1) * d->pool.plane_stride + (d->num_pages - 1) * d->pool.page_stride +
                                (d->pool.num_kv_heads - 1) * d->pool.head_stride + (long long) d->page_rows * d->pool.head_dim))
        return refuse(call, "the linear rows must not overlap the pool");
    const int rc = esda_detail::check_device();
    if (rc || d->rows == 0) return rc;
    RowsParams p{};
    p.pool = pool_params(d->pool, d->page_rows);
    p.N = d->num_pages;
    p.R = d->page_rows;
    p.shift = __builtin_ctz((unsigned) d->page_rows);
    p.P = d->max_pages;
    p.batch = d->batch;
    p.rows = d->rows;
    p.table_stride = d->table_stride;
    p.plane_stride = d->linear_plane_stride;
    p.seq_stride = d->linear_seq_stride;
    p.head_stride = d->linear_head_stride;
    p.table = table;
    p.row0 = row0;
    p.linear = static_cast<uint16_t *>(linear);
    const int per = std::min(p.R, p.pool.rows_per_piece());
    p.pieces = (unsigned) (d->rows / per + 2);
    const __int128 waves = (__int128) p.pool.planes * p.pool.heads * p.batch * p.pieces;
    if (waves > (__int128) 1 << 60) return refuse(call, "too many rows");
    const unsigned groups = (unsigned) std::min<__int128>(kCopyGroups, (waves + 3) / 4);
    if (write) hipLaunchKernelGGL(rows_kernel<true>, dim3(groups), dim3(256), 0, st, p);
    else hipLaunchKernelGGL(rows_kernel<false>, dim3(groups), dim3(256), 0, st, p);
    return launched(call);
}

}  // namespace

extern "C" {

int esda_pages_workspace_size(const esda_pages *c, size_t *bytes) {
    const char *call = "esda_pages_workspace_size";
    if (!c || !bytes) return refuse(call, "null argument");
    if (const char *why = check_table(c->num_pages, 16, c->slots, 1, 1)) return refuse(call, why);
    if (c->max_pages <= 0 || c->max_pages > kMaxTable) return refuse(call, "max_pages must be 1 .. 2^20");
    *bytes = layout(c->num_pages, c->slots, c->max_pages).bytes;
    return ESDA_OK;
}

int esda_pages_reserve(const esda_pages *c, const int32_t *slots, const int32_t *rows, int32_t n, void *stream) {
    const char *call = "esda_pages_reserve";
    Params p;
    if (const int rc = page_params(call, c, &p)) return rc;
    for (const int32_t *list : {slots, rows})
        if (const char *why = check_list(list, n)) return refuse(call, why);
    if (const int rc = esda_detail::check_device()) return rc;
    if (n == 0) return ESDA_OK;
    hipLaunchKernelGGL(reserve_kernel, dim3(1), dim3(kOneGroup), 0, static_cast<hipStream_t>(stream), p, slots, rows, n);
    return launched(call);
}

int esda_pages_free(const esda_pages *c, const int32_t *slots, int32_t n, void *stream) {
    const char *call = "esda_pages_free";
    Params p;
    if (const int rc = page_params(call, c, &p)) return rc;
    if (const char *why = check_list(slots, n)) return refuse(call, why);
    if (const int rc = esda_detail::check_device()) return rc;
    if (n == 0) return ESDA_OK;
    hipLaunchKernelGGL(free_kernel, dim3(n), dim3(256), 0, static_cast<hipStream_t>(stream), p, slots);
    return launched(call);
}

int esda_pages_fork(const esda_pages *c, const int32_t *src, const int32_t *dst, const int32_t *rows, int32_t n, void *stream) {
    const char *call = "esda_pages_fork";
    Params p;
    if (const int rc = page_params(call, c, &p)) return rc;
    for (const int32_t *list : {src, dst, rows ? rows : dst})
        if (const char *why = check_list(list, n)) return refuse(call, why);
    if (n > c->slots) return refuse(call, "more entries than slots");
    if (const int rc = esda_detail::check_device()) return rc;
    if (n == 0) return ESDA_OK;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    if (n <= kSmallFork && p.P <= kSmallForkTable) {
        hipLaunchKernelGGL(fork_small_kernel, dim3(1), dim3(kOneGroup), 0, st, p, src, dst, rows, n);
    } else {
        hipLaunchKernelGGL(fork_kernel, dim3(n), dim3(256), 0, st, p, src, dst, rows);
        hipLaunchKernelGGL(fork_pages_kernel, dim3(1), dim3(kOneGroup), 0, st, p, n);
    }
    hipLaunchKernelGGL(fork_copy_kernel, dim3(n + copy_groups(p, n)), dim3(256), 0, st, p, n);
    return launched(call);
}

int esda_pages_compact(const esda_pages *c, void *stream) {
    const char *call = "esda_pages_compact";
    Params p;
    if (const int rc = page_params(call, c, &p)) return rc;
    if (const int rc = esda_detail::check_device()) return rc;
    const hipStream_t st = static_cast<hipStream_t>(stream);
    const long long moves = p.num_pools ? p.N / 2 : 0;
    hipLaunchKernelGGL(compact_kernel, dim3(1), dim3(kOneGroup), 0, st, p);
    hipLaunchKernelGGL(compact_copy_kernel, dim3(std::max(copy_groups(p, moves), (unsigned) std::min(256LL, ((long long) p.S * p.P + 255) / 256))),
                       dim3(256), 0, st, p);
    return launched(call);
}

int esda_pages_status(void *workspace, int32_t *left_out, void *stream) {
    const char *call = "esda_pages_status";
    if (!workspace || !aligned(workspace, 16) || !left_out) return refuse(call, "null or unaligned argument");
    const hipStream_t st = static_cast<hipStream_t>(stream);
    hipStreamCaptureStatus capture = hipStreamCaptureStatusNone;
    hipError_t e = hipStreamIsCapturing(st, &capture);
    if (e == hipSuccess && capture != hipStreamCaptureStatusNone) return refuse(call, "waits for the stream, and cannot be captured");
    if (e == hipSuccess) e = hipMemcpyAsync(left_out, workspace, sizeof(int32_t), hipMemcpyDeviceToHost, st);
    if (e == hipSuccess) e = hipMemsetAsync(workspace, 0, sizeof(int32_t), st);
    if (e == hipSuccess) e = hipStreamSynchronize(st);
    return e == hipSuccess ? ESDA_OK : fail(ESDA_ERR_HIP, std::string(call) + ": " + hipGetErrorString(e));
}

int esda_pages_write(const esda_page_rows_desc *d, const int32_t *table, const int32_t *row0, const void *linear, void *stream) {
    return rows_call("esda_pages_write", true, d, table, row0, const_cast<void *>(linear), static_cast<hipStream_t>(stream));
}

int esda_pages_read(const esda_page_rows_desc *d, const int32_t *table, const int32_t *row0, void *linear, void *stream) {
    return rows_call("esda_pages_read", false, d, table, row0, linear, static_cast<hipStream_t>(stream));
}

int esda_tree_commit(const esda_pages *c, const int32_t *accept, int64_t accept_stride, int32_t max_accept, const int32_t *count,
                     void *stream) {
    const char *call = "esda_tree_commit";
    if (!c) return refuse(call, "null cache");
    const bool linear = !c->table;
    if (const char *why = check_table(c->num_pages, linear ? 16 : c->page_rows, c->slots, linear ? 1 : c->max_pages, linear ? 1 : c->table_stride))
        return refuse(call, why);
    if (linear && (c->max_pages != 1 || c->num_pages != c->slots || c->page_rows <= 0 || c->page_rows > 1 << 30))
        return refuse(call, "without a table: slots pages, one a slot, of 1 .. 2^30 rows");
    if (!c->length || !aligned(c->length, 4) || !aligned(c->table, 4)) return refuse(call, "table and length must be 4-byte aligned device memory");
    if (const char *why = check_pools(c, c->page_rows)) return refuse(call, why);
    if (max_accept < 1 || max_accept > 64 || accept_stride < max_accept || accept_stride > 1LL << 40)
        return refuse(call, "max_accept must be 1 .. 64, accept_stride at least that");
    if (!accept || !count || !aligned(accept, 4) || !aligned(count, 4))
        return refuse(call, "accept and count must be 4-byte aligned device memory");
    CommitParams p{};
    p.N = c->num_pages;
    p.linear = linear;
    p.shift = linear ? 30 : __builtin_ctz((unsigned) c->page_rows);
    p.S = c->slots;
    p.P = c->max_pages;
    p.cap = c->page_rows;
    p.table_stride = c->table_stride;
    p.accept_stride = accept_stride;
    p.table = c->table;
    p.accept = accept;
    p.count = count;
    p.length = c->length;
    p.max_accept = max_accept;
    p.num_pools = c->num_pools;
    p.head = static_cast<Header *>(c->workspace);
    long long groups = 0;
    for (int i = 0; i < c->num_pools; ++i) {
        p.pools[i] = pool_params(c->pools[i], c->page_rows);
        groups += commit_groups(p.pools[i]);
    }
    groups = std::max(1LL, groups);
    if (groups * c->slots > 1LL << 23) return refuse(call, "too many slots, planes and heads");
    p.groups = (unsigned) groups;
    if (!c->workspace || c->workspace_bytes < zeroed(c->slots) || !aligned(c->workspace, 16))
        return fail(ESDA_ERR_WORKSPACE, "esda_tree_commit: workspace missing or smaller than esda_pages_workspace_size");
    if (const char *why = check_workspace(c, zeroed(c->slots))) return refuse(call, why);
    const int rc = esda_detail::check_device();
    if (rc) return rc;
    hipLaunchKernelGGL(commit_kernel, dim3((unsigned) (groups * c->slots)), dim3(256), 0, static_cast<hipStream_t>(stream), p);
    return launched(call);
}

}  // extern "C"
