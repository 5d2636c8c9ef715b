// paged_cache.hip — the paged KV cache's bookkeeping and row movement for gfx950: append,
// grow, fork, free, compact, copy (include/ythip.h). Everything is decided on the device
// from (ref, table, len), so no call waits for the host and all of them can be captured.
//
// Shape of the work: what a call decides (which free page goes to whom) is a prefix sum over
// the page counts, done by one workgroup; what it moves (whole pages of every layer, rows) is
// a second launch over all CUs, bound by HBM (a page is read once and written once).

#include <algorithm>
#include <climits>

#include "launch.hpp"

namespace ythip {
namespace {

constexpr int PLAN_THREADS = 1024;  // the deciding workgroup
constexpr int PLAN_ROWS = 4;        // pages a thread looks at per step
constexpr int MAX_SEQS = 4096;      // sequences of a grow, pairs of a fork: their prefix sums lie in LDS
constexpr int MAX_COLUMNS = 65536;
constexpr int MAX_POOLS = 4;
constexpr int64_t MOST_COPIES = 1 << 23;  // pieces a launch
constexpr int COPY_BYTES = 16384;  // of a page, a workgroup of 256 threads: four 16-byte loads in flight each

__device__ __forceinline__ int pages_of(int rows, int shift) { return (int)(((int64_t)rows + (1ll << shift) - 1) >> shift); }
__device__ __forceinline__ void flag(int32_t* status, int bits) {
    if (status != nullptr) atomicOr(status, bits);
}

// Sum of v over the threads before this one, and over all; every thread of the workgroup calls it.
__device__ __forceinline__ int block_scan(int v, int* lds, int& total) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    int inc = v;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const int x = __shfl_up(inc, off, 64);
        if (lane >= off) inc += x;
    }
    __syncthreads();  // the last call's totals are read
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    int before = 0, all = 0;
#pragma unroll
    for (int w = 0; w < PLAN_THREADS / 64; ++w) {
        const int x = lds[w];
        before += w < wave ? x : 0;
        all += x;
    }
    total = all;
    return before + inc - v;
}

// Calls found(rank, page) for the free pages in ascending order until `want` of them were met
// (the last step may pass it); returns how many were met.
template <class F>
__device__ __forceinline__ int scan_free(const int32_t* ref, int pages, int want, int* lds, F&& found) {
    int met = 0;
    for (int base = 0; base < pages && met < want; base += PLAN_THREADS * PLAN_ROWS) {
        const int p0 = base + (int)threadIdx.x * PLAN_ROWS;
        bool is_free[PLAN_ROWS];
        int c = 0;
#pragma unroll
        for (int k = 0; k < PLAN_ROWS; ++k) {
            is_free[k] = p0 + k < pages && ref[p0 + k] <= 0;
            c += is_free[k];
        }
        int total;
        int r = met + block_scan(c, lds, total);
#pragma unroll
        for (int k = 0; k < PLAN_ROWS; ++k)
            if (is_free[k]) found(r++, p0 + k);
        met += total;
    }
    return met;
}

// (ref, table, len) into the arrays that a call writes, where those are others; `here`: by the
// deciding workgroup itself (a few words a thread), else in a launch before it.
struct StateArgs {
    bool here;
    int B, columns, pages;
    const int32_t *ref, *table, *len;
    int64_t ld, ld_out;
    int32_t *ref_out, *table_out, *len_out;
};
__device__ __forceinline__ void copy_state_words(const StateArgs& a, int64_t at, int64_t step) {
    if (a.ref_out != a.ref)
        for (int64_t i = at; i < a.pages; i += step) a.ref_out[i] = a.ref[i];
    if (a.len_out != a.len)
        for (int64_t i = at; i < a.B; i += step) a.len_out[i] = a.len[i];
    if (a.table_out != a.table)
        for (int64_t i = at; i < (int64_t)a.B * a.columns; i += step) {
            const int64_t b = i / a.columns, c = i % a.columns;
            a.table_out[b * a.ld_out + c] = a.table[b * a.ld + c];
        }
}
__global__ __launch_bounds__(256) void cache_state_copy(StateArgs a) {
    copy_state_words(a, (int64_t)blockIdx.x * 256 + threadIdx.x, (int64_t)gridDim.x * 256);
}

struct GrowArgs {
    int B, columns, pages, shift;
    const int32_t* n_new;
    int32_t *ref, *table, *len;  // in place
    int64_t ld;
    int32_t* status;
    StateArgs state;
};
// The prefix sum of the pages that the sequences need gives each its ranks among the free
// pages; a free page's rank then finds its sequence by bisection. One workgroup: the counts' sums
// need all of them, and its round trips (counts, users, table) are the time (16 sequences 3.4 us).
__global__ __launch_bounds__(PLAN_THREADS) void cache_grow_kernel(GrowArgs a) {
    constexpr int LIST = 4096;  // more pages than that: the free ones are looked up twice
    __shared__ int s_off[MAX_SEQS + 1], s_have[MAX_SEQS], s_list[LIST], s_scan[PLAN_THREADS / 64];
    if (a.state.here) {
        copy_state_words(a.state, threadIdx.x, PLAN_THREADS);
        __syncthreads();
    }
    const int64_t cap = (int64_t)a.columns << a.shift;
    int want = 0;
    for (int base = 0; base < a.B; base += PLAN_THREADS) {
        const int b = base + (int)threadIdx.x;
        int need = 0;
        if (b < a.B) {
            const int len = a.len[b], n = a.n_new[b];
            const bool sane = len >= 0 && n >= 0, fits = (int64_t)len + n <= cap;
            if (!sane) flag(a.status, YTHIP_CACHE_ERR_INDEX);
            else if (!fits) flag(a.status, YTHIP_CACHE_ERR_FULL);
            const int have = sane ? pages_of(len, a.shift) : 0;
            if (sane && fits) need = pages_of(len + n, a.shift) - have;
            s_have[b] = sane && fits ? have : -1;
        }
        int total;
        const int off = want + block_scan(need, s_scan, total);
        if (b < a.B) s_off[b] = off;
        want += total;
    }
    if (threadIdx.x == 0) s_off[a.B] = want;
    __syncthreads();
    const int met = scan_free(a.ref, a.pages, want, s_scan, [&](int r, int p) {
        if (r < LIST) s_list[r] = p;
    });
    const int got = met < want ? met : want;
    __syncthreads();
    auto give = [&](int r, int p) {
        if (r >= got) return;
        int lo = 0, hi = a.B;  // s_off[lo] <= r < s_off[hi]
        while (hi - lo > 1) {
            const int mid = (lo + hi) >> 1;
            if (s_off[mid] <= r) lo = mid;
            else hi = mid;
        }
        if (s_off[lo + 1] > got) return;  // its sequence finds too few
        a.table[lo * a.ld + s_have[lo] + (r - s_off[lo])] = p;
        a.ref[p] = 1;
    };
    if (got <= LIST) {
        for (int r = threadIdx.x; r < got; r += PLAN_THREADS) give(r, s_list[r]);
    } else {
        // a page's count is read before any of the same step's is written, and never again
        scan_free(a.ref, a.pages, got, s_scan, give);
    }
    for (int b = threadIdx.x; b < a.B; b += PLAN_THREADS) {
        if (s_have[b] < 0) continue;
        if (s_off[b + 1] == s_off[b] || s_off[b + 1] <= got) a.len[b] += a.n_new[b];
        else flag(a.status, YTHIP_CACHE_ERR_FULL);
    }
}

struct PoolSet {
    char* data[MAX_POOLS];
    int64_t ls[MAX_POOLS], ps[MAX_POOLS], bytes[MAX_POOLS];
    int chunks[MAX_POOLS];  // COPY_BYTES pieces of a page
    bool wide[MAX_POOLS];   // 16-byte moves
    int n, layers;
};

// Piece `chunk` of page `from` over page `to`.
__device__ __forceinline__ void copy_piece(const PoolSet& ps, int k, int layer, int from, int to, int chunk) {
    const int64_t at = (int64_t)layer * ps.ls[k], b0 = (int64_t)chunk * COPY_BYTES;
    const char* src = ps.data[k] + at + from * ps.ps[k] + b0;
    char* dst = ps.data[k] + at + to * ps.ps[k] + b0;
    const int64_t left = ps.bytes[k] - b0;
    const int bytes = left < COPY_BYTES ? (int)left : COPY_BYTES;
    if (ps.wide[k]) {
        constexpr int N = COPY_BYTES / (256 * 16);
        const u32x4* s = reinterpret_cast<const u32x4*>(src);
        u32x4* d = reinterpret_cast<u32x4*>(dst);
        const int n = bytes >> 4;
        u32x4 v[N];
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __builtin_nontemporal_load(s + min(i * 256 + (int)threadIdx.x, n - 1));
#pragma unroll
        for (int i = 0; i < N; ++i)
            if (i * 256 + (int)threadIdx.x < n) __builtin_nontemporal_store(v[i], d + i * 256 + threadIdx.x);
    } else {
        const uint32_t* s = reinterpret_cast<const uint32_t*>(src);
        uint32_t* d = reinterpret_cast<uint32_t*>(dst);
        for (int i = threadIdx.x; i < bytes >> 2; i += 256) d[i] = s[i];
    }
}

// Unit u of the copies of `n` pages in all pools: which pool, layer, page and piece.
struct Unit {
    int k, layer, i, chunk;
};
__device__ __forceinline__ bool unit_of(const PoolSet& ps, int n, int64_t u, Unit& x) {
    for (x.k = 0; x.k < ps.n; ++x.k) {
        const int64_t mine = (int64_t)n * ps.layers * ps.chunks[x.k];
        if (u < mine) {
            x.chunk = (int)(u % ps.chunks[x.k]);
            u /= ps.chunks[x.k];
            x.i = (int)(u % n);
            x.layer = (int)(u / n);
            return true;
        }
        u -= mine;
    }
    return false;
}

struct ForkArgs {
    int B, columns, pages, shift, n;
    const int32_t *src, *dst;
    int32_t *ref, *table, *len;  // in place
    int64_t ld;
    int4* plan;  // per pair: source, destination (-1: refused), whole pages, the fresh page (-1: none)
    int32_t* status;
    StateArgs state;
};
__global__ __launch_bounds__(PLAN_THREADS) void cache_fork_plan(ForkArgs a) {
    __shared__ int s_dst[MAX_SEQS], s_who[MAX_SEQS], s_page[MAX_SEQS], s_scan[PLAN_THREADS / 64];
    if (a.state.here) copy_state_words(a.state, threadIdx.x, PLAN_THREADS);
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS) s_dst[i] = a.dst[i];
    __syncthreads();
    const int64_t cap = (int64_t)a.columns << a.shift;
    int want = 0;
    for (int base = 0; base < a.n; base += PLAN_THREADS) {
        const int i = base + (int)threadIdx.x;
        int need = 0, bits = 0;
        int4 pl = {-1, -1, 0, -1};
        if (i < a.n) {
            const int s = a.src[i], d = s_dst[i];
            if (s < 0 || s >= a.B || d < 0 || d >= a.B) {
                bits = YTHIP_CACHE_ERR_INDEX;
            } else {
                const int len = a.len[s];
                bool twice = false;
                for (int j = 0; j < i && !twice; ++j) twice = s_dst[j] == d;
                if (len < 0 || len > cap) bits = YTHIP_CACHE_ERR_INDEX;
                else if (twice || a.len[d] != 0) bits = YTHIP_CACHE_ERR_BUSY;
                else {
                    pl = int4{s, d, len >> a.shift, -1};
                    need = (len & ((1 << a.shift) - 1)) != 0;
                }
            }
            if (bits) flag(a.status, bits);
        }
        int total;
        const int r = want + block_scan(need, s_scan, total);
        if (need) s_who[r] = i;
        if (i < a.n) a.plan[i] = pl;
        want += total;
    }
    __syncthreads();
    const int met = scan_free(a.ref, a.pages, want, s_scan, [&](int r, int p) {
        if (r < want) s_page[r] = p;
    });
    const int got = met < want ? met : want;
    __syncthreads();  // every length is read
    for (int r = threadIdx.x; r < want; r += PLAN_THREADS) {
        const int i = s_who[r];
        int4 pl = a.plan[i];
        if (r < got) {
            pl.w = s_page[r];
            a.ref[pl.w] = 1;
        } else {
            pl.y = -1;
            flag(a.status, YTHIP_CACHE_ERR_FULL);
        }
        a.plan[i] = pl;
    }
    __syncthreads();
    // a dst is empty, so no pair that takes rows reads a length written here
    for (int i = threadIdx.x; i < a.n; i += PLAN_THREADS) {
        const int4 pl = a.plan[i];
        if (pl.y < 0) continue;
        const int rest = pl.w >= 0 ? a.len[pl.x] & ((1 << a.shift) - 1) : 0;
        if (pl.z > 0 || rest > 0) a.len[pl.y] = (pl.z << a.shift) + rest;
    }
}

// Workgroups [0, n): pair i's row and page counts; the others its partial page, in every pool.
// Bound by the copies' bytes (8 pairs, 28 layers, 119 MB read and written 21.4 us, 5.5 TB/s).
__global__ __launch_bounds__(256) void cache_fork_copy(ForkArgs a, PoolSet ps, int64_t first) {
    const int64_t w = first + blockIdx.x;
    if (w < a.n) {
        const int4 pl = a.plan[w];
        if (pl.y < 0) return;
        const int32_t* from = a.table + pl.x * a.ld;
        int32_t* to = a.table + pl.y * a.ld;
        for (int c = threadIdx.x; c < pl.z; c += 256) {
            const int p = from[c];
            to[c] = p;
            if (p >= 0 && p < a.pages) atomicAdd(a.ref + p, 1);
            else flag(a.status, YTHIP_CACHE_ERR_INDEX);
        }
        if (threadIdx.x == 0 && pl.w >= 0) to[pl.z] = pl.w;
        return;
    }
    Unit u;
    if (!unit_of(ps, a.n, w - a.n, u)) return;
    const int4 pl = a.plan[u.i];
    if (pl.y < 0 || pl.w < 0) return;
    const int from = a.table[pl.x * a.ld + pl.z];
    if (from < 0 || from >= a.pages) {
        if (threadIdx.x == 0) flag(a.status, YTHIP_CACHE_ERR_INDEX);
        return;
    }
    copy_piece(ps, u.k, u.layer, from, pl.w, u.chunk);
}

struct FreeArgs {
    int B, columns, pages, shift, n;
    const int32_t* seqs;
    int32_t *ref, *table, *len;  // in place
    int64_t ld;
    int32_t* status;
    StateArgs state;
};
// One wave a mention; the one that finds rows takes them all (an exchange of the length). Bound by
// its round trips (length, table, users): 32 sequences of up to 41 pages 6 us.
__global__ __launch_bounds__(PLAN_THREADS) void cache_free_kernel(FreeArgs a) {
    if (a.state.here) {  // one workgroup then, whose barrier orders its own memory
        copy_state_words(a.state, threadIdx.x, PLAN_THREADS);
        __syncthreads();
    }
    const int lane = threadIdx.x & 63, waves = blockDim.x >> 6;
    for (int i = blockIdx.x * waves + (threadIdx.x >> 6); i < a.n; i += gridDim.x * waves) {
        const int s = a.seqs[i];
        if (s < 0 || s >= a.B) {
            if (lane == 0) flag(a.status, YTHIP_CACHE_ERR_INDEX);
            continue;
        }
        int len = 0;
        if (lane == 0) len = atomicExch(a.len + s, 0);
        len = __builtin_amdgcn_readfirstlane(len);
        if (len < 0 && lane == 0) flag(a.status, YTHIP_CACHE_ERR_INDEX);
        if (len <= 0) continue;
        const int held = min(pages_of(len, a.shift), a.columns);
        int32_t* row = a.table + s * a.ld;
        for (int c = lane; c < a.columns; c += 64) {
            if (c < held) {
                const int p = row[c];
                if (p < 0 || p >= a.pages) {
                    flag(a.status, YTHIP_CACHE_ERR_INDEX);
                } else if (atomicSub(a.ref + p, 1) <= 0) {  // it had no user
                    atomicAdd(a.ref + p, 1);
                    flag(a.status, YTHIP_CACHE_ERR_INDEX);
                }
            }
            row[c] = -1;
        }
    }
}

// The plan: one workgroup gives the holes below the live count the live pages above it, both
// ascending (4.7 us for 2048 pages). The move: bound by its bytes (1.77 GB read and written 289-321 us, 5.5-6.1 TB/s).
struct CompactArgs {
    int B, columns, pages, shift;
    const int32_t *ref, *table, *len;
    int64_t ld, ld_out;
    int32_t *ref_out, *table_out, *live;
    int32_t* count;  // moves
    int32_t *map, *from, *to;
};
__global__ __launch_bounds__(PLAN_THREADS) void cache_compact_plan(CompactArgs a) {
    __shared__ int s_scan[PLAN_THREADS / 64];
    int mine = 0, live;
    for (int p = threadIdx.x; p < a.pages; p += PLAN_THREADS) mine += a.ref[p] > 0;
    block_scan(mine, s_scan, live);
    // the free pages below `live` and the used ones from there on: as many of each, and a
    // page is at most one of them, so both counts go through one scan
    int holes = 0, moves = 0;
    for (int base = 0; base < a.pages; base += PLAN_THREADS * PLAN_ROWS) {
        const int p0 = base + (int)threadIdx.x * PLAN_ROWS;
        bool hole[PLAN_ROWS], move[PLAN_ROWS];
        int c = 0;
#pragma unroll
        for (int k = 0; k < PLAN_ROWS; ++k) {
            const int p = p0 + k, r = p < a.pages ? a.ref[p] : 0;
            hole[k] = p < live && r <= 0;
            move[k] = p >= live && r > 0;
            c += (hole[k] ? 1 : 0) + (move[k] ? 1 << 16 : 0);
            if (p < a.pages) {
                if (a.ref_out != a.ref) a.ref_out[p] = r;
                a.map[p] = p;
            }
        }
        int total;
        const int r = block_scan(c, s_scan, total);
        int h = holes + (r & 0xffff), m = moves + (r >> 16);
#pragma unroll
        for (int k = 0; k < PLAN_ROWS; ++k) {
            if (hole[k]) a.to[h++] = p0 + k;
            if (move[k]) a.from[m++] = p0 + k;
        }
        holes += total & 0xffff;
        moves += total >> 16;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < moves; i += PLAN_THREADS) {
        const int f = a.from[i], t = a.to[i];
        a.ref_out[t] = a.ref[f];
        a.ref_out[f] = 0;
        a.map[f] = t;
    }
    if (threadIdx.x == 0) {
        *a.count = moves;
        *a.live = live;
    }
}

__global__ __launch_bounds__(256) void cache_compact_move(CompactArgs a, PoolSet ps) {
    const int64_t entries = (int64_t)a.B * a.columns, step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < entries; i += step) {
        const int64_t b = i / a.columns;
        const int c = (int)(i % a.columns), p = a.table[b * a.ld + c], len = a.len[b];
        const bool held = len > 0 && c < pages_of(len, a.shift) && p >= 0 && p < a.pages;
        a.table_out[b * a.ld_out + c] = held ? a.map[p] : p;
    }
    const int n = *a.count;
    if (n <= 0) return;
    Unit u;
    for (int64_t w = blockIdx.x; unit_of(ps, n, w, u); w += gridDim.x)
        copy_piece(ps, u.k, u.layer, a.from[u.i], a.to[u.i], u.chunk);
}

__global__ __launch_bounds__(256) void cache_copy_kernel(int pages, int n, const int32_t* src, const int32_t* dst,
                                                         PoolSet ps, int32_t* status, int64_t first) {
    Unit u;
    if (!unit_of(ps, n, first + blockIdx.x, u)) return;
    const int from = src[u.i], to = dst[u.i];
    if (from < 0 || from >= pages || to < 0 || to >= pages) {
        if (threadIdx.x == 0) flag(status, YTHIP_CACHE_ERR_INDEX);
        return;
    }
    copy_piece(ps, u.k, u.layer, from, to, u.chunk);
}

struct AppendArgs {
    int layers, B, Hkv, T, pages, shift, slots, columns;
    const char *Kn, *Vn;
    char *Kp, *Vp;
    int64_t ns0, ns1, ns2, ns3;  // bytes
    int64_t ps0, ps1, ps2, ps3;
    float* sums;
    int64_t ss0, ss1, ss2;  // elements
    const int32_t *table, *kv_len, *count, *path;
    int64_t ld_table, ld_path;
    int chunks;  // 16-byte chunks of a row
    bool to;     // count: the lengths afterwards, not the new rows
    int32_t* status;
};
// A workgroup of NW waves takes one page that the new rows of one (layer, sequence, KV head)
// touch: thread = (row group, 16-byte chunk), so that a row moves as one run of bytes. It adds
// the rows that are there and the new ones, which it writes, to fp32 partials in registers (row
// r to group r % groups, ascending), then the groups in order, so the sum is determined by
// the page's rows alone. Bound by the latency of the lengths, the table and the rows in turn, so
// a page of up to 64 rows is one wave and all pages of a step are in flight at once
// (16 sequences, 28 layers, 45 MB: 18.3 us; with four waves a page 20.8).
// Where the lengths afterwards are given, a sequence that its grow refused has none to write, and rows that are in
// use but not among the T given are zeros (a workgroup then takes every slots-th page: the grid counts T rows).
template <class T, int NW>
__global__ __launch_bounds__(64 * NW) void cache_append_kernel(AppendArgs a) {
    constexpr int VN = Vec<T>::n, AHEAD = 8;
    __shared__ float s_sum[64 * NW * VN];
    int w = blockIdx.x;
    const int i = w % a.slots;
    w /= a.slots;
    const int h = w % a.Hkv;
    w /= a.Hkv;
    const int b = w % a.B, l = w / a.B;
    const int page = 1 << a.shift;
    const int len = a.kv_len[b], count = a.count != nullptr ? a.count[b] : a.T;
    const int64_t end = a.to ? count : (int64_t)len + min(count, a.T);  // rows in use afterwards
    const bool tells = a.to && l == 0 && h == 0 && threadIdx.x == 0;
    if (tells && i == 0 && end != len && (len < 0 || end < len || end - len > a.T || end > (int64_t)a.columns << a.shift))
        flag(a.status, YTHIP_CACHE_ERR_INDEX);
    if (len < 0 || end <= len) return;
    const int groups = 64 * NW / a.chunks;  // rows at a time
    const int rg = (int)threadIdx.x / a.chunks, ch = (int)threadIdx.x % a.chunks;
    const bool works = rg < groups;
    const char* kn = a.Kn + l * a.ns0 + b * a.ns1 + h * a.ns2 + ch * 16;
    const char* vn = a.Vn + l * a.ns0 + b * a.ns1 + h * a.ns2 + ch * 16;
    for (int slot = (len >> a.shift) + i; slot < a.columns && ((int64_t)slot << a.shift) < end; slot += a.slots) {
        const int p = a.table[b * a.ld_table + slot];
        if (p < 0 || p >= a.pages) {
            if (tells) flag(a.status, YTHIP_CACHE_ERR_INDEX);
            continue;
        }
        const int r0 = slot << a.shift;                                           // the page's first row
        const int lo = max(len - r0, 0), all = (int)min(end - r0, (int64_t)page);  // its new rows
        const int hi = (int)min((int64_t)len + a.T - r0, (int64_t)all);            // those that are given
        char* kp = a.Kp + l * a.ps0 + p * a.ps1 + h * a.ps2 + ch * 16;
        char* vp = a.Vp + l * a.ps0 + p * a.ps1 + h * a.ps2 + ch * 16;
        float acc[VN];
#pragma unroll
        for (int e = 0; e < VN; ++e) acc[e] = 0.f;
        auto add = [&](u32x4 v) {
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                if constexpr (VN == 4) acc[e] += __uint_as_float(v[e]);
                else {
                    acc[2 * e] += lo_as_f32(T{}, v[e]);
                    acc[2 * e + 1] += hi_as_f32(T{}, v[e]);
                }
            }
        };
        // AHEAD rows of a thread at a time: all their loads before the first use, without a branch around
        // them (past the end: the last row again, dropped)
        if (a.sums != nullptr && works && rg < lo)
            for (int r = rg; r < lo; r += AHEAD * groups) {
                u32x4 k[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) k[u] = *reinterpret_cast<const u32x4*>(kp + min(r + u * groups, lo - 1) * a.ps3);
#pragma unroll
                for (int u = 0; u < AHEAD; ++u)
                    if (r + u * groups < lo) add(k[u]);
            }
        if (works)
            for (int r = lo + (rg - lo % groups + groups) % groups; r < hi; r += AHEAD * groups) {
                u32x4 k[AHEAD], v[AHEAD];
                int from[AHEAD];
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int j = r0 + min(r + u * groups, hi - 1) - len;
                    from[u] = a.path != nullptr ? a.path[b * a.ld_path + j] : j;
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const bool is = from[u] >= 0 && from[u] < a.T;
                    k[u] = *reinterpret_cast<const u32x4*>(kn + (is ? from[u] : 0) * a.ns3);
                    v[u] = *reinterpret_cast<const u32x4*>(vn + (is ? from[u] : 0) * a.ns3);
                    if (!is) k[u] = v[u] = u32x4{0u, 0u, 0u, 0u};
                }
#pragma unroll
                for (int u = 0; u < AHEAD; ++u) {
                    const int row = r + u * groups;
                    if (row >= hi) break;
                    *reinterpret_cast<u32x4*>(kp + row * a.ps3) = k[u];
                    *reinterpret_cast<u32x4*>(vp + row * a.ps3) = v[u];
                    if (a.sums != nullptr) add(k[u]);
                }
            }
        if (works && hi < all)
            for (int r = max(lo, hi) + rg; r < all; r += groups)
                *reinterpret_cast<u32x4*>(kp + r * a.ps3) = *reinterpret_cast<u32x4*>(vp + r * a.ps3) = u32x4{0u, 0u, 0u, 0u};
        if (a.sums == nullptr) continue;
        const int d = a.chunks * VN;
        __syncthreads();  // the last page's sums are read
        if (works) {
#pragma unroll
            for (int e = 0; e < VN; ++e) s_sum[rg * d + ch * VN + e] = acc[e];
        }
        __syncthreads();
        float* out = a.sums + l * a.ss0 + p * a.ss1 + h * a.ss2;
        for (int e = threadIdx.x; e < d; e += 64 * NW) {
            float t = 0.f;
            for (int g = 0; g < groups; ++g) t += s_sum[g * d + e];
            out[e] = t;
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int page_shift(int page) {
    for (int s = 4; s <= 15; ++s)
        if (page == 1 << s) return s;
    return -1;
}

int check_table(const char* who, int B, int columns, int pages, int page, const void* table, int64_t ld,
                const void* len) {
    if (B < 0 || columns < 0 || pages < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    if (page_shift(page) < 0) return fail(YTHIP_EINVAL, "%s: a page of %d rows (a power of two from 16 to 32768)", who, page);
    if (columns > MAX_COLUMNS || (int64_t)columns * page > 1 << 30)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d columns of %d rows (at most 65536 columns, 2^30 rows)", who, columns, page);
    if (B > 0 && (len == nullptr || (columns > 0 && table == nullptr))) return fail(YTHIP_EINVAL, "%s: table or len is NULL", who);
    if (ld < columns) return fail(YTHIP_EINVAL, "%s: a table row of %d entries at a stride of %lld", who, columns, (long long)ld);
    return 0;
}

int check_state(const char* who, int B, int columns, int pages, int page, const void* ref, const void* table,
                int64_t ld, const void* len, const void* ref_out, const void* table_out, int64_t ld_out,
                const void* len_out) {
    if (const int st = check_table(who, B, columns, pages, page, table, ld, len)) return st;
    if (const int st = check_table(who, B, columns, pages, page, table_out, ld_out, len_out)) return st;
    if (pages > 0 && (ref == nullptr || ref_out == nullptr)) return fail(YTHIP_EINVAL, "%s: ref is NULL", who);
    if (table == table_out && ld != ld_out) return fail(YTHIP_EINVAL, "%s: one table with two strides", who);
    return 0;
}

int make_pools(const char* who, int n_pools, int layers, const ythip_page_pool* pools, PoolSet& ps) {
    if (n_pools < 0 || n_pools > MAX_POOLS || layers < 0) return fail(YTHIP_EINVAL, "%s: %d pools of %d layers", who, n_pools, layers);
    if (n_pools > 0 && pools == nullptr) return fail(YTHIP_EINVAL, "%s: pools is NULL", who);
    ps.n = n_pools;
    ps.layers = layers;
    for (int k = 0; k < n_pools; ++k) {
        const ythip_page_pool& p = pools[k];
        const int64_t all = (int64_t)(uintptr_t)p.data | (layers > 1 ? p.layer_stride : 0) | p.page_stride | p.page_bytes;
        if (p.data == nullptr || p.page_bytes <= 0 || (all & 3) != 0 || p.page_bytes > ((int64_t)INT_MAX / 2) * COPY_BYTES)
            return fail(YTHIP_EINVAL, "%s: pool %d (data, strides and bytes: multiples of 4, bytes > 0)", who, k);
        ps.data[k] = static_cast<char*>(p.data);
        ps.ls[k] = p.layer_stride;
        ps.ps[k] = p.page_stride;
        ps.bytes[k] = p.page_bytes;
        ps.chunks[k] = (int)((p.page_bytes + COPY_BYTES - 1) / COPY_BYTES);
        ps.wide[k] = (all & 15) == 0;
    }
    return 0;
}

int64_t units(const PoolSet& ps, int64_t n) {
    int64_t u = 0;
    for (int k = 0; k < ps.n; ++k) u += n * ps.layers * ps.chunks[k];
    return u;
}

// `alone`: the call's first kernel is not one workgroup
StateArgs copy_state(StateArgs a, bool alone, hipStream_t s) {
    a.here = false;
    if (a.ref == a.ref_out && a.table == a.table_out && a.len == a.len_out) return a;
    const int64_t words = (int64_t)a.B * a.columns, most = words > a.pages ? words : a.pages;
    a.here = !alone && words + a.pages <= 16 * PLAN_THREADS;
    if (a.here) return a;
    const int64_t grid = (most > a.B ? most + 255 : (int64_t)a.B + 255) / 256;
    if (grid > 0) cache_state_copy<<<(int)(grid < 1024 ? grid : 1024), 256, 0, s>>>(a);
    return a;
}

int append(const char* who, int dtype, int layers, int B, int Hkv, int T, int d, const void* Kn, const void* Vn,
           const int64_t* new_str, void* Kp, void* Vp, const int64_t* pool_str, int pages, int page, float* sums,
           const int64_t* sums_str, const int32_t* table, int64_t ld_table, int columns, const int32_t* kv_len,
           const int32_t* count, bool to, const int32_t* path, int64_t ld_path, int32_t* status, void* stream) {
    if (dtype != YTHIP_F32 && dtype != YTHIP_F16 && dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, dtype);
    if (layers < 0 || B < 0 || Hkv < 0 || T < 0 || d <= 0) return fail(YTHIP_EINVAL, "%s: bad size", who);
    if (const int st = check_table(who, B, columns, pages, page, table, ld_table, kv_len)) return st;
    if (layers == 0 || B == 0 || Hkv == 0 || T == 0 || pages == 0 || columns == 0) return 0;
    if (!Kn || !Vn || !Kp || !Vp || !new_str || !pool_str || (sums && !sums_str)) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if (path && ld_path < T) return fail(YTHIP_EINVAL, "%s: a path of %d entries at a stride of %lld", who, T, (long long)ld_path);
    const int es = dtype == YTHIP_F32 ? 4 : 2;
    if ((int64_t)d * es % 16 != 0 || (int64_t)d * es > 4096)
        return fail(YTHIP_EUNSUPPORTED, "%s: rows of %lld bytes (a multiple of 16, at most 4096)", who, (long long)d * es);
    int64_t all = (int64_t)(uintptr_t)Kn | (int64_t)(uintptr_t)Vn | (int64_t)(uintptr_t)Kp | (int64_t)(uintptr_t)Vp;
    const int new_dims[4] = {layers, B, Hkv, T}, pool_dims[4] = {layers, pages, Hkv, page};
    for (int i = 0; i < 4; ++i) all |= (new_dims[i] > 1 ? new_str[i] * es : 0) | (pool_dims[i] > 1 ? pool_str[i] * es : 0);
    if ((all & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
    AppendArgs a;
    a.layers = layers, a.B = B, a.Hkv = Hkv, a.T = T, a.pages = pages, a.shift = page_shift(page), a.columns = columns;
    a.slots = (int)(((int64_t)T + page - 2) / page + 1);  // pages that T rows touch at most
    a.Kn = static_cast<const char*>(Kn), a.Vn = static_cast<const char*>(Vn);
    a.Kp = static_cast<char*>(Kp), a.Vp = static_cast<char*>(Vp);
    a.ns0 = new_str[0] * es, a.ns1 = new_str[1] * es, a.ns2 = new_str[2] * es, a.ns3 = new_str[3] * es;
    a.ps0 = pool_str[0] * es, a.ps1 = pool_str[1] * es, a.ps2 = pool_str[2] * es, a.ps3 = pool_str[3] * es;
    a.sums = sums;
    a.ss0 = sums ? sums_str[0] : 0, a.ss1 = sums ? sums_str[1] : 0, a.ss2 = sums ? sums_str[2] : 0;
    a.table = table, a.kv_len = kv_len, a.count = count, a.path = path, a.ld_table = ld_table, a.ld_path = ld_path;
    a.to = to, a.status = status;
    a.chunks = (int)((int64_t)d * es / 16);
    const int64_t grid = (int64_t)a.slots * Hkv * B * layers;
    // a wave where a page is a few loads of it, more for long pages and rows
    const int waves = page <= 64 && a.chunks <= 64 ? 1 : page <= 512 ? 4 : 16;
    if (!launchable(grid, 64 * waves)) return fail(YTHIP_EUNSUPPORTED, "%s: %lld pages to write", who, (long long)grid);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T = decltype(t);
        if (waves == 1) cache_append_kernel<T, 1><<<(int)grid, 64, 0, s>>>(a);
        else if (waves == 4) cache_append_kernel<T, 4><<<(int)grid, 256, 0, s>>>(a);
        else cache_append_kernel<T, 16><<<(int)grid, 1024, 0, s>>>(a);
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

}  // namespace
}  // namespace ythip

using namespace ythip;

extern "C" {

__attribute__((visibility("default"))) int ythip_cache_append(
    int dtype, int layers, int B, int Hkv, int T, int d, const void* Kn, const void* Vn, const int64_t new_str[4],
    void* Kp, void* Vp, const int64_t pool_str[4], int pages, int page, float* sums, const int64_t sums_str[3],
    const int32_t* table, int64_t ld_table, int columns, const int32_t* kv_len, const int32_t* n_new,
    const int32_t* path, int64_t ld_path, void* stream) {
    return append("ythip_cache_append", dtype, layers, B, Hkv, T, d, Kn, Vn, new_str, Kp, Vp, pool_str, pages, page, sums,
                  sums_str, table, ld_table, columns, kv_len, n_new, false, path, ld_path, nullptr, stream);
}

__attribute__((visibility("default"))) int ythip_cache_append_to(
    int dtype, int layers, int B, int Hkv, int T, int d, const void* Kn, const void* Vn, const int64_t new_str[4],
    void* Kp, void* Vp, const int64_t pool_str[4], int pages, int page, float* sums, const int64_t sums_str[3],
    const int32_t* table, int64_t ld_table, int columns, const int32_t* kv_len, const int32_t* new_len,
    const int32_t* path, int64_t ld_path, int32_t* status, void* stream) {
    if (B > 0 && new_len == nullptr) return fail(YTHIP_EINVAL, "ythip_cache_append_to: new_len is NULL");
    if (B > 0 && new_len == kv_len) return fail(YTHIP_EINVAL, "ythip_cache_append_to: kv_len and new_len are one array, so no row is new");
    return append("ythip_cache_append_to", dtype, layers, B, Hkv, T, d, Kn, Vn, new_str, Kp, Vp, pool_str, pages, page, sums,
                  sums_str, table, ld_table, columns, kv_len, new_len, true, path, ld_path, status, stream);
}

__attribute__((visibility("default"))) int ythip_cache_grow(int B, int columns, int pages, int page, const int32_t* ref,
                                                            const int32_t* table, int64_t ld_table, const int32_t* len,
                                                            const int32_t* n_new, int32_t* ref_out, int32_t* table_out,
                                                            int64_t ld_out, int32_t* len_out, int32_t* status,
                                                            void* stream) {
    const char* who = "ythip_cache_grow";
    if (const int st = check_state(who, B, columns, pages, page, ref, table, ld_table, len, ref_out, table_out, ld_out, len_out)) return st;
    if (B > MAX_SEQS) return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences (at most %d)", who, B, MAX_SEQS);
    if (B > 0 && n_new == nullptr) return fail(YTHIP_EINVAL, "%s: n_new is NULL", who);
    // (the lengths are copied there before the counts are read)
    if (B > 0 && n_new == len_out && len != len_out) return fail(YTHIP_EINVAL, "%s: n_new and the lengths to write are one array", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const StateArgs st = copy_state({false, B, columns, pages, ref, table, len, ld_table, ld_out, ref_out, table_out, len_out}, B == 0, s);
    if (B > 0) cache_grow_kernel<<<1, PLAN_THREADS, 0, s>>>({B, columns, pages, page_shift(page), n_new, ref_out, table_out, len_out, ld_out, status, st});
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) size_t ythip_cache_fork_workspace_size(int n) {
    return n > 0 ? (size_t)n * sizeof(int4) : 0;
}

__attribute__((visibility("default"))) int ythip_cache_fork(int B, int columns, int pages, int page, const int32_t* ref,
                                                            const int32_t* table, int64_t ld_table, const int32_t* len,
                                                            int n, const int32_t* src, const int32_t* dst,
                                                            int32_t* ref_out, int32_t* table_out, int64_t ld_out,
                                                            int32_t* len_out, int n_pools, int layers,
                                                            const ythip_page_pool* pools, int32_t* status,
                                                            void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "ythip_cache_fork";
    if (const int st = check_state(who, B, columns, pages, page, ref, table, ld_table, len, ref_out, table_out, ld_out, len_out)) return st;
    if (n < 0 || (n > 0 && (!src || !dst))) return fail(YTHIP_EINVAL, "%s: %d pairs, or src or dst is NULL", who, n);
    if (n > MAX_SEQS) return fail(YTHIP_EUNSUPPORTED, "%s: %d pairs (at most %d)", who, n, MAX_SEQS);
    PoolSet ps;
    if (const int st = make_pools(who, n_pools, layers, pools, ps)) return st;
    const size_t need = ythip_cache_fork_workspace_size(n);
    if (need > 0 && (workspace == nullptr || ws_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return fail(YTHIP_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need, ws_bytes);
    const int64_t all = n + units(ps, n);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const StateArgs st = copy_state({false, B, columns, pages, ref, table, len, ld_table, ld_out, ref_out, table_out, len_out}, n == 0, s);
    if (n > 0) {
        const ForkArgs a = {B, columns, pages, page_shift(page), n, src, dst, ref_out, table_out, len_out, ld_out, static_cast<int4*>(workspace), status, st};
        cache_fork_plan<<<1, PLAN_THREADS, 0, s>>>(a);
        for (int64_t w = 0; w < all; w += MOST_COPIES) cache_fork_copy<<<(int)std::min(all - w, MOST_COPIES), 256, 0, s>>>(a, ps, w);
    }
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) int ythip_cache_free(int B, int columns, int pages, int page, const int32_t* ref,
                                                            const int32_t* table, int64_t ld_table, const int32_t* len,
                                                            int n, const int32_t* seqs, int32_t* ref_out,
                                                            int32_t* table_out, int64_t ld_out, int32_t* len_out,
                                                            int32_t* status, void* stream) {
    const char* who = "ythip_cache_free";
    if (const int st = check_state(who, B, columns, pages, page, ref, table, ld_table, len, ref_out, table_out, ld_out, len_out)) return st;
    if (n < 0 || (n > 0 && !seqs)) return fail(YTHIP_EINVAL, "%s: %d sequences, or seqs is NULL", who, n);
    hipStream_t s = static_cast<hipStream_t>(stream);
    const StateArgs st = copy_state({false, B, columns, pages, ref, table, len, ld_table, ld_out, ref_out, table_out, len_out}, n == 0 || n > 256, s);
    const FreeArgs a = {B, columns, pages, page_shift(page), n, seqs, ref_out, table_out, len_out, ld_out, status, st};
    if (n > 0 && st.here) cache_free_kernel<<<1, PLAN_THREADS, 0, s>>>(a);
    else if (n > 0) cache_free_kernel<<<n < 4096 ? (n + 3) / 4 : 1024, 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) size_t ythip_cache_compact_workspace_size(int pages) {
    return pages > 0 ? (4 + 3 * (size_t)pages) * sizeof(int32_t) : 16;
}

__attribute__((visibility("default"))) int ythip_cache_compact(int B, int columns, int pages, int page,
                                                               const int32_t* ref, const int32_t* table,
                                                               int64_t ld_table, const int32_t* len, int32_t* ref_out,
                                                               int32_t* table_out, int64_t ld_out, int32_t* live,
                                                               int n_pools, int layers, const ythip_page_pool* pools,
                                                               void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "ythip_cache_compact";
    if (const int st = check_state(who, B, columns, pages, page, ref, table, ld_table, len, ref_out, table_out, ld_out, len)) return st;
    if (live == nullptr) return fail(YTHIP_EINVAL, "%s: live is NULL", who);
    PoolSet ps;
    if (const int st = make_pools(who, n_pools, layers, pools, ps)) return st;
    const size_t need = ythip_cache_compact_workspace_size(pages);
    if (workspace == nullptr || ws_bytes < need || ((uintptr_t)workspace & 3) != 0)
        return fail(YTHIP_EINVAL, "%s: needs a workspace of %zu bytes, got %zu", who, need, ws_bytes);
    int32_t* ws = static_cast<int32_t*>(workspace);
    const CompactArgs a = {B, columns, pages, page_shift(page), ref, table, len, ld_table, ld_out, ref_out, table_out, live,
                           ws, ws + 4, ws + 4 + pages, ws + 4 + 2 * (int64_t)pages};
    hipStream_t s = static_cast<hipStream_t>(stream);
    cache_compact_plan<<<1, PLAN_THREADS, 0, s>>>(a);
    // how many pages move is known on the device alone: enough workgroups to fill the chip
    // many times over walk the pieces (2048 of them 340 us for 1.77 GB, 8192 328)
    int64_t grid = units(ps, pages / 2);
    const int64_t entries = ((int64_t)B * columns + 255) / 256;
    if (grid < entries) grid = entries;
    if (grid > 8192) grid = 8192;
    if (grid > 0) cache_compact_move<<<(int)grid, 256, 0, s>>>(a, ps);
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) int ythip_cache_copy_pages(int pages, int n, const int32_t* src,
                                                                  const int32_t* dst, int n_pools, int layers,
                                                                  const ythip_page_pool* pools, int32_t* status,
                                                                  void* stream) {
    const char* who = "ythip_cache_copy_pages";
    if (pages < 0 || n < 0 || (n > 0 && (!src || !dst))) return fail(YTHIP_EINVAL, "%s: %d pages, or src or dst is NULL", who, n);
    PoolSet ps;
    if (const int st = make_pools(who, n_pools, layers, pools, ps)) return st;
    const int64_t all = units(ps, n);
    if (all == 0) return 0;
    for (int64_t w = 0; w < all; w += MOST_COPIES)
        cache_copy_kernel<<<(int)std::min(all - w, MOST_COPIES), 256, 0, static_cast<hipStream_t>(stream)>>>(pages, n, src, dst, ps, status, w);
    return status_of(hipGetLastError());
}

}  // extern "C"
