// paged.hpp — what the attention kernels over pages share (paged_attn.hip, paged_q4.hip): the call's arguments, the cut
// of a batch's work, the merge of what several workgroups have of a sequence, and the host's checks.
#pragma once

#include <algorithm>
#include <climits>
#include <cmath>

#include "launch.hpp"

namespace ythip {
namespace {

constexpr int MAX_TREE = 4096;  // new tokens under `parents`

struct PagedArgs {
    int B, Hq, Hkv, G, T, pages, shift, columns;
    const void *Q, *Kn, *Vn, *Kp, *Vp;
    int64_t qs[3], kns[3], vns[3], ps[3], os[3];  // elements
    const int32_t *table, *kv_len, *parents, *new_len;
    int64_t ld_table, ld_par;
    void* O;
    float scale_log2;
    int32_t* sel;  // sparse: [B][Hkv][T][top_k]
    int top_k;
    const float* sums;
    int64_t ss[2];
    uint64_t* rank;  // sparse: [B][Hkv][T][columns], the pages' scores as rank_of has them
    int target, stage, items, row_tiles;  // the cut: ranges (0: a sequence each; sparse: of a token), tiles of a stage
    bool even;      // the cut of a few sequences: each by itself
    int short_run;  // stages up to which half as many ranges are better
    float *part, *part_ml;  // partials of items: [items][Hkv][rows][d] and (max, sum)
    int window, sinks;      // 0: no window
};

__device__ __forceinline__ int rows_in_use(const PagedArgs& a, int b) {
    const int64_t cap = (int64_t)a.columns << a.shift;
    return (int)min((int64_t)max(a.kv_len[b], 0), cap);
}
__device__ __forceinline__ int new_rows(const PagedArgs& a, int b) {
    return a.new_len != nullptr ? min(max(a.new_len[b], 0), a.T) : a.T;
}

__device__ __forceinline__ int uniform(int v) { return __builtin_amdgcn_readfirstlane(v); }
__device__ __forceinline__ int64_t uniform(int64_t v) {
    const uint32_t lo = uniform((int)(uint64_t)v), hi = uniform((int)((uint64_t)v >> 32));
    return (int64_t)((uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ const char* uniform(const char* p) {
    return reinterpret_cast<const char*>((uintptr_t)uniform((int64_t)(uintptr_t)p));
}

// The tiles of cached rows that a sequence's new tokens see: with a window the first `sinks`, then those from where the
// window of a token right behind the cache begins; the rows between are nobody's. Tile i of them holds the rows from
// row(i) on.
struct Seen {
    int tiles, first, gap;  // how many; of which lie in front of the tiles left out; how many are left out
    __device__ __forceinline__ int row(int i, int kt) const { return (i < first ? i : i + gap) * kt; }
};
__device__ __forceinline__ Seen seen_rows(const PagedArgs& a, int len, int kt) {
    const int all = (int)(((int64_t)len + kt - 1) / kt);
    if (a.window == 0) return {all, 0, 0};
    const int low = max(len + 1 - a.window, 0) / kt, sinks = (int)(((int64_t)min(a.sinks, len) + kt - 1) / kt);
    const int first = min(sinks, low);
    return {all - (low - first), first, low - first};
}
__device__ __forceinline__ int tiles_of(const PagedArgs& a, int len, int tn, int kt) {
    return seen_rows(a, len, kt).tiles + (a.Kn != nullptr ? (tn + kt - 1) / kt : 0);
}

// What of a sequence's tiles (seen_rows', then those of the new tokens) one workgroup's tokens see under a window, of
// its range [c0, c1): those from `low` on, then, downwards too, those below `sink_end`. at(i): the i-th, c0 - 1 behind
// the last. `clean`: all its tokens see the tiles from there on whole, up to their own.
struct Window {
    int c0, high, low, sink_end, clean;
    __device__ __forceinline__ int count() const { return max(high - low, 0) + max(sink_end - c0, 0); }
    __device__ __forceinline__ int at(int i) const {
        const int n = max(high - low, 0);
        if (i < n) return high - 1 - i;
        return max(sink_end - 1 - (i - n), c0 - 1);
    }
};
// The workgroup's tokens are up to t_last: none lies further behind the cache, and none nearer than `nearest`.
__device__ __forceinline__ Window window_of(const PagedArgs& a, const Seen& seen, int len, int c0, int c1, int nearest, int t_last, int kt) {
    Window w;
    const int64_t from = (int64_t)len + nearest + 1 - a.window;  // the first row or new token that one of them sees
    int low = 0, end;
    if (from > len) low = seen.tiles + (int)((from - len) / kt);
    else if (from > 0) low = max((int)(from / kt) - seen.gap, seen.first);
    if (from <= 0) end = 0;  // no row is left out
    else if (a.sinks > len) end = seen.tiles + (min(a.sinks - len, t_last + 1) + kt - 1) / kt;
    else end = seen.gap > 0 ? seen.first : (a.sinks + kt - 1) / kt;
    w.c0 = c0;
    w.high = min(c1, seen.tiles + t_last / kt + 1);
    w.low = max(max(low, end), c0);
    w.sink_end = min(end, w.high);
    const int64_t whole = (int64_t)len + t_last + 1 - a.window;
    w.clean = whole <= 0 ? 0 : whole <= len ? (int)((whole + kt - 1) / kt) - seen.gap : seen.tiles + (int)((whole - len + kt - 1) / kt);
    return w;
}

// The cut of the batch: the tiles (KT cached rows or new tokens each) of all sequences in a row,
// at least one a sequence, are dealt in `target` equal ranges, so that a ragged batch gives
// the workgroups the same work; a range that holds the end of one sequence and the start of
// another is two items, one a sequence. Item r + b is what range r holds of sequence b: the
// pairs that occur form a staircase, so the sums are distinct and a sequence's lie side by
// side. Where there are few ranges a sequence (`even`) that would leave the longest range well above
// the average, so each sequence is cut by itself: into equal items of at most the fewest stages
// with which all items number no more than `target` (two chunks of 512 over 2048 and 8192 rows,
// 8 items 82.5 -> 79 us; three trees of 7, 96 items 14.4 -> 14.9, left as they were).
// A range has at least `least_stages`: the more ranges, the longer the merge of their partials.
// Every wave works the cut out for itself from the lengths, one sequence a lane.
struct Cut {
    int b, first, count;  // the sequence, its first item and how many it has
    int chunk, at;        // tiles of an item, the item's first tile (before the sequence's start: negative)
    int len, tn;          // rows_in_use and new_rows of the sequence
};
// Sums (or the maxima of numbers that are not negative) over the lanes up to this one (DPP:
// within rows of 16, then across them).
template <class Op>
__device__ __forceinline__ int wave_scan(int v, Op op) {
    auto add = [&](int x, auto ctrl, auto rows) {
        return op(x, __builtin_amdgcn_update_dpp(0, x, decltype(ctrl)::value, decltype(rows)::value, 0xf, false));
    };
    using std::integral_constant;
    v = add(v, integral_constant<int, 0x111>{}, integral_constant<int, 0xf>{});  // row_shr 1, 2, 4, 8
    v = add(v, integral_constant<int, 0x112>{}, integral_constant<int, 0xf>{});
    v = add(v, integral_constant<int, 0x114>{}, integral_constant<int, 0xf>{});
    v = add(v, integral_constant<int, 0x118>{}, integral_constant<int, 0xf>{});
    v = add(v, integral_constant<int, 0x142>{}, integral_constant<int, 0xa>{});  // row_bcast 15 into rows 1 and 3
    v = add(v, integral_constant<int, 0x143>{}, integral_constant<int, 0xc>{});  // row_bcast 31 into rows 2 and 3
    return v;
}
__device__ __forceinline__ int wave_scan(int v) {
    return wave_scan(v, [](int x, int y) { return x + y; });
}
__device__ __forceinline__ int over(int x, int y) { return (int)(((uint32_t)x + y - 1) / (uint32_t)y); }

// The fewest stages a range has, of `all` in the batch and `longest` in a sequence. The merge takes about
// 1/20 of a stage's time a partial, so n ranges of s = longest / n stages cost the least at
// s = sqrt(longest / 20) (1 token, 1 KV head, 30000 rows: 512 ranges 34 us, 256 22, 128 17.4, 64 16.6).
// And where a tile's rows are shared, half of the ranges are better than fewer than four stages each:
// one workgroup a CU (5 trees of 16, 4 heads a group, over up to 4097 rows: 64 ranges 31 us, 32 27).
__device__ __forceinline__ int least_stages(const PagedArgs& a, int all, int longest) {
    const int root = (int)ceilf(__builtin_amdgcn_sqrtf((float)longest * 0.05f));
    return max(max(root, 1), over(all, a.target) < a.short_run ? over(all, (a.target + 1) / 2) : 1);
}
// b < 0: of the sequence that `item` belongs to (b = -1: to none)
__device__ __forceinline__ Cut cut_of(const PagedArgs& a, int kt, int item, int b) {
    const int lane = threadIdx.x & 63;
    int len = 0, tn = 0, mine = 0, inc = 0;
    auto load = [&](int i) {
        const bool is = i < a.B;
        len = is ? rows_in_use(a, i) : 0;
        tn = is ? new_rows(a, i) : 0;
        mine = is ? max(tiles_of(a, len, tn, kt), 1) : 0;
        inc = wave_scan(mine);
    };
    Cut c;
    if (a.even) {
        load(lane);
        const int stages = over(mine, a.stage), all = __builtin_amdgcn_readlane(wave_scan(stages), 63);
        // of 64 lengths of an item, a lane each, the shortest that will do; the last one does: of a
        // sequence's items all but one are full
        const int least = least_stages(a, all, __builtin_amdgcn_readlane(wave_scan(stages, [](int x, int y) { return max(x, y); }), 63));
        const int low = max(over(all, a.target), least), most = max(over(all, a.target - a.B + 1), low), by = max(over(most - low, 63), 1);
        int sum = 0;
        for (int i = 0; i < a.B; ++i) sum += over(__builtin_amdgcn_readlane(stages, i), low + lane * by);
        const int longest = low + by * __builtin_ctzll(__ballot(sum <= a.target));
        const int n = over(stages, longest), end = wave_scan(n);
        if (b < 0) b = __popcll(__ballot(lane < a.B && end <= item));
        c.b = b < a.B ? b : -1;
        b = min(b, a.B - 1);
        c.count = __builtin_amdgcn_readlane(n, b);
        c.first = __builtin_amdgcn_readlane(end, b) - c.count;
        c.chunk = over(__builtin_amdgcn_readlane(stages, b), c.count) * a.stage;
        c.at = (item - c.first) * c.chunk;
        c.len = __builtin_amdgcn_readlane(len, b);
        c.tn = __builtin_amdgcn_readlane(tn, b);
        return c;
    }
    int total = 0, longest = 0;
    for (int base = (a.B - 1) & ~63; base >= 0; base -= 64) {  // the first 64 last: they are kept
        load(base + lane);
        total += __builtin_amdgcn_readlane(inc, 63);
        longest = max(longest, __builtin_amdgcn_readlane(wave_scan(mine, [](int x, int y) { return max(x, y); }), 63));
    }
    total = over(total, a.stage);
    c.chunk = max(over(total, a.target), least_stages(a, total, over(longest, a.stage))) * a.stage;
    for (int base = 0, before = 0;; ) {
        const int start = before + inc - mine, n = min(a.B - base, 64);
        const int first = (int)((uint32_t)start / (uint32_t)c.chunk) + base + lane;
        const int last = (int)((uint32_t)(before + inc - 1) / (uint32_t)c.chunk) + base + lane;
        int at = -1;
        if (b >= 0) {
            if (b < base + 64) at = b - base;
        } else {
            const int below = __popcll(__ballot(lane < n && last < item));
            if (below < n) at = below;
        }
        if (at >= 0) {
            c.b = base + at;
            c.first = __builtin_amdgcn_readlane(first, at);
            c.count = __builtin_amdgcn_readlane(last, at) - c.first + 1;
            c.at = (item - c.b) * c.chunk - __builtin_amdgcn_readlane(start, at);
            c.len = __builtin_amdgcn_readlane(len, at);
            c.tn = __builtin_amdgcn_readlane(tn, at);
            if (b < 0 && item < c.first) c.b = -1;  // a range ended with a sequence: one sum is left out
            return c;
        }
        before += __builtin_amdgcn_readlane(inc, 63);
        base += 64;
        if (base >= a.B) break;
        load(base + lane);
    }
    c.b = -1;
    return c;
}

// The bits from i on (i < 0: all; i > 63: none).
__device__ __forceinline__ uint64_t from_bit(int64_t i) { return i <= 0 ? ~0ull : i > 63 ? 0 : ~0ull << (int)i; }

// A wave-uniform word through the scalar cache: read like this, page ids do not count as
// vector loads, whose in-order return would make each wait for the rows in flight.
__device__ __forceinline__ int scalar_word(const int32_t* p) {
#if defined(__HIP_DEVICE_COMPILE__)
    typedef const __attribute__((address_space(4))) int32_t word;
    return *(word*)(uintptr_t)p;
#else
    return 0;
#endif
}

// Two weights as two pairs of 16-bit numbers that the matrix cores take one after the other: `hi` their first bits
// (truncated, 8 or 11 of them), `rest` what is left. The weights taken are w (1 + 2^-23) (bf16) and w (1 + 2^-10)
// (fp16), of all keys alike, so that their sum has the factor too and it cancels; it keeps `rest` above 0 for any weight
// that is, and an infinite V times the two never makes inf - inf or 0 . inf. Of a weight 2^-16 (bf16) or 2^-21 (fp16)
// is lost at most.
template <class T>
__device__ __forceinline__ void split2(float x, float y, uint32_t& hi, uint32_t& rest) {
    constexpr float ABOVE = std::is_same_v<T, BF16> ? 1.0f + 0x1p-23f : 1.0f + 0x1p-10f;
#if defined(__HIP_DEVICE_COMPILE__)
    if constexpr (std::is_same_v<T, BF16>) hi = __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
    else hi = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
#endif
    rest = pack2<T>(fmaf(x, ABOVE, -lo_as_f32(T{}, hi)), fmaf(y, ABOVE, -hi_as_f32(T{}, hi)));
}

// Joins the partials of a sequence that several items worked on, in the order of the items: D / 4
// lanes a row of O (token, head), each four elements of every partial, MERGE_AHEAD of them in
// flight. Bound by the partials' bytes for many rows, by four round trips to memory (lengths,
// maxima and sums, partials, O) for few, whose partials the four waves of a workgroup share
// (SHARE). 33.5 MB of partials 13 us, 16 sequences' 256 rows of about 4 each 4.7 us.
constexpr int MERGE_AHEAD = 8;
template <class T, int D, bool SPARSE, bool SHARE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a, int kt) {
    constexpr int LPR = D / 4, RPW = 64 / LPR;
    const int lane = threadIdx.x & 63, sub = lane % LPR, group = lane / LPR;
    const int h = blockIdx.y, b = blockIdx.z;
    const int wave = uniform((int)threadIdx.x >> 6);
    const int r = (SHARE ? blockIdx.x : blockIdx.x * 4 + wave) * RPW + group;
    const int R = SPARSE ? a.G : a.T * a.G;
    int64_t first;
    int count, tn, t, gh;
    const int64_t step = (int64_t)a.Hkv * R;  // rows between an item's partial and the next one's
    if constexpr (SPARSE) {
        const int len = rows_in_use(a, b);
        tn = new_rows(a, b);
        t = r / a.G, gh = r - t * a.G;
        const int nsel = min(a.top_k, (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift));
        const int nt = (int)((((int64_t)nsel << a.shift) + kt - 1) / kt) + (a.Kn != nullptr ? (t + kt) / kt : 0);
        const int chunk = max((nt + a.target - 1) / a.target, a.stage);
        count = max((nt + chunk - 1) / chunk, 1);
        first = (((int64_t)(b * a.T + t) * a.target) * a.Hkv + h) * a.G + gh;
    } else {
        const Cut c = cut_of(a, kt, 0, b);
        count = c.count, tn = c.tn;
        if (count == 1) return;
        t = r / a.G, gh = r - t * a.G;
        first = ((int64_t)c.first * a.Hkv + h) * R + r;
    }
    if (t >= tn || t >= a.T) count = 1;  // nothing to join: it stays for the others' shuffles, on partial 0
    const bool join = count > 1;
    if (__ballot(join) == 0) return;
    if (!join) first = 0;
    const float* ml = a.part_ml + 2 * first;
    const float* src = a.part + first * D + sub * 4;
    float M = -INFINITY, L = 0.f;
    f32x4 acc = {0.f, 0.f, 0.f, 0.f};
    for (int s = sub; s < count; s += LPR) M = __builtin_elementwise_maximum(M, ml[2 * s * step]);
#pragma unroll
    for (int off = LPR / 2; off >= 1; off >>= 1) M = __builtin_elementwise_maximum(M, __shfl_xor(M, off, 64));
    const float ref = M == -INFINITY ? 0.f : M;
    int most = count;
#pragma unroll
    for (int off = 32; off >= LPR; off >>= 1) most = max(most, __shfl_xor(most, off, 64));
    most = uniform(most);
    for (int s0 = 0; s0 < most; s0 += LPR) {
        // loads without a branch around them (past the last partial: the last again, with no weight),
        // so that they are in flight together
        const float* mine = ml + 2 * min(s0 + sub, count - 1) * step;
        const float w = s0 + sub < count ? __builtin_amdgcn_exp2f(mine[0] - ref) : 0.f;
        L += s0 + sub < count ? w * mine[1] : 0.f;
        for (int s = SHARE ? wave * MERGE_AHEAD : 0; s < min(most - s0, LPR); s += SHARE ? 4 * MERGE_AHEAD : MERGE_AHEAD) {
            f32x4 v[MERGE_AHEAD];
#pragma unroll
            for (int u = 0; u < MERGE_AHEAD; ++u)
                v[u] = *reinterpret_cast<const f32x4*>(src + min(s0 + s + u, count - 1) * step * D);
#pragma unroll
            for (int u = 0; u < MERGE_AHEAD; ++u)
                if (s0 + s + u < count) acc += __shfl(w, group * LPR + s + u, 64) * v[u];
        }
    }
#pragma unroll
    for (int off = LPR / 2; off >= 1; off >>= 1) L += __shfl_xor(L, off, 64);
    if constexpr (SHARE) {
        __shared__ f32x4 s_acc[4][64];
        s_acc[wave][lane] = acc;
        __syncthreads();
        if (wave != 0) return;
        acc = (s_acc[0][lane] + s_acc[1][lane]) + (s_acc[2][lane] + s_acc[3][lane]);
    }
    if (!join) return;
    const float inv = M == -INFINITY ? 0.f : 1.0f / L;
    const f32x4 o = M == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : acc * inv;
    const int64_t at = b * a.os[0] + (int64_t)(h * a.G + gh) * a.os[1] + t * a.os[2] + sub * 4;
    if constexpr (std::is_same_v<T, F32>) *reinterpret_cast<f32x4*>(static_cast<float*>(a.O) + at) = o;
    else *reinterpret_cast<u32x2*>(static_cast<uint16_t*>(a.O) + at) = u32x2{pack2<T>(o[0], o[1]), pack2<T>(o[2], o[3])};
}

template <class T, int D, bool SPARSE>
void merge_partials(const PagedArgs& a, int kt, hipStream_t s) {
    constexpr int ROWS = 256 / D;  // of a wave
    const int rows = a.T * a.G;
    // few rows: a workgroup's waves share them (16 rows of 32 partials 6.8 -> 4.9 us; 5000 rows of
    // about 12 8.3 -> 9.9)
    if ((int64_t)a.B * a.Hkv * rows <= 512)
        paged_merge_kernel<T, D, SPARSE, true><<<dim3((rows + ROWS - 1) / ROWS, a.Hkv, a.B), 256, 0, s>>>(a, kt);
    else
        paged_merge_kernel<T, D, SPARSE, false><<<dim3((rows + 4 * ROWS - 1) / (4 * ROWS), a.Hkv, a.B), 256, 0, s>>>(a, kt);
}

// How a call is cut. Both the size of the workspace and the launch come from this alone.
struct Plan {
    int qt, wr, kt;  // the workgroup's shape
    int target, stage, row_tiles;
    bool even = false;
    int short_run;
    int64_t items;
    size_t part_bytes, ml_bytes, rank_bytes;  // multiples of 16
    size_t bytes() const { return part_bytes + ml_bytes + rank_bytes; }
};
constexpr int SLOTS = 512;
constexpr int EVEN_SEQS = 8;  // sequences whose cut is one by one at most: its search asks each in turn
constexpr int WHOLE = 6;  // stages up to which a sequence stays with one workgroup

int check_window(const char* who, int window, int sinks) {
    if (window < 0 || sinks < 0) return fail(YTHIP_EINVAL, "%s: a window of %d and %d sinks", who, window, sinks);
    return 0;
}
// A window that reaches every position is none.
void trim_window(int T, int columns, int page, int& window, int& sinks) {
    const int64_t rows = (int64_t)columns * page + T;
    if (window >= rows) window = 0;
    sinks = window > 0 ? (int)std::min<int64_t>(sinks, rows) : 0;
}

int check_workspace(const char* who, size_t need, const void* ws, size_t bytes) {
    if (need > 0 && (ws == nullptr || bytes < need || ((uintptr_t)ws & 15) != 0))
        return fail(YTHIP_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need, bytes);
    return 0;
}

struct Call {
    int dtype, B, Hq, Hkv, T, d;
    const void* Q;
    const int64_t* q_str;
    const void* Kn;
    const int64_t* kn_str;
    const void* Vn;
    const int64_t* vn_str;
    const void *Kp, *Vp;
    const int64_t* pool_str;
    int pages, page;
    const int32_t* table;
    int64_t ld_table;
    int columns;
    const int32_t *kv_len, *parents;
    int64_t ld_par;
    const int32_t* new_len;
    void* O;
    const int64_t* o_str;
    float scale;
};

// Checks what both entry points share; `done`: nothing to compute.
int prepare(const char* who, const Call& c, PagedArgs& a, bool& done) {
    done = false;
    if (c.dtype != YTHIP_F32 && c.dtype != YTHIP_F16 && c.dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, c.dtype);
    if (c.B < 0 || c.Hq < 0 || c.Hkv < 0 || c.T < 0 || c.pages < 0 || c.columns < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    if (c.d != 64 && c.d != 128) return fail(YTHIP_EUNSUPPORTED, "%s: head dim %d (64 or 128)", who, c.d);
    a.shift = -1;
    for (int s = 4; s <= 15; ++s)
        if (c.page == 1 << s) a.shift = s;
    if (a.shift < 0) return fail(YTHIP_EINVAL, "%s: a page of %d rows (a power of two from 16 to 32768)", who, c.page);
    if (c.B == 0 || c.Hq == 0 || c.T == 0) {
        done = true;
        return 0;
    }
    if (c.Hkv == 0 || c.Hq % c.Hkv != 0) return fail(YTHIP_EINVAL, "%s: %d query heads over %d KV heads", who, c.Hq, c.Hkv);
    if (c.columns > 65536 || (int64_t)c.columns * c.page > 1 << 30)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d columns of %d rows (at most 65536 columns, 2^30 rows)", who, c.columns, c.page);
    if ((int64_t)c.B * c.columns * c.page > (int64_t)1 << 34)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences of %d columns of %d rows (2^34 rows in all)", who, c.B, c.columns, c.page);
    if ((int64_t)c.T * c.Hq > 1 << 30) return fail(YTHIP_EUNSUPPORTED, "%s: %d new tokens of %d heads (2^30 in all)", who, c.T, c.Hq);
    if (c.parents != nullptr && c.T > MAX_TREE) return fail(YTHIP_EUNSUPPORTED, "%s: a tree of %d tokens (at most %d)", who, c.T, MAX_TREE);
    if (!c.Q || !c.O || !c.kv_len || !c.q_str || !c.o_str || !c.pool_str) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if ((c.Kn == nullptr) != (c.Vn == nullptr) || (c.Kn && (!c.kn_str || !c.vn_str))) return fail(YTHIP_EINVAL, "%s: Kn and Vn go together, with their strides", who);
    if (c.columns > 0 && (!c.table || (c.pages > 0 && (!c.Kp || !c.Vp)))) return fail(YTHIP_EINVAL, "%s: table or a pool is NULL", who);
    if (c.ld_table < c.columns) return fail(YTHIP_EINVAL, "%s: a table row of %d entries at a stride of %lld", who, c.columns, (long long)c.ld_table);
    if (c.parents && c.ld_par < c.T) return fail(YTHIP_EINVAL, "%s: a parents row of %d entries at a stride of %lld", who, c.T, (long long)c.ld_par);
    const int es = c.dtype == YTHIP_F32 ? 4 : 2;
    int64_t all = (int64_t)(uintptr_t)c.Q | (int64_t)(uintptr_t)c.O | (int64_t)(uintptr_t)c.Kn | (int64_t)(uintptr_t)c.Vn |
                  (int64_t)(uintptr_t)c.Kp | (int64_t)(uintptr_t)c.Vp;
    // the stride of a dim of one element may be anything, and is taken as 0
    const int q_dims[3] = {c.B, c.Hq, c.T}, new_dims[3] = {c.B, c.Hkv, c.T}, pool_dims[3] = {c.pages, c.Hkv, c.page};
    auto real = [](const int64_t* str, const int* dims, int i) { return dims[i] > 1 ? str[i] : 0; };
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = real(c.q_str, q_dims, i), a.os[i] = real(c.o_str, q_dims, i), a.ps[i] = real(c.pool_str, pool_dims, i);
        a.kns[i] = c.Kn ? real(c.kn_str, new_dims, i) : 0, a.vns[i] = c.Kn ? real(c.vn_str, new_dims, i) : 0;
        all |= (a.qs[i] | a.os[i] | a.ps[i] | a.kns[i] | a.vns[i]) * es;
    }
    if ((all & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
    for (const int64_t row : {a.ps[2], a.kns[2], a.vns[2]})  // 16 rows within 32-bit offsets
        if (row < 0 || row >= 1 << 24) return fail(YTHIP_EUNSUPPORTED, "%s: K or V rows at a stride of %lld (0 to 2^24 - 1)", who, (long long)row);
    a.B = c.B, a.Hq = c.Hq, a.Hkv = c.Hkv, a.G = c.Hq / c.Hkv, a.T = c.T, a.pages = c.pages, a.columns = c.columns;
    a.Q = c.Q, a.Kn = c.Kn, a.Vn = c.Vn, a.Kp = c.Kp, a.Vp = c.Vp;
    a.table = c.table, a.kv_len = c.kv_len, a.parents = c.parents, a.new_len = c.new_len;
    a.ld_table = c.ld_table, a.ld_par = c.ld_par, a.O = c.O;
    a.scale_log2 = (c.scale == 0.f ? 1.0f / sqrtf((float)c.d) : c.scale) * 1.4426950408889634f;
    a.sel = nullptr, a.top_k = 0, a.sums = nullptr, a.rank = nullptr, a.window = a.sinks = 0;
    if (((int64_t)c.columns * c.page / 16 + c.T / 16 + 2) * c.B > INT_MAX)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences of %d new tokens over up to %lld rows (2^35 in all)", who, c.B, c.T, (long long)c.columns * c.page);
    if (c.B > 65535 || c.Hq > 65535) return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences, %d heads (at most 65535 each)", who, c.B, c.Hq);
    return 0;
}

}  // namespace
}  // namespace ythip
