// paged_attn.hip — attention of new tokens over a paged KV cache (include/ythip.h,
// ythip_paged_attn) and over the pages that a score selects (ythip_paged_attn_sparse).

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
};

// What the DMA reads in place of rows that are not in use.
static __device__ const u32x4 zeros[1] = {{0u, 0u, 0u, 0u}};

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

__device__ __forceinline__ int tiles_of(const PagedArgs& a, int len, int tn, int kt) {
    return (int)(((int64_t)len + kt - 1) / kt) + (a.Kn != nullptr ? (tn + kt - 1) / kt : 0);
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

// dma16_soff for rows that this launch reads once: kept out of the caches' way (16 x 1 token over
// 8192 rows 82 -> 73 us, a tree of 64 over 131072 rows 140 -> 125 us).
__device__ __forceinline__ void dma16_stream(const void* sbase, uint32_t voff, uint32_t lds_wave_base) {
#if defined(__HIP_DEVICE_COMPILE__)
    asm volatile("s_mov_b32 m0, %2\n\tglobal_load_lds_dwordx4 %0, %1 nt"
                 :
                 : "v"(voff), "s"(sbase), "s"(lds_wave_base)
                 : "memory", "m0");
#endif
}

// mfma_chunk over 16 keys: lane l holds k = 4 (l / 16) + 0..3.
__device__ __forceinline__ f32x4 mfma_half(BF16, u32x2 a, u32x2 b, f32x4 c) {
    return __builtin_amdgcn_mfma_f32_16x16x16bf16_1k(__builtin_bit_cast(v4i16, a), __builtin_bit_cast(v4i16, b), c, 0, 0, 0);
}
__device__ __forceinline__ f32x4 mfma_half(F16, u32x2 a, u32x2 b, f32x4 c) {
    typedef _Float16 f16x4 __attribute__((ext_vector_type(4)));
    return __builtin_amdgcn_mfma_f32_16x16x16f16(__builtin_bit_cast(f16x4, a), __builtin_bit_cast(f16x4, b), c, 0, 0, 0);
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

__device__ __forceinline__ void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

// The order of a product's instructions: AHEAD of its READS reads from LDS first, then MF MFMAs and
// PER reads in turn; left to itself each read is waited for right away (a tree of 64 over
// 131072 rows 126 -> 122 us, two chunks of 512 85 -> 83).
template <int READS, int PER, int MF, int AHEAD>
__device__ __forceinline__ void interleave() {
#if defined(__HIP_DEVICE_COMPILE__)
    __builtin_amdgcn_sched_group_barrier(0x100, AHEAD < READS ? AHEAD : READS, 0);
#pragma unroll
    for (int i = AHEAD; i < READS; i += PER) {
        __builtin_amdgcn_sched_group_barrier(0x008, MF, 0);
        __builtin_amdgcn_sched_group_barrier(0x100, PER, 0);
    }
    __builtin_amdgcn_sched_group_barrier(0x008, (AHEAD < READS ? AHEAD : READS) / PER * MF, 0);
#endif
}

template <class T, int D, int QT, int WR>
struct Shape {
    static constexpr int ES = sizeof(typename T::raw), ROWB = D * ES, CH = ROWB / 16;
    static constexpr int KT = 16 * WR;       // keys of a tile
    static constexpr int RPI = 1024 / ROWB;  // rows of one DMA instruction
    static constexpr int IPG = 16 / RPI;     // instructions of 16 rows
    static constexpr int WK = 4 / WR;        // key groups of the workgroup
    static constexpr int KG = KT / 16, GPW = KG / WR, NI = GPW * IPG;
    static constexpr int TILE = KT * CH, STG = WK * TILE;  // in 16-byte chunks
    static constexpr int KS = CH / 4, DT = D / 16, RW = 16 * QT * WR;
    static constexpr int OLD = D + 4;  // floats of a row of O in LDS: 16 rows fall in different banks
    static constexpr int EPI = WK == 1 ? 0 : (WK * RW * (OLD + 2) * 4 + 15) / 16;  // the epilogue's use of the stages
    static constexpr int LDS = 4 * STG > EPI ? 4 * STG : EPI;
    static_assert(KG % WR == 0, "a wave stages whole groups of 16 rows");
};

// One workgroup: RW = 16 QT WR query rows of one KV head (row = token * G + head of the group)
// over a chunk of its sequence's tiles. Its waves are WR row groups x WK key groups: few
// rows share out the keys (WR = 1: each wave streams its own tiles, no barrier in the loop),
// many rows share the staged tile.
//   S^T = K . Q^T and O^T = V^T . P^T on the matrix cores, lane l holding query l % 16: the
//   softmax statistics are per lane, joined over the four lanes of a query by row swaps.
//   K and V reach LDS by DMA (16 rows of one page an address; a stage ahead), K chunks
//   XOR-swizzled by key, V 32-byte blocks likewise and read transposed.
//   Tiles run from the last to the first: new tokens, whose path is walked down from each
//   query's token once, then cached rows.
// Numerics: scores, maxima, sums and O in fp32; the weights of 16-bit inputs enter the second product
//   (and their sum) as two 16-bit numbers each (split2), a 256th or less of O's own rounding away
//   from fp32's. As one number each, half a step of O's type off, they would make O's error a third
//   larger and the kernel faster (1 token over 300 rows 8.2 -> 7.8 us, a tree of 64 over 131072 rows
//   137 -> 119, two chunks of 512 93 -> 78, a first chunk of 8192 665 -> 588). The comparisons by which the
//   cut and the loads were chosen, here and below, were made with one number.
// Measured (MI355X): 16 sequences, 1 token, 335 MB of rows 57 us (5.9 TB/s) and 5 us for the merge; a tree
//   of 64 over 131072 rows, 537 MB 131 us (4.1 TB/s, the matrix cores busy 41%) and 14; two chunks of 512 over up to 8192
//   rows, 45 GFLOP 91 us (500 TFLOP/s, the matrix cores busy 35%, no LDS conflicts: a stage's loads,
//   two products and softmax overlap only as far as two workgroups a CU let them) and 10; 1 token over
//   300 rows 8.2 us, trips to memory one after the other (lengths, pages, five stages of rows of which two are
//   in flight, O).
template <class T, int D, int QT, int WR, bool SPARSE>
__global__ __launch_bounds__(256, 2) void paged_attn_kernel(PagedArgs a) {
    using S = Shape<T, D, QT, WR>;
    constexpr int KT = S::KT;
    using raw = typename T::raw;
    constexpr bool F = std::is_same_v<T, F32>;
    constexpr int KMASK = S::CH - 1 < 15 ? S::CH - 1 : 15;
    constexpr int BMASK = (S::DT < 8 ? S::DT : 8) - 1;
    __shared__ u32x4 smem[S::LDS];
    __shared__ int16_t s_up[MAX_TREE];  // parents of the sequence's new tokens
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int l16 = lane & 15, g = lane >> 4;

    // (item, KV head, row tile): the row tiles of an item and head read the same rows, so
    // they go to one XCD (workgroup w runs on XCD w % 8)
    int gi, rt;
    {
        const int w = blockIdx.x, q = w >> 3;
        rt = q % a.row_tiles;
        gi = (q / a.row_tiles) * 8 + (w & 7);
    }
    if (gi >= a.items * a.Hkv) return;
    const int h = gi % a.Hkv;
    // the last items first: those with new tokens, whose tiles cost more, do not end alone
    const int item = a.items - 1 - gi / a.Hkv;

    const int R = SPARSE ? a.G : a.T * a.G;
    const int r0 = rt * S::RW;
    int b, t_one = 0;
    Cut cut;
    if constexpr (SPARSE) {
        t_one = item / a.target % a.T;
        b = item / a.target / a.T;
    } else if (a.target == 0) {  // a sequence a workgroup
        b = item;
    } else {
        cut = cut_of(a, KT, item, -1);
        if (cut.b < 0) return;
        b = cut.b;
    }
    int len, tn;
    if (!SPARSE && a.target > 0) len = cut.len, tn = cut.tn;
    else len = rows_in_use(a, b), tn = new_rows(a, b);
    b = uniform(b), len = uniform(len), tn = uniform(tn);
    const int t_first = SPARSE ? t_one : r0 / a.G, t_last = SPARSE ? t_one : min((min(R, r0 + S::RW) - 1) / a.G, tn - 1);
    const int32_t* table = a.table + b * a.ld_table;
    const int32_t* sel = nullptr;
    int nsel = 0, nct, lim = tn;
    if constexpr (SPARSE) {
        sel = a.sel + (((int64_t)b * a.Hkv + h) * a.T + t_one) * a.top_k;
        nsel = min(a.top_k, (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift));
        nct = (int)((((int64_t)nsel << a.shift) + KT - 1) / KT);
        lim = t_one + 1;
    } else {
        nct = (len + KT - 1) / KT;
    }
    const int nt = nct + (a.Kn != nullptr ? (lim + KT - 1) / KT : 0);
    // this workgroup's tiles of the sequence, and whether they are all
    int c0 = 0, c1 = nt;
    bool whole;
    if constexpr (SPARSE) {
        const int chunk = max((nt + a.target - 1) / a.target, a.stage), split = item % a.target;
        if (t_one >= tn || (split > 0 && split * chunk >= nt)) return;
        c0 = split * chunk;
        c1 = min(nt, c0 + chunk);
        whole = c0 == 0 && c1 == nt;
    } else if (a.target == 0) {
        whole = true;
    } else {
        c0 = max(cut.at, 0);
        c1 = min(cut.at + cut.chunk, nt);
        whole = cut.count == 1;
    }
    c0 = uniform(c0), c1 = uniform(c1);
    if (t_first >= tn) return;
    const int nst = (max(c1 - c0, 0) + S::WK - 1) / S::WK;

    // for the walks, where the chunk holds new tokens
    const bool walk = a.parents != nullptr && c1 > nct;
    if (walk) {
        for (int u = tid; u < tn; u += 256) {
            const int p = a.parents[b * a.ld_par + u];
            s_up[u] = (int16_t)(p >= 0 && p < u ? p : -1);
        }
        __syncthreads();
    }

    // this lane's query rows
    int tok[QT], cur[QT];
    u32x4 qf[QT][S::KS];
    constexpr uint32_t SIGN = F ? 0x80000000u : 0x80008000u;
    const float c = fabsf(a.scale_log2);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = r0 + wr * 16 * QT + qt * 16 + l16;
        // a row past the last reads the last's query, and what comes of it is not stored
        const int rq = min(r, R - 1), t = SPARSE ? t_one : rq / a.G, gh = SPARSE ? rq : rq - t * a.G;
        tok[qt] = r < R && t < tn ? t : -1;
        cur[qt] = tok[qt];
        const raw* qp = static_cast<const raw*>(a.Q) + b * a.qs[0] + (int64_t)(h * a.G + gh) * a.qs[1] + t * a.qs[2];
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks) qf[qt][ks] = *reinterpret_cast<const u32x4*>(qp + (ks * 4 + g) * (16 / S::ES));
    }

    // DMA: lane -> (row of the instruction, chunk), the chunk swizzled by the row in its 16: the
    // first instruction's, which the e-th turns by a constant
    const int dma_row = lane / S::CH;
    uint32_t kx, vx;  // bytes in the row
    {
        const int ps = lane % S::CH, r = dma_row;
        kx = (ps ^ (r & KMASK)) * 16;
        vx = F ? (ps ^ (((r >> 2) & 3) << 2)) * 16 : (((ps >> 1) ^ (r & BMASK)) * 32 + (ps & 1) * 16);
    }
    auto k_turn = [](int e) { return (uint32_t)((e * S::RPI & KMASK) * 16); };
    auto v_turn = [](int e) { return (uint32_t)(F ? (((e * S::RPI) >> 2 & 3) << 2) * 16 : (e * S::RPI & BMASK) * 32); };
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    const char *Kp = static_cast<const char*>(a.Kp) + h * a.ps[1] * S::ES, *Vp = static_cast<const char*>(a.Vp) + h * a.ps[1] * S::ES;
    const char* Kn = static_cast<const char*>(a.Kn) + (b * a.kns[0] + h * a.kns[1]) * S::ES;
    const char* Vn = static_cast<const char*>(a.Vn) + (b * a.vns[0] + h * a.vns[1]) * S::ES;

    auto tile_at = [&](int s) { return c1 - 1 - (s * S::WK + wk); };
    // The pages of stage s, looked up ahead: the table's columns, then the ids in the pool.
    int col[S::KG], id[S::KG];
    auto columns = [&](int s) {
        const int row = tile_at(s) * KT;
#pragma unroll
        for (int i = 0; i < S::KG; ++i) {
            const int slot = (row + 16 * i) >> a.shift;
            if constexpr (SPARSE) {
                col[i] = -1;
                if (row >= c0 * KT && slot < nsel) col[i] = scalar_word(sel + slot);
            } else {
                col[i] = slot;
            }
        }
    };
    auto ids = [&](int s) {
        const int ti = tile_at(s);
#pragma unroll
        for (int i = 0; i < S::KG; ++i) {
            id[i] = -1;
            if (ti >= c0 && ti < nct && col[i] >= 0 && col[i] << a.shift < len) id[i] = scalar_word(table + col[i]);
        }
    };
    // Stage s: the rows in use of each 16 (5 bits a group; 0: nothing was staged, the tile is
    // skipped) and this wave's share of the DMA. Rows that are not in use read zeros.
    int cols[S::KG];  // of the stage that `id` is for
    auto issue = [&](int s, auto with_new) {
        const int ti = tile_at(s);
        uint32_t pack = 0;
        if (ti < c0) return pack;
        const char *kb[S::KG], *vb[S::KG];
        const bool cached = !decltype(with_new)::value || ti < nct;
#pragma unroll
        for (int i = 0; i < S::KG; ++i) {
            int n;
            if (cached) {
                const int off = (ti * KT + 16 * i) & ((1 << a.shift) - 1);
                n = (uint32_t)id[i] < (uint32_t)a.pages ? min(max(len - (cols[i] << a.shift) - off, 0), 16) : 0;
                const int64_t at = (id[i] * a.ps[0] + off * a.ps[2]) * S::ES;
                kb[i] = Kp + at;
                vb[i] = Vp + at;
            } else {
                const int u = (ti - nct) * KT + 16 * i;
                n = u > t_last ? 0 : min(max(lim - u, 0), 16);
                kb[i] = Kn + u * a.kns[2] * S::ES;
                vb[i] = Vn + u * a.vns[2] * S::ES;
            }
            pack |= (uint32_t)n << (5 * i);
        }
        if (pack == 0) return pack;
#pragma unroll
        for (int j = 0; j < S::GPW; ++j) {
            // the wave's groups are i = wr GPW + j: selected without indexing by a variable
            const char *k = kb[j], *v = vb[j];
            if constexpr (WR > 1) {
#pragma unroll
                for (int i = 1; i < S::KG; ++i)
                    if (i == wr * S::GPW + j) k = kb[i], v = vb[i];
            }
            const int i = wr * S::GPW + j, n = (pack >> (5 * i)) & 31;
            const uint32_t lk = lds0 + ((s & 1) * 2 * S::STG + wk * S::TILE + i * 16 * S::CH) * 16, lv = lk + S::STG * 16;
            const int kr = (int)(cached ? a.ps[2] : a.kns[2]) * S::ES, vr = (int)(cached ? a.ps[2] : a.vns[2]) * S::ES;
            // the lane offsets anew each time: kept, they would not all fit the registers, and a register
            // read back from memory waits for every row in flight
            uint32_t kl = kx, vl = vx;
            int lane_row = dma_row;
            asm volatile("" : "+v"(kl), "+v"(vl), "+v"(lane_row));
            if (n == 16) {
                k = uniform(k), v = uniform(v);
#pragma unroll
                for (int e = 0; e < S::IPG; ++e) {
                    dma16_stream(k + (int64_t)e * S::RPI * kr, lane_row * kr + (kl ^ k_turn(e)), lk + e * 1024);
                    dma16_stream(v + (int64_t)e * S::RPI * vr, lane_row * vr + (vl ^ v_turn(e)), lv + e * 1024);
                }
            } else {
#pragma unroll
                for (int e = 0; e < S::IPG; ++e) {
                    const int row = e * S::RPI + lane_row;
                    const char* zero = reinterpret_cast<const char*>(zeros);
                    const char* ka = row < n ? k + (int64_t)row * kr + (kl ^ k_turn(e)) : zero;
                    const char* va = row < n ? v + (int64_t)row * vr + (vl ^ v_turn(e)) : zero;
                    dma16_async(ka, smem + (lk - lds0) / 16 + e * 64);
                    dma16_async(va, smem + (lv - lds0) / 16 + e * 64);
                }
            }
        }
        return pack;
    };

    // The largest weight in the running reference's unit is 2^UNIT: float16 has no number between 0 and 2^-24, so weights
    // against a largest of 1 would be lost below 2^-25 of it (and in the ranges that hold it alone); 2^14, the unit that
    // leaves room above, takes that to 2^-39. L and O have the same unit, so it cancels.
    constexpr float UNIT = std::is_same_v<T, F16> ? 14.f : 0.f;
    float m[QT];  // the largest score so far, before the scale
    f32x4 l[QT];  // ones . P^T: the sum of the weights as the product takes them, from the matrix cores
    f32x4 o[QT][S::DT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -INFINITY;
        l[qt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int t = 0; t < S::DT; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    const char* lds = reinterpret_cast<const char*>(smem);
    const int k_frag = l16 * S::ROWB + ((g ^ (l16 & KMASK)) << 4);
    const int v_key = 4 * g + (l16 >> 2);
    const int v_frag = F ? 4 * g * S::ROWB + ((l16 >> 2) ^ (g << 2)) * 16 + (l16 & 3) * 4
                         : v_key * S::ROWB + ((v_key & BMASK) << 5) + 8 * (l16 & 3);
    constexpr uint32_t EXP2 = std::is_same_v<T, BF16> ? 0x7f807f80u : 0x7c007c00u, STEP2 = std::is_same_v<T, BF16> ? 0x00800080u : 0x04000400u;
    constexpr int PK = F ? S::KG : S::KG >= 2 ? S::KG / 2 : 1;
    // over 32 keys, or the 16 that a tile has
    auto mfma_keys = [](u32x4 a, u32x4 b, f32x4 acc) {
        if constexpr (F) return acc;
        else if constexpr (S::KG >= 2) return mfma_chunk(T{}, a, b, acc);
        else return mfma_half(T{}, u32x2{a[0], a[1]}, u32x2{b[0], b[1]}, acc);
    };
    // o += V^T . P^T for output rows 16 t..16 t + 15 over the kk-th keys of the tile (CLEAN: elements of V that are
    // not finite taken as 0); pk: p as the MFMA takes it, in 16 bits with what is left of it in `rest`
    auto pv = [&](int v_at, int t, int kk, const u32x4 (&pk)[QT][PK], const u32x4 (&rest)[QT][PK], auto clean) {
        constexpr bool CLEAN = decltype(clean)::value;
        if constexpr (F) {
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                // chunk 4 t + l16 / 4 of key 16 kk + 4 g + j, stored at the chunk ^ 4 g
                float v = *reinterpret_cast<const float*>(lds + ((v_at ^ (t << 6)) + (kk * 16 + j) * S::ROWB));
                if (CLEAN) v = fabsf(v) < INFINITY ? v : 0.f;
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    o[qt][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, __uint_as_float(pk[qt][kk][j]), o[qt][t], 0, 0, 0);
            }
        } else {
            u32x4 vf = {0u, 0u, 0u, 0u};
#pragma unroll
            for (int hh = 0; hh < (S::KG >= 2 ? 2 : 1); ++hh) {
                // 32-byte block t of key 16 (2 kk + hh) + 4 g + l16 / 4, stored at the block ^ (key & BMASK)
                const u32x2 w = lds_read_tr16(smem, (v_at ^ (t << 5)) + (2 * kk + hh) * 16 * S::ROWB);
                vf[2 * hh] = w[0];
                vf[2 * hh + 1] = w[1];
            }
            if (CLEAN) {
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    // an exponent of ones carries into the bit above it
                    const uint32_t odd = (((vf[e] & EXP2) + STEP2) >> 15) & 0x00010001u;
                    vf[e] &= ~(odd * 0xffffu);
                }
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) o[qt][t] = mfma_keys(vf, pk[qt][kk], o[qt][t]);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) o[qt][t] = mfma_keys(vf, rest[qt][kk], o[qt][t]);
        }
    };

    auto compute = [&](int s, uint32_t pack, auto with_new) {
        constexpr bool NEW = decltype(with_new)::value;
        const int ti = tile_at(s);
        // LDS bytes of this lane's first K and V fragments; the others are a constant's turn and distance
        // away (worked out each time: kept, they would not all fit the registers)
        const int stage = ((s & 1) * 2 * S::STG + wk * S::TILE) * 16;
        int k_at = stage + k_frag, v_at = stage + S::STG * 16 + v_frag;
        asm volatile("" : "+v"(k_at), "+v"(v_at));
        const u32x4* cV = smem + (stage >> 4) + S::STG;
        const bool cached = !NEW || ti < nct;
        uint64_t see[QT];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) see[qt] = 0;
        bool paths = false;  // some query does not see all of a tile of new tokens
        if (!cached) {
            // the new tokens of this tile on each query's path
            const int u0 = (ti - nct) * KT;
            bool any = false;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                if (walk) {
                    while (cur[qt] >= u0) {
                        if (cur[qt] < u0 + KT) see[qt] |= 1ull << (cur[qt] - u0);
                        cur[qt] = s_up[cur[qt]];
                    }
                } else if (tok[qt] >= u0) {
                    see[qt] = tok[qt] - u0 >= 63 ? ~0ull : (2ull << (tok[qt] - u0)) - 1;
                }
                any = any || see[qt] != 0;
                paths = paths || see[qt] != (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
            }
            if (__ballot(any) == 0) return;
            paths = __ballot(paths) != 0;
        }
        __builtin_amdgcn_s_setprio(1);  // the matrix cores' turns first: the other wave has its softmax to go on with
        f32x4 p[QT][S::KG];
#pragma unroll
        for (int kt = 0; kt < S::KG; ++kt) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(lds + ((k_at ^ (ks << 6)) + kt * 16 * S::ROWB));
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) p[qt][kt] = mfma_chunk(T{}, kf, qf[qt][ks], p[qt][kt]);
            }
        }
        if constexpr (!F) interleave<S::KG * S::KS, 1, QT, 6>();
        constexpr uint32_t FULL = S::KG == 1 ? 16u : S::KG == 2 ? 16u | 16u << 5 : 16u | 16u << 5 | 16u << 10 | 16u << 15;
        __builtin_amdgcn_s_setprio(0);
        if (paths || pack != FULL) {
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt) {
                // the rows in use of the group, and the path's bits, of this lane's four keys
                const int n = (int)((pack >> (5 * kt)) & 31) - 4 * g;
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) {
                    const uint32_t vis = !paths ? 15u : (uint32_t)(see[qt] >> (kt * 16 + 4 * g));
#pragma unroll
                    for (int r = 0; r < 4; ++r) p[qt][kt][r] = r < n && (vis >> r & 1) ? p[qt][kt][r] : -INFINITY;
                }
            }
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float mx = -INFINITY;  // of the scores before the scale (it is positive: a negative one went into Q)
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, p[qt][kt][r]);
            const float top = __builtin_elementwise_maximum(m[qt], max_across_rows(mx));
            const float ref = top == -INFINITY ? 0.f : top;  // nothing seen yet: every weight is 0
            const float corr = __builtin_amdgcn_exp2f((m[qt] - ref) * c);
            m[qt] = top;
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    // the difference first: scaled, the largest score is rounded, by more than an exponent can hold
                    // where it is beyond 2^31
                    p[qt][kt][r] = __builtin_amdgcn_exp2f(fmaf(p[qt][kt][r] - ref, c, UNIT));
                }
            l[qt] *= corr;
            if (__ballot(corr != 1.0f) != 0) {
#pragma unroll
                for (int t = 0; t < S::DT; ++t) o[qt][t] *= corr;
            }
        }
        uint64_t odd = 0;
        if (paths) {
            // 0 . V is NaN for a V that is not finite: such elements are left out of the product and
            // added (their weight cannot change what comes of them) for the queries that see the row
#pragma unroll 4
            for (int i = 0; i < S::TILE / 64; ++i) {
                const u32x4 v = cV[i * 64 + lane];
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (F) bad = bad || (v[e] & 0x7f800000u) == 0x7f800000u;
                    else bad = bad || (((v[e] & EXP2) + STEP2) & 0x80008000u) != 0;
                }
                const uint64_t w = __ballot(bad);
                if (w != 0) {
#pragma unroll
                    for (int r = 0; r < S::RPI; ++r)
                        if (w >> (r * S::CH) & ((S::CH == 64 ? 0ull : 1ull << S::CH) - 1)) odd |= 1ull << (i * S::RPI + r);
                }
            }
        }
        u32x4 pk[QT][PK], rest[QT][PK];
        // the kk-th keys' weights as the product takes them, and their sum
        auto weigh = [&](int kk) {
            constexpr uint32_t ONE2 = std::is_same_v<T, BF16> ? 0x3F803F80u : 0x3C003C00u;
            constexpr u32x4 ones = {ONE2, ONE2, ONE2, ONE2};
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                if constexpr (F) {
                    pk[qt][kk] = __builtin_bit_cast(u32x4, p[qt][kk]);
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        l[qt] = __builtin_amdgcn_mfma_f32_16x16x4f32(1.0f, __uint_as_float(pk[qt][kk][j]), l[qt], 0, 0, 0);
                } else {
#pragma unroll
                    for (int i = 0; i < (S::KG >= 2 ? 4 : 2); ++i) {
                        const f32x4 x = p[qt][S::KG >= 2 ? 2 * kk + i / 2 : 0];
                        uint32_t hi, left;
                        split2<T>(x[2 * (i & 1)], x[2 * (i & 1) + 1], hi, left);
                        pk[qt][kk][i] = hi;
                        rest[qt][kk][i] = left;
                    }
                }
            }
            if constexpr (!F) {
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) l[qt] = mfma_keys(ones, pk[qt][kk], l[qt]);
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) l[qt] = mfma_keys(ones, rest[qt][kk], l[qt]);
            }
        };
        // in 16 bits over cached rows the weights of later keys are split while the matrix cores have those of earlier
        // ones (a tree of 64 over 131072 rows 147 -> 140 us); with new tokens the registers do not reach for that
        constexpr bool AS_IT_GOES = !NEW && !F;
        if constexpr (!AS_IT_GOES) {
#pragma unroll
            for (int kk = 0; kk < PK; ++kk) weigh(kk);
        }
        auto product = [&](auto clean) {
#pragma unroll
            for (int kk = 0; kk < PK; ++kk) {
                if constexpr (AS_IT_GOES) weigh(kk);
#pragma unroll
                for (int t = 0; t < S::DT; ++t) pv(v_at, t, kk, pk, rest, clean);
            }
            if constexpr (!F && !decltype(clean)::value) interleave<S::DT * S::KG, S::KG >= 2 ? 2 : 1, 2 * QT, 10>();
        };
        if (!NEW || odd == 0) {
            __builtin_amdgcn_s_setprio(1);
            product(std::false_type{});
            __builtin_amdgcn_s_setprio(0);
            return;
        }
        asm volatile("" ::: "memory");  // or the two products are run both and one result taken
        product(std::true_type{});
        for (uint64_t left = odd; left != 0; left &= left - 1) {
            const int u = __builtin_ctzll(left);
            const char* row = reinterpret_cast<const char*>(cV) + u * S::ROWB;
#pragma unroll
            for (int t = 0; t < S::DT; ++t) {
                float v[4];
                if constexpr (F) {
                    const f32x4 w = *reinterpret_cast<const f32x4*>(row + ((4 * t + g) ^ (((u >> 2) & 3) << 2)) * 16);
                    for (int i = 0; i < 4; ++i) v[i] = w[i];
                } else {
                    const u32x2 w = *reinterpret_cast<const u32x2*>(row + (t ^ (u & BMASK)) * 32 + g * 8);
                    for (int i = 0; i < 2; ++i) v[2 * i] = lo_as_f32(T{}, w[i]), v[2 * i + 1] = hi_as_f32(T{}, w[i]);
                }
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const float add = fabsf(v[i]) < INFINITY ? 0.f : v[i];
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) o[qt][t][i] += (see[qt] >> u & 1) ? add : 0.f;
                }
            }
        }
    };

    uint32_t here = 0, next = 0;  // what is staged for s and s + 1
    auto step = [&](int s, auto with_new) {
        // the lookups of stage s + 2 run beside the arithmetic of stage s
        ids(s + 2);
#pragma unroll
        for (int i = 0; i < S::KG; ++i) cols[i] = col[i];
        columns(s + 3);
        if (next != 0) wait_vmcnt<2 * S::NI>();  // stage s has landed, s + 1 is in flight
        else wait_vmcnt<0>();
        if constexpr (WR > 1) wg_barrier();
        else asm volatile("" ::: "memory");
        if (here != 0) compute(s, here, with_new);
        if constexpr (WR > 1) wg_barrier();
        else asm volatile("" ::: "memory");
        here = next;
        next = s + 2 < nst ? issue(s + 2, with_new) : 0;
    };
    // stages with new tokens, then those of cached rows alone: a loop of its own, that holds none of
    // the paths' state in registers
    const int s_new = (max(c1 - max(c0, nct), 0) + S::WK - 1) / S::WK;
    {
        // the first two stages: both lookups and the queries' latency side by side
        int ids0[S::KG], col0[S::KG];
        columns(0);
        ids(0);
#pragma unroll
        for (int i = 0; i < S::KG; ++i) ids0[i] = id[i], col0[i] = col[i];
        columns(1);
        ids(1);
        int ids1[S::KG], col1[S::KG];
#pragma unroll
        for (int i = 0; i < S::KG; ++i) ids1[i] = id[i], col1[i] = col[i];
        columns(2);
        // the queries are there before the first DMA: waited for in the loop they would have every
        // row in flight waited for
        const uint32_t flip = a.scale_log2 < 0.f ? SIGN : 0u;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks) {
                qf[qt][ks] ^= u32x4{flip, flip, flip, flip};
                asm volatile("" : "+v"(qf[qt][ks]));
            }
        for (int s = 0; s < 2; ++s) {
#pragma unroll
            for (int i = 0; i < S::KG; ++i) id[i] = s == 0 ? ids0[i] : ids1[i], cols[i] = s == 0 ? col0[i] : col1[i];
            here = next;
            next = s < nst ? issue(s, std::true_type{}) : 0;
        }
    }
    for (int s = 0; s < s_new; ++s) step(s, std::true_type{});
    for (int s = s_new; s < nst; ++s) step(s, std::false_type{});
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) m[qt] *= c;
    // the place of row r's result: O itself, or this item's partial
    auto store4 = [&](int r, int d, f32x4 v, float M, float L) {
        const int t = SPARSE ? t_one : r / a.G, gh = SPARSE ? r : r - t * a.G;
        if (r >= R || t >= tn) return;
        if (whole) {
            raw* op = static_cast<raw*>(a.O) + b * a.os[0] + (int64_t)(h * a.G + gh) * a.os[1] + t * a.os[2] + d;
            const float inv = M == -INFINITY ? 0.f : 1.0f / L;
            v = M == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : v * inv;
            if constexpr (F) *reinterpret_cast<f32x4*>(op) = v;
            else *reinterpret_cast<u32x2*>(op) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            return;
        }
        const int64_t at = ((int64_t)item * a.Hkv + h) * R + r;
        *reinterpret_cast<f32x4*>(a.part + at * D + d) = v;
        if (d == 0) {
            a.part_ml[2 * at] = M;
            a.part_ml[2 * at + 1] = L;
        }
    };
    if constexpr (S::WK == 1) {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int t = 0; t < S::DT; ++t) store4(r0 + wr * 16 * QT + qt * 16 + l16, 16 * t + 4 * g, o[qt][t], m[qt], l[qt][0]);
    } else {
        // the key groups' results side by side in LDS, then joined
        float* so = reinterpret_cast<float*>(smem);
        float* sm = so + S::WK * S::RW * S::OLD;
        __syncthreads();
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            const int row = wk * S::RW + wr * 16 * QT + qt * 16 + l16;
#pragma unroll
            for (int t = 0; t < S::DT; ++t) *reinterpret_cast<f32x4*>(so + row * S::OLD + 16 * t + 4 * g) = o[qt][t];
            if (g == 0) {
                sm[2 * row] = m[qt];
                sm[2 * row + 1] = l[qt][0];
            }
        }
        __syncthreads();
        for (int i = tid; i < S::RW * D / 4; i += 256) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float M = -INFINITY, L = 0.f;
#pragma unroll
            for (int k = 0; k < S::WK; ++k) M = __builtin_elementwise_maximum(M, sm[2 * (k * S::RW + row)]);
            const float ref = M == -INFINITY ? 0.f : M;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < S::WK; ++k) {
                const float w = __builtin_amdgcn_exp2f(sm[2 * (k * S::RW + row)] - ref);
                L += w * sm[2 * (k * S::RW + row) + 1];
                v += w * *reinterpret_cast<const f32x4*>(so + (k * S::RW + row) * S::OLD + d);
            }
            store4(r0 + row, d, v, M, L);
        }
    }
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

// ---------------------------------------------------------------------------
// The choice of pages
// ---------------------------------------------------------------------------

// A score as an unsigned number of the same order: NaN lowest (as -inf), both zeros alike.
__device__ __forceinline__ uint64_t rank_of(double s) {
    s = s == s ? s + 0.0 : -INFINITY;
    const uint64_t u = __builtin_bit_cast(uint64_t, s);
    return (int64_t)u < 0 ? ~u : u | 1ull << 63;
}
constexpr uint64_t RANK_TOP = ~0ull;  // the last page's: above every score's

// The sum of a token's queries of one KV head, lane l16's D / 16 of it (dims 64 v + 4 l16 + 0..3).
template <class T, int D>
__device__ __forceinline__ void query_sum(const PagedArgs& a, int b, int h, int t, int l16, double (&q)[D / 16]) {
#pragma unroll
    for (int e = 0; e < D / 16; ++e) q[e] = 0.0;
    for (int g = 0; g < a.G; ++g) {
        const int64_t at = b * a.qs[0] + (int64_t)(h * a.G + g) * a.qs[1] + t * a.qs[2] + l16 * 4;
#pragma unroll
        for (int e = 0; e < D / 16; ++e) q[e] += (double)load_as_f32<T>(a.Q, at + e / 4 * 64 + e % 4);
    }
}
// Key sums of U pages of a sequence (first, first + 4, ...): 16 lanes a page, all in flight together.
template <int D, int U>
struct PageSums {
    static constexpr int E = D / 16, V = E / 4;
    int id[U];
    f32x4 x[U][V];
    __device__ __forceinline__ void load(const PagedArgs& a, int b, int h, int first, int n, int l16) {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            id[u] = first + 4 * u < n ? a.table[b * a.ld_table + first + 4 * u] : -1;
            if ((uint32_t)id[u] >= (uint32_t)a.pages) id[u] = -1;
        }
#pragma unroll
        for (int u = 0; u < U; ++u)
#pragma unroll
            for (int v = 0; v < V; ++v) {
                x[u][v] = f32x4{0.f, 0.f, 0.f, 0.f};
                // 16 lanes read 256 consecutive bytes
                if (id[u] >= 0) {
                    const float* p = a.sums + id[u] * a.ss[0] + h * a.ss[1] + v * 64 + l16 * 4;
                    x[u][v] = f32x4{p[0], p[1], p[2], p[3]};
                }
            }
    }
    // out[i]: page i's rank, the last page's above all
    __device__ __forceinline__ void ranks(const double (&q)[E], int first, int n, int l16, uint64_t* out) const {
#pragma unroll
        for (int u = 0; u < U; ++u) {
            double s = 0.0;
#pragma unroll
            for (int e = 0; e < E; ++e) s = fma(q[e], (double)x[u][e / 4][e % 4], s);
#pragma unroll
            for (int off = 8; off >= 1; off >>= 1) s += __shfl_xor(s, off, 64);
            const int i = first + 4 * u;
            if (l16 == 0 && i < n) out[i] = i == n - 1 ? RANK_TOP : rank_of(id[u] >= 0 ? s : -INFINITY);
        }
    }
};

// Scores of 64 pages of one KV head for TB tokens: 16 lanes a page (D / 16 dims each), four
// pages a wave at a time, all a lane's pages in flight together. The products are of float32 sums
// and sums of the group's queries, all in 64 bits (the fp64 rate is the fp32 rate here, and the
// time is that of the sums' bytes): scores that differ in their first 50 bits keep their order,
// so the choice does not depend on how they were added up.
// 8 MB of sums, 1 token 5.3 us; 16 sequences, 4 tokens, 21 MB 14 us.
template <class T, int D, int TB>
__global__ __launch_bounds__(256) void paged_score_kernel(PagedArgs a) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, l16 = lane & 15;
    const int h = blockIdx.y % a.Hkv, t0 = blockIdx.y / a.Hkv * TB, b = blockIdx.z;
    const int tn = new_rows(a, b), len = rows_in_use(a, b);
    const int n = (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift);
    const int first = (blockIdx.x * 4 + wave) * 16 + (lane >> 4);  // and + 4, + 8, + 12
    if (t0 >= tn || blockIdx.x * 64 >= n) return;
    PageSums<D, 4> sums;
    sums.load(a, b, h, first, n, l16);
#pragma unroll
    for (int k = 0; k < TB; ++k) {
        const int t = t0 + k;
        if (t >= tn) return;
        double q[D / 16];
        query_sum<T, D>(a, b, h, t, l16, q);
        sums.ranks(q, first, n, l16, a.rank + (((int64_t)b * a.Hkv + h) * a.T + t) * a.columns);
    }
}

// The top_k highest of a row of ranks, ascending by page: the k-th highest rank is found eight
// bits at a time (a histogram in LDS of the ranks that agree with the bits so far, in 16
// copies: ranks of like scores fall into few bins), until a bin is taken whole; scores are
// far apart in their first 24 bits, so that is three rounds mostly. Then a wave takes a run of pages
// each and writes its share in order. Bound by the rounds' barriers: 8 rows of 2048 ranks and 512 rows
// of up to 512 both 7.8 us. Where SCORE, the workgroup scores its row's pages itself, a launch less:
// at most SCORED, what its waves have in flight at once (4 sequences, 5 tokens, 88 pages 23.7 -> 19.5 us in all;
// 250 pages in two turns 18.3 -> 20.8).
constexpr int SCORED = 128;
constexpr int SEL_KEEP = 8;  // ranks a thread keeps in registers (longer rows are read again)
template <class T, int D, int SEL, bool SCORE>  // SEL threads
__global__ __launch_bounds__(SEL) void paged_select_kernel(PagedArgs a) {
    static_assert(!SCORE || SCORED == SEL / 64 * 32);
    constexpr int COPIES = 16;
    __shared__ uint64_t s_rank[SCORE ? SCORED : 1];
    __shared__ int s_hist[256 * COPIES], s_bin[256], s_found[3], s_count[SEL / 64][2];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z;
    const int64_t row = ((int64_t)b * a.Hkv + h) * a.T + t;
    int32_t* sel = a.sel + row * a.top_k;
    const int len = rows_in_use(a, b);
    const int n = t < new_rows(a, b) ? (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift) : 0;
    if (n <= a.top_k) {
        for (int i = tid; i < a.top_k; i += SEL) sel[i] = i < n ? i : -1;
        return;
    }
    const uint64_t* rank = SCORE ? s_rank : a.rank + row * a.columns;
    if constexpr (SCORE) {
        double q[D / 16];
        query_sum<T, D>(a, b, h, t, lane & 15, q);
        const int first = wave * 32 + (lane >> 4);
        PageSums<D, 8> sums;
        sums.load(a, b, h, first, n, lane & 15);
        sums.ranks(q, first, n, lane & 15, s_rank);
        __syncthreads();
    }
    // wave w has the pages from w * run on, 64 at a time
    const int run = (n + SEL - 1) / SEL * 64;
    const bool kept = n <= SEL * SEL_KEEP;
    uint64_t r[SEL_KEEP];
    if (kept) {
#pragma unroll
        for (int j = 0; j < SEL_KEEP; ++j) {
            const int i = wave * run + j * 64 + lane;
            r[j] = j * 64 < run && i < n ? rank[i] : 0;
        }
    }
    // f(j-th rank of this lane, whether it exists)
    auto each = [&](auto f) {
        if (kept) {
#pragma unroll
            for (int j = 0; j < SEL_KEEP; ++j)
                if (j * 64 < run) f(r[j], wave * run + j * 64 + lane, wave * run + j * 64 + lane < n);
        } else {
            for (int j = 0; j * 64 < run; ++j) {
                const int i = wave * run + j * 64 + lane;
                f(i < n ? rank[i] : 0, i, i < n);
            }
        }
    };
    uint64_t prefix = 0;  // of the k-th highest rank, above bit `low`
    int low = 64, want = a.top_k;  // still to be taken among the ranks with that prefix
    for (;;) {
        low -= 8;
        for (int i = tid; i < 256 * COPIES; i += SEL) s_hist[i] = 0;
        __syncthreads();
        each([&](uint64_t x, int, bool is) {
            if (is && (low == 56 || x >> (low + 8) == prefix)) atomicAdd(&s_hist[(int)(x >> low & 255) * COPIES + (lane & (COPIES - 1))], 1);
        });
        __syncthreads();
        if (tid < 256) {
            int c = 0;
#pragma unroll
            for (int i = 0; i < COPIES; ++i) c += s_hist[tid * COPIES + ((i + tid) & (COPIES - 1))];
            s_bin[tid] = c;
        }
        __syncthreads();
        if (wave == 0) {
            // lane l sums bins 255 - 4 l down; the bin that brings the sum to `want`
            int v[4], mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine += v[i] = s_bin[255 - 4 * lane - i];
            int before = wave_scan(mine) - mine;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (before < want && before + v[i] >= want) {
                    s_found[0] = 255 - 4 * lane - i;
                    s_found[1] = want - before;
                    s_found[2] = v[i];
                }
                before += v[i];
            }
        }
        __syncthreads();
        prefix = prefix << 8 | (uint64_t)s_found[0];
        want = s_found[1];
        if (low == 0 || s_found[2] == want) break;
    }
    // above the prefix: taken; with it: the first `want`
    int over = 0, same = 0;
    each([&](uint64_t x, int, bool is) {
        over += __popcll(__ballot(is && x >> low > prefix));
        same += __popcll(__ballot(is && x >> low == prefix));
    });
    if (lane == 0) s_count[wave][0] = over, s_count[wave][1] = same;
    __syncthreads();
    over = same = 0;
    for (int w = 0; w < wave; ++w) over += s_count[w][0], same += s_count[w][1];
    const uint64_t below = (1ull << lane) - 1;
    each([&](uint64_t x, int i, bool is) {
        const uint64_t o = __ballot(is && x >> low > prefix), e = __ballot(is && x >> low == prefix);
        const int eq = same + __popcll(e & below), at = over + __popcll(o & below) + min(eq, want);
        if ((o >> lane & 1) || ((e >> lane & 1) && eq < want)) sel[at] = i;
        over += __popcll(o);
        same += __popcll(e);
    });
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
Plan plan_of(int dtype, int B, int Hkv, int G, int T, int d, int columns, int page, int top_k) {
    const int rows = top_k > 0 ? G : (int)std::min<int64_t>((int64_t)T * G, 1 << 20);
    Plan p;
    // 16 rows or 32 leave the keys to the four waves; more share each staged tile between
    // two or four of them
    p.qt = rows <= 16 ? 1 : 2;
    p.wr = rows <= 32 || top_k > 0 ? 1 : rows <= 64 ? 2 : 4;
    p.kt = 16 * p.wr;
    const int64_t all_rows = top_k > 0 ? G : (int64_t)T * G;
    const int rw = 16 * p.qt * p.wr;
    p.row_tiles = (int)((all_rows + rw - 1) / rw);
    const int64_t per = (int64_t)Hkv * p.row_tiles;
    p.stage = 4 / p.wr;
    // Workgroups that the work is dealt to: the 512 that run at once (of 768 that stream their own rows
    // a third waits: 16 sequences, 1 token, up to 8192 rows 60 -> 63 us; 1024 that share tiles: a tree of 64 over
    // 131072 rows 126 -> 146 us).
    // Half of them where a workgroup has a CU to itself (128 rows of fp32, d 128: 136 KB of LDS) and the
    // sequences are few, whose items are alike (a tree of 64 over 32768 rows 219 -> 198 us; 16 ragged
    // sequences 152 -> 188 us, left as they were).
    const bool alone = dtype == YTHIP_F32 && d == 128 && p.wr > 1 && B <= EVEN_SEQS;
    // And half where rows are streamed and a sequence has many ranges, which are alike then and whose
    // partials cost more than the second workgroup of a CU brings (1 token, 4 KV heads, 60000 rows 32 ->
    // 29 us; 16 sequences, 8 heads, 4 ranges each 60 -> 67 us, left as they were).
    const bool many = p.wr == 1 && SLOTS / per >= 8 * (int64_t)B * (top_k > 0 ? T : 1);
    const int64_t slots = alone || many ? SLOTS / 2 : SLOTS;
    p.short_run = p.wr > 1 ? 4 : 0;
    const int64_t new_tiles = ((int64_t)T + p.kt - 1) / p.kt;
    const int64_t seq_rows = (int64_t)std::min(top_k > 0 ? top_k : columns, columns) * page;
    const int64_t tiles = (seq_rows + p.kt - 1) / p.kt + new_tiles, most = (tiles + p.stage - 1) / p.stage;
    int64_t part_items = 0;
    if (top_k > 0) {
        // (a token's pages in ranges of at least the stages that least_stages explains)
        const int64_t root = std::max<int64_t>(1, (int64_t)std::ceil(std::sqrt((double)most / 20)));
        p.target = (int)std::max<int64_t>(1, std::min((most + root - 1) / root, (slots + per * B * T - 1) / (per * B * T)));
        p.items = (int64_t)B * T * p.target;
        if (p.target > 1) part_items = p.items;
    } else if (most <= WHOLE) {
        p.target = 0;
        p.items = B;
    } else {
        int64_t ranges = slots / per;
        p.even = B <= EVEN_SEQS && B <= ranges && ranges <= 8 * B;
        // the items at the ends of a few sequences count among the slots too
        if (!p.even && B - 1 <= ranges / 2) ranges -= B - 1;
        p.target = (int)std::min(std::max<int64_t>(1, ranges), B * most);
        p.items = (int64_t)p.target + (p.even ? 0 : B - 1);
        if (p.target > 1) part_items = p.items;  // one range holds every sequence whole
    }
    const int64_t part_rows = part_items * Hkv * all_rows;
    p.part_bytes = (size_t)part_rows * d * sizeof(float);
    p.ml_bytes = ((size_t)part_rows * 2 * sizeof(float) + 15) / 16 * 16;
    // (the partials behind them are read 16 bytes at a time)
    p.rank_bytes = top_k > 0 ? ((size_t)B * Hkv * T * columns * sizeof(uint64_t) + 15) / 16 * 16 : 0;
    return p;
}

template <class T, int D, int QT, int WR, bool SPARSE>
int launch(const PagedArgs& a, const Plan& p, hipStream_t s) {
    const int64_t groups = (p.items * a.Hkv + 7) / 8 * 8;
    using S = Shape<T, D, QT, WR>;
    paged_attn_kernel<T, D, QT, WR, SPARSE><<<(int)(groups * p.row_tiles), 256, 0, s>>>(a);
    if (p.part_bytes > 0) {
        constexpr int ROWS = 256 / D;  // of a wave
        const int rows = a.T * a.G;
        // few rows: a workgroup's waves share them (16 rows of 32 partials 6.8 -> 4.9 us; 5000 rows of
        // about 12 8.3 -> 9.9)
        if ((int64_t)a.B * a.Hkv * rows <= 512)
            paged_merge_kernel<T, D, SPARSE, true><<<dim3((rows + ROWS - 1) / ROWS, a.Hkv, a.B), 256, 0, s>>>(a, S::KT);
        else
            paged_merge_kernel<T, D, SPARSE, false><<<dim3((rows + 4 * ROWS - 1) / (4 * ROWS), a.Hkv, a.B), 256, 0, s>>>(a, S::KT);
    }
    return status_of(hipGetLastError());
}
template <class T, int D, bool SPARSE>
int run_typed(const PagedArgs& a, const Plan& p, hipStream_t s) {
    if constexpr (SPARSE) {
        constexpr int TB = 4;
        const dim3 rows(a.T, a.Hkv, a.B);
        if (a.columns <= SCORED) {
            paged_select_kernel<T, D, 256, true><<<rows, 256, 0, s>>>(a);
        } else {
            if (a.columns > 0)
                paged_score_kernel<T, D, TB><<<dim3((a.columns + 63) / 64, a.Hkv * ((a.T + TB - 1) / TB), a.B), 256, 0, s>>>(a);
            if (a.columns > 1024) paged_select_kernel<T, D, 1024, false><<<rows, 1024, 0, s>>>(a);
            else paged_select_kernel<T, D, 256, false><<<rows, 256, 0, s>>>(a);
        }
    }
    if (p.qt == 1) return launch<T, D, 1, 1, SPARSE>(a, p, s);
    if constexpr (!SPARSE) {
        if (p.wr == 2) return launch<T, D, 2, 2, SPARSE>(a, p, s);
        if (p.wr == 4) return launch<T, D, 2, 4, SPARSE>(a, p, s);
    }
    return launch<T, D, 2, 1, SPARSE>(a, p, s);
}
template <bool SPARSE>
int run(int dtype, int d, PagedArgs& a, void* ws, hipStream_t s) {
    const Plan p = plan_of(dtype, a.B, a.Hkv, a.G, a.T, d, a.columns, 1 << a.shift, SPARSE ? a.top_k : 0);
    if (!launchable((p.items * a.Hkv + 8) * p.row_tiles, 256))
        return fail(YTHIP_EUNSUPPORTED, "paged attention: %lld workgroups (2^24 - 1 at most)", (long long)(p.items * a.Hkv * p.row_tiles));
    a.target = p.target, a.stage = p.stage, a.items = (int)p.items, a.row_tiles = p.row_tiles, a.even = p.even, a.short_run = p.short_run;
    char* w = static_cast<char*>(ws);
    a.rank = reinterpret_cast<uint64_t*>(w);
    a.part = reinterpret_cast<float*>(w + p.rank_bytes);
    a.part_ml = reinterpret_cast<float*>(w + p.rank_bytes + p.part_bytes);
    if (dtype == YTHIP_F32) return d == 64 ? run_typed<F32, 64, SPARSE>(a, p, s) : run_typed<F32, 128, SPARSE>(a, p, s);
    if (dtype == YTHIP_F16) return d == 64 ? run_typed<F16, 64, SPARSE>(a, p, s) : run_typed<F16, 128, SPARSE>(a, p, s);
    return d == 64 ? run_typed<BF16, 64, SPARSE>(a, p, s) : run_typed<BF16, 128, SPARSE>(a, p, s);
}

size_t workspace(int dtype, int B, int Hq, int Hkv, int T, int d, int columns, int page, int top_k) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || d <= 0 || columns < 0 || page <= 0 || top_k < 0 || Hq % Hkv != 0) return 0;
    return plan_of(dtype, B, Hkv, Hq / Hkv, T, d, columns, page, top_k).bytes();
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
    a.sel = nullptr, a.top_k = 0, a.sums = nullptr, a.rank = nullptr;
    if (((int64_t)c.columns * c.page / 16 + c.T / 16 + 2) * c.B > INT_MAX)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences of %d new tokens over up to %lld rows (2^35 in all)", who, c.B, c.T, (long long)c.columns * c.page);
    if (c.B > 65535 || c.Hq > 65535) return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences, %d heads (at most 65535 each)", who, c.B, c.Hq);
    return 0;
}

}  // namespace
}  // namespace ythip

using namespace ythip;

extern "C" {

__attribute__((visibility("default"))) size_t ythip_paged_attn_workspace_size(int dtype, int B, int Hq, int Hkv, int T,
                                                                              int d, int columns, int page) {
    return workspace(dtype, B, Hq, Hkv, T, d, columns, page, 0);
}

__attribute__((visibility("default"))) int ythip_paged_attn(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[3], int pages, int page, const int32_t* table, int64_t ld_table, int columns,
    const int32_t* kv_len, const int32_t* parents, int64_t ld_parents, const int32_t* new_len, void* O,
    const int64_t o_str[3], float scale, void* workspace_, size_t ws_bytes, void* stream) {
    const char* who = "ythip_paged_attn";
    PagedArgs a;
    bool done;
    const Call c = {dtype, B, Hq, Hkv, T, d, Q, q_str, Kn, kn_str, Vn, vn_str, Kp, Vp, pool_str, pages, page,
                    table, ld_table, columns, kv_len, parents, ld_parents, new_len, O, o_str, scale};
    const int st = prepare(who, c, a, done);
    if (st || done) return st;
    if (const int e = check_workspace(who, workspace(dtype, B, Hq, Hkv, T, d, columns, page, 0), workspace_, ws_bytes)) return e;
    return run<false>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
}

__attribute__((visibility("default"))) size_t ythip_paged_attn_sparse_workspace_size(int dtype, int B, int Hq, int Hkv,
                                                                                     int T, int d, int columns,
                                                                                     int page, int top_k) {
    return top_k > 0 ? workspace(dtype, B, Hq, Hkv, T, d, columns, page, top_k) : 0;
}

__attribute__((visibility("default"))) int ythip_paged_attn_sparse(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[3], int pages, int page, const float* sums, const int64_t sums_str[2], const int32_t* table,
    int64_t ld_table, int columns, const int32_t* kv_len, const int32_t* parents, int64_t ld_parents,
    const int32_t* new_len, int top_k, int32_t* sel, void* O, const int64_t o_str[3], float scale, void* workspace_,
    size_t ws_bytes, void* stream) {
    const char* who = "ythip_paged_attn_sparse";
    PagedArgs a;
    bool done;
    const Call c = {dtype, B, Hq, Hkv, T, d, Q, q_str, Kn, kn_str, Vn, vn_str, Kp, Vp, pool_str, pages, page,
                    table, ld_table, columns, kv_len, parents, ld_parents, new_len, O, o_str, scale};
    const int st = prepare(who, c, a, done);
    if (st || done) return st;
    if ((int64_t)Hkv * T > 65535) return fail(YTHIP_EUNSUPPORTED, "%s: %d tokens of %d KV heads (at most 65535)", who, T, Hkv);
    if (top_k < 1 || top_k > 4096) return fail(YTHIP_EINVAL, "%s: top_k %d (1 to 4096)", who, top_k);
    if (!sel || !sums_str || (pages > 0 && !sums)) return fail(YTHIP_EINVAL, "%s: sel or sums is NULL", who);
    if (const int e = check_workspace(who, workspace(dtype, B, Hq, Hkv, T, d, columns, page, top_k), workspace_, ws_bytes)) return e;
    a.sel = sel, a.top_k = top_k, a.sums = sums, a.ss[0] = sums_str[0], a.ss[1] = sums_str[1];
    return run<true>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
}

}  // extern "C"
