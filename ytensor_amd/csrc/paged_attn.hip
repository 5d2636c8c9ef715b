// paged_attn.hip — attention of new tokens over a paged KV cache (include/ythip.h,
// ythip_paged_attn) and over the pages that a score selects (ythip_paged_attn_sparse).

#include <algorithm>
#include <climits>
#include <cmath>

#include "paged.hpp"

namespace ythip {
namespace {

// What the DMA reads in place of rows that are not in use.
static __device__ const u32x4 zeros[1] = {{0u, 0u, 0u, 0u}};

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
// With a window (WIN) the tiles that no query sees are left out of the cut and of the loop (seen_rows, window_of); those that
//   some queries see whole and others not are taken as tiles of new tokens are, by bits.
template <class T, int D, int QT, int WR, bool SPARSE, bool WIN>
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
    Seen seen;
    if constexpr (SPARSE) {
        sel = a.sel + (((int64_t)b * a.Hkv + h) * a.T + t_one) * a.top_k;
        nsel = min(a.top_k, (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift));
        nct = (int)((((int64_t)nsel << a.shift) + KT - 1) / KT);
        lim = t_one + 1;
    } else if constexpr (WIN) {
        seen = seen_rows(a, len, KT);
        nct = seen.tiles;
    } else {
        nct = (len + KT - 1) / KT;
    }
    auto row_of = [&](int ti) { return WIN ? seen.row(ti, KT) : ti * KT; };
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
    Window win;
    if constexpr (WIN) win = window_of(a, seen, len, c0, c1, a.parents != nullptr ? 0 : t_first, t_last, KT);
    const int nst = ((WIN ? win.count() : max(c1 - c0, 0)) + S::WK - 1) / S::WK;

    // for the walks, where the chunk holds new tokens (or their places count)
    const bool walk = a.parents != nullptr && (WIN || c1 > nct);
    if (walk) {
        for (int u = tid; u < tn; u += 256) {
            const int p = a.parents[b * a.ld_par + u];
            s_up[u] = (int16_t)(p >= 0 && p < u ? p : -1);
        }
        __syncthreads();
    }

    // this lane's query rows
    int tok[QT], cur[QT];
    int deep[QT], up[QT], lo[QT];  // with a window: how far behind the cache, the steps walked, the first row seen
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
        if constexpr (WIN) {
            deep[qt] = tok[qt];
            if (walk) {
                deep[qt] = -1;
                for (int u = tok[qt]; u >= 0; u = s_up[u]) ++deep[qt];
            }
            up[qt] = 0;
            lo[qt] = (int)max((int64_t)len + deep[qt] + 1 - a.window, (int64_t)0);
        }
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

    auto tile_at = [&](int s) { return WIN ? win.at(s * S::WK + wk) : c1 - 1 - (s * S::WK + wk); };
    // The pages of stage s, looked up ahead: the table's columns, then the ids in the pool.
    int col[S::KG], id[S::KG];
    auto columns = [&](int s) {
        const int row = row_of(tile_at(s));
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
                const int off = (row_of(ti) + 16 * i) & ((1 << a.shift) - 1);
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
                        const bool in = !WIN || up[qt] < a.window || deep[qt] - up[qt] < a.sinks - len;
                        if (in && cur[qt] < u0 + KT) see[qt] |= 1ull << (cur[qt] - u0);
                        cur[qt] = s_up[cur[qt]];
                        if constexpr (WIN) ++up[qt];
                    }
                } else if (tok[qt] >= u0) {
                    see[qt] = tok[qt] - u0 >= 63 ? ~0ull : (2ull << (tok[qt] - u0)) - 1;
                    if constexpr (WIN) see[qt] &= from_bit((int64_t)tok[qt] + 1 - a.window - u0) | ~from_bit((int64_t)a.sinks - len - u0);
                }
                any = any || see[qt] != 0;
                paths = paths || see[qt] != (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
            }
            if (__ballot(any) == 0) return;
            paths = __ballot(paths) != 0;
        } else if (WIN && NEW) {
            const int j0 = row_of(ti);
            bool any = false;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                see[qt] = from_bit(lo[qt] - j0) | ~from_bit(a.sinks - j0);
                const uint64_t here = see[qt] & (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
                any = any || here != 0;
                paths = paths || here != (KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1);
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
    auto step = [&](int s, auto issue_new, auto with_new) {
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
        next = s + 2 < nst ? issue(s + 2, issue_new) : 0;
    };
    // stages with new tokens, then those of cached rows alone: a loop of its own, that holds none of
    // the paths' state in registers
    // (with a window and no tree, new tokens before the first query's are as cached rows are)
    const int own = WIN && a.parents == nullptr && a.sinks <= len ? (t_first + 1) / KT : 0;
    const int s_new = WIN ? (max(win.high - max(win.low, nct + own), 0) + max(win.sink_end - max(c0, nct), 0) + S::WK - 1) / S::WK
                          : (max(c1 - max(c0, nct), 0) + S::WK - 1) / S::WK;
    const int s_whole = WIN ? max(s_new, max(win.high - max(win.low, win.clean), 0) / S::WK) : nst;
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
    for (int s = 0; s < s_new; ++s) step(s, std::true_type{}, std::true_type{});
    for (int s = s_new; s < s_whole; ++s) step(s, std::bool_constant<WIN>{}, std::false_type{});
    if constexpr (WIN)
        for (int s = s_whole; s < nst; ++s) step(s, std::true_type{}, std::true_type{});
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

// How a call is cut (plan_q4 in paged_q4.hip: for 4-bit pages).
Plan plan_of(int dtype, int B, int Hkv, int G, int T, int d, int columns, int page, int top_k, int window, int sinks) {
    const int rows = top_k > 0 ? G : (int)std::min<int64_t>((int64_t)T * G, 1 << 20);
    Plan p;
    // 16 rows or 32 leave the keys to the four waves; more share each staged tile between
    // two or four of them
    p.qt = rows <= 16 ? 1 : 2;
    p.wr = rows <= 32 || top_k > 0 ? 1 : rows <= 64 ? 2 : 4;
    p.kt = 16 * p.wr;
    const int64_t all_rows = top_k > 0 ? G : (int64_t)T * G;
    // a window leaves a row tile few keys: half the rows a workgroup where that fills the second place of the CUs
    // (float32, d 64, 1024 tokens, window 256: 62 -> 25.7 us; 4 chunks of 512 after 4096 rows, window 4096: 196 -> 135)
    const bool windowed = window > 0 && p.wr == 4;
    if (windowed && (int64_t)B * Hkv * ((all_rows + 127) / 128) < SLOTS && (int64_t)B * Hkv * ((all_rows + 63) / 64) >= SLOTS / 2)
        p.wr = 2, p.kt = 32;
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
    int64_t seq_rows = (int64_t)std::min(top_k > 0 ? top_k : columns, columns) * page;
    if (window > 0) seq_rows = std::min(seq_rows, (int64_t)window + sinks + 2 * p.kt);  // (a tile more at either end)
    const int64_t tiles = (seq_rows + p.kt - 1) / p.kt + new_tiles, most = (tiles + p.stage - 1) / p.stage;
    int64_t part_items = 0;
    if (windowed && B * per >= SLOTS / 2) {
        // Each row tile sees tiles of its own: ranges of all that one of them sees would leave most workgroups few (4 chunks
        // of 512, window 1024 51 us, cut into ranges 72; 16 of 128, window 4096 148 and 217). That takes items of about one
        // length: a window that is long beside most of the sequences leaves one of them nearly all of the work (chunks of
        // 512, window 4096: over 4 times 4096 rows 154 us either way, over 4096 and three times 600 126 us, cut 82; window
        // 16384 over 16384 and three times 600 442 and 158).
        p.target = 0;
        p.items = B;
    } else if (top_k > 0) {
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

template <class T, int D, int QT, int WR, bool SPARSE, bool WIN>
int launch(const PagedArgs& a, const Plan& p, hipStream_t s) {
    const int64_t groups = (p.items * a.Hkv + 7) / 8 * 8;
    using S = Shape<T, D, QT, WR>;
    paged_attn_kernel<T, D, QT, WR, SPARSE, WIN><<<(int)(groups * p.row_tiles), 256, 0, s>>>(a);
    if (p.part_bytes > 0) merge_partials<T, D, SPARSE>(a, S::KT, s);
    return status_of(hipGetLastError());
}
template <class T, int D, bool SPARSE, bool WIN>
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
    if (p.qt == 1) return launch<T, D, 1, 1, SPARSE, WIN>(a, p, s);
    if constexpr (!SPARSE) {
        if (p.wr == 2) return launch<T, D, 2, 2, SPARSE, WIN>(a, p, s);
        if (p.wr == 4) return launch<T, D, 2, 4, SPARSE, WIN>(a, p, s);
    }
    return launch<T, D, 2, 1, SPARSE, WIN>(a, p, s);
}
template <bool SPARSE, bool WIN>
int run(int dtype, int d, PagedArgs& a, void* ws, hipStream_t s) {
    const Plan p = plan_of(dtype, a.B, a.Hkv, a.G, a.T, d, a.columns, 1 << a.shift, SPARSE ? a.top_k : 0, a.window, a.sinks);
    if (!launchable((p.items * a.Hkv + 8) * p.row_tiles, 256))
        return fail(YTHIP_EUNSUPPORTED, "paged attention: %lld workgroups (2^24 - 1 at most)", (long long)(p.items * a.Hkv * p.row_tiles));
    a.target = p.target, a.stage = p.stage, a.items = (int)p.items, a.row_tiles = p.row_tiles, a.even = p.even, a.short_run = p.short_run;
    char* w = static_cast<char*>(ws);
    a.rank = reinterpret_cast<uint64_t*>(w);
    a.part = reinterpret_cast<float*>(w + p.rank_bytes);
    a.part_ml = reinterpret_cast<float*>(w + p.rank_bytes + p.part_bytes);
    if (dtype == YTHIP_F32) return d == 64 ? run_typed<F32, 64, SPARSE, WIN>(a, p, s) : run_typed<F32, 128, SPARSE, WIN>(a, p, s);
    if (dtype == YTHIP_F16) return d == 64 ? run_typed<F16, 64, SPARSE, WIN>(a, p, s) : run_typed<F16, 128, SPARSE, WIN>(a, p, s);
    return d == 64 ? run_typed<BF16, 64, SPARSE, WIN>(a, p, s) : run_typed<BF16, 128, SPARSE, WIN>(a, p, s);
}

size_t workspace(int dtype, int B, int Hq, int Hkv, int T, int d, int columns, int page, int top_k, int window = 0, int sinks = 0) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || d <= 0 || columns < 0 || page <= 0 || top_k < 0 || Hq % Hkv != 0 || window < 0 || sinks < 0) return 0;
    trim_window(T, columns, page, window, sinks);
    return plan_of(dtype, B, Hkv, Hq / Hkv, T, d, columns, page, top_k, window, sinks).bytes();
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
    return run<false, false>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
}

__attribute__((visibility("default"))) size_t ythip_paged_attn_window_workspace_size(int dtype, int B, int Hq, int Hkv,
                                                                                     int T, int d, int columns,
                                                                                     int page, int window, int sinks) {
    return workspace(dtype, B, Hq, Hkv, T, d, columns, page, 0, window, sinks);
}

__attribute__((visibility("default"))) int ythip_paged_attn_window(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[3], int pages, int page, const int32_t* table, int64_t ld_table, int columns,
    const int32_t* kv_len, const int32_t* parents, int64_t ld_parents, const int32_t* new_len, int window, int sinks,
    void* O, const int64_t o_str[3], float scale, void* workspace_, size_t ws_bytes, void* stream) {
    const char* who = "ythip_paged_attn_window";
    PagedArgs a;
    bool done;
    const Call c = {dtype, B, Hq, Hkv, T, d, Q, q_str, Kn, kn_str, Vn, vn_str, Kp, Vp, pool_str, pages, page,
                    table, ld_table, columns, kv_len, parents, ld_parents, new_len, O, o_str, scale};
    if (const int e = check_window(who, window, sinks)) return e;
    const int st = prepare(who, c, a, done);
    if (st || done) return st;
    if (const int e = check_workspace(who, workspace(dtype, B, Hq, Hkv, T, d, columns, page, 0, window, sinks), workspace_, ws_bytes)) return e;
    trim_window(T, columns, page, window, sinks);
    a.window = window, a.sinks = sinks;
    if (window == 0) return run<false, false>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
    return run<false, true>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
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
    return run<true, false>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
}

}  // extern "C"
