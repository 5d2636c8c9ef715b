// paged_attn.hip — attention of new tokens over a paged KV cache (include/ythip.h,
// ythip_paged_attn) and over the pages that a score selects (ythip_paged_attn_sparse).

#include <algorithm>
#include <climits>

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
    double* score;  // sparse: [B][Hkv][T][columns]
    int target, min_chunk, items, row_tiles;  // the cut: items aimed at (sparse: of a token), tiles an item has at least
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

__device__ __forceinline__ int64_t tiles_of(const PagedArgs& a, int len, int tn, int kt) {
    return ((int64_t)len + kt - 1) / kt + (a.Kn != nullptr ? (tn + kt - 1) / kt : 0);
}

// The cut of the batch: sequence b's tiles (KT cached rows or new tokens each) are dealt in
// chunks of the same size to ceil(tiles / chunk) workgroup items (one for none), so that a
// ragged batch gives every workgroup the same work; the chunk is what makes about
// a.target items of all the batch's tiles. Every wave works it out for itself from the
// lengths (one sequence a lane): `first` and `count` of the items of sequence b when `item`
// is negative, else b, its first item and count for that item (b = -1: past the last).
struct Cut {
    int b, first, count, chunk;
};
__device__ __forceinline__ Cut cut_of(const PagedArgs& a, int kt, int item, int b) {
    const int lane = threadIdx.x & 63;
    auto tiles = [&](int i) { return i < a.B ? tiles_of(a, rows_in_use(a, i), new_rows(a, i), kt) : 0; };
    int64_t total = 0, n0 = tiles(lane);
    for (int base = 0; base < a.B; base += 64) {
        int64_t n = base == 0 ? n0 : tiles(base + lane);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) n += __shfl_xor(n, off, 64);
        total += n;
    }
    const int64_t even = (total + a.target - 1) / a.target;
    Cut c;
    c.chunk = __builtin_amdgcn_readfirstlane((int)(even < a.min_chunk ? a.min_chunk : even));
    int before = 0;
    for (int base = 0; base < a.B; base += 64) {
        const int64_t n = base == 0 ? n0 : tiles(base + lane);
        const int mine = base + lane < a.B ? max((int)((n + c.chunk - 1) / c.chunk), 1) : 0;
        int inc = mine;
#pragma unroll
        for (int off = 1; off < 64; off <<= 1) {
            const int x = __shfl_up(inc, off, 64);
            if (lane >= off) inc += x;
        }
        const int all = __shfl(inc, 63, 64);
        int at = -1;
        if (item >= 0) {
            if (item < before + all) at = __popcll(__ballot(before + inc <= item));
        } else if (b < base + 64) {
            at = b - base;
        }
        if (at >= 0) {
            c.b = __builtin_amdgcn_readfirstlane(base + at);
            c.count = __builtin_amdgcn_readfirstlane(__shfl(mine, at, 64));
            c.first = __builtin_amdgcn_readfirstlane(before + __shfl(inc - mine, at, 64));
            return c;
        }
        before += all;
    }
    c.b = -1, c.first = before, c.count = 0;
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

__device__ __forceinline__ const char* uniform(const char* p) {
    const uint64_t v = (uint64_t)(uintptr_t)p;
    const uint32_t lo = __builtin_amdgcn_readfirstlane((uint32_t)v), hi = __builtin_amdgcn_readfirstlane((uint32_t)(v >> 32));
    return reinterpret_cast<const char*>((uintptr_t)((uint64_t)hi << 32 | lo));
}

__device__ __forceinline__ void wg_barrier() { asm volatile("s_barrier" ::: "memory"); }

template <class T, int D, int QT, int WR, int KT>
struct Shape {
    static constexpr int ES = sizeof(typename T::raw), ROWB = D * ES, CH = ROWB / 16;
    static constexpr int RPI = 1024 / ROWB;  // rows of one DMA instruction
    static constexpr int IPG = 16 / RPI;     // instructions of 16 rows
    static constexpr int WK = 4 / WR;        // key groups of the workgroup
    static constexpr int KG = KT / 16, GPW = KG / WR, NI = GPW * IPG;
    static constexpr int TILE = KT * CH, STG = WK * TILE;  // in 16-byte chunks
    static constexpr int KS = CH / 4, DT = D / 16, RW = 16 * QT * WR;
    static constexpr int OLD = D + 4;  // floats of a row of O in LDS: 16 rows fall in different banks
    static constexpr int EPI = WK == 1 ? 0 : (WK * RW * (OLD + 2) * 4 + 15) / 16;  // the epilogue's use of the stages
    static constexpr int LDS = 4 * STG > EPI ? 4 * STG : EPI;
    static_assert(KG % WR == 0 && (ES == 4 || KT % 32 == 0), "tile");
};

// One workgroup: RW = 16 QT WR query rows of one KV head (row = token * G + head of the group)
// over a chunk of its sequence's tiles. Its four waves are WR row groups x WK key groups: few
// rows share out the keys (WR = 1: each wave streams its own tiles, no barrier in the loop),
// many rows share the staged tile.
//   S^T = K . Q^T and O^T = V^T . P^T on the matrix cores, lane l holding query l % 16: the
//   softmax statistics are per lane, joined over the four lanes of a query by row swaps.
//   K and V reach LDS by DMA (16 rows of one page an address; a stage ahead), K chunks
//   XOR-swizzled by key, V 32-byte blocks likewise and read transposed.
//   Tiles run from the last to the first: new tokens, whose path is walked down from each
//   query's token once, then cached rows.
// Numerics: scores, maxima, sums and O in fp32; p is rounded to the inputs' 16-bit type for
// the second product (2^-9 of each weight in bf16, as the rounding of O).
template <class T, int D, int QT, int WR, int KT, bool SPARSE>
__global__ __launch_bounds__(256) void paged_attn_kernel(PagedArgs a) {
    using S = Shape<T, D, QT, WR, KT>;
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
    const int h = gi % a.Hkv, item = gi / a.Hkv;

    int b, split, nsplit, chunk, t_one = 0;
    if constexpr (SPARSE) {
        split = item % a.target;
        t_one = item / a.target % a.T;
        b = item / a.target / a.T;
    } else {
        const Cut c = cut_of(a, KT, item, 0);
        if (c.b < 0) return;
        b = c.b, split = item - c.first, nsplit = c.count, chunk = c.chunk;
    }
    const int len = __builtin_amdgcn_readfirstlane(rows_in_use(a, b)), tn = __builtin_amdgcn_readfirstlane(new_rows(a, b));
    const int R = SPARSE ? a.G : a.T * a.G;
    const int r0 = rt * S::RW;
    const int t_first = SPARSE ? t_one : r0 / a.G, t_last = SPARSE ? t_one : min((min(R, r0 + S::RW) - 1) / a.G, tn - 1);
    if (t_first >= tn) return;
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
    if constexpr (SPARSE) {
        chunk = max((nt + a.target - 1) / a.target, a.min_chunk);
        nsplit = max((nt + chunk - 1) / chunk, 1);
        if (split >= nsplit) return;
    }
    const int c0 = split * chunk, c1 = min(nt, c0 + chunk);
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
    bool real[QT];
    u32x4 qf[QT][S::KS];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = r0 + wr * 16 * QT + qt * 16 + l16;
        const int t = SPARSE ? t_one : r / a.G, gh = SPARSE ? r : r - t * a.G;
        real[qt] = r < R && t < tn;
        tok[qt] = real[qt] ? t : -1;
        cur[qt] = tok[qt];
        const raw* qp = static_cast<const raw*>(a.Q) + b * a.qs[0] + (int64_t)(h * a.G + gh) * a.qs[1] + t * a.qs[2];
#pragma unroll
        for (int ks = 0; ks < S::KS; ++ks) {
            qf[qt][ks] = u32x4{0u, 0u, 0u, 0u};
            if (real[qt]) qf[qt][ks] = *reinterpret_cast<const u32x4*>(qp + (ks * 4 + g) * (16 / S::ES));
        }
    }

    // DMA: lane -> (row of the instruction, chunk), the chunk swizzled by the row in its 16
    uint32_t kof[S::IPG], vof[S::IPG], kch[S::IPG], vch[S::IPG];
    const int pool_row = (int)a.ps[2] * S::ES;
#pragma unroll
    for (int i = 0; i < S::IPG; ++i) {
        const int row = i * S::RPI + lane / S::CH, ps = lane % S::CH;
        kch[i] = (ps ^ (row & KMASK)) * 16;
        vch[i] = F ? (ps ^ (((row >> 2) & 3) << 2)) * 16 : (((ps >> 1) ^ (row & BMASK)) * 32 + (ps & 1) * 16);
        kof[i] = row * pool_row + kch[i];
        vof[i] = row * pool_row + vch[i];
    }
    const uint32_t lds0 = __builtin_amdgcn_readfirstlane((uint32_t)(uintptr_t)smem);
    const char *Kp = static_cast<const char*>(a.Kp) + h * a.ps[1] * S::ES, *Vp = static_cast<const char*>(a.Vp) + h * a.ps[1] * S::ES;
    const char* Kn = static_cast<const char*>(a.Kn) + (b * a.kns[0] + h * a.kns[1]) * S::ES;
    const char* Vn = static_cast<const char*>(a.Vn) + (b * a.vns[0] + h * a.vns[1]) * S::ES;

    // Stage s: the rows in use of each 16 (5 bits a group; 0: nothing was staged, the tile is
    // skipped) and this wave's share of the DMA. Rows that are not in use read zeros.
    auto tile_at = [&](int s) { return c1 - 1 - (s * S::WK + wk); };
    auto issue = [&](int s) {
        const int ti = tile_at(s);
        uint32_t pack = 0;
        if (ti < c0) return pack;
        const char *kb[S::KG], *vb[S::KG];
        const bool cached = ti < nct;
#pragma unroll
        for (int i = 0; i < S::KG; ++i) {
            int n;
            if (cached) {
                const int row = ti * KT + 16 * i, slot = row >> a.shift, off = row & ((1 << a.shift) - 1);
                int lp = slot;
                if constexpr (SPARSE) lp = slot < nsel ? scalar_word(sel + slot) : -1;
                n = lp < 0 ? 0 : min(max(len - (lp << a.shift) - off, 0), 16);
                const int p = n > 0 ? scalar_word(table + lp) : -1;
                if ((uint32_t)p >= (uint32_t)a.pages) n = 0;
                const int64_t at = (p * a.ps[0] + off * a.ps[2]) * S::ES;
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
            if (cached && n == 16) {
                k = uniform(k), v = uniform(v);
#pragma unroll
                for (int e = 0; e < S::IPG; ++e) {
                    dma16_soff(k, kof[e], lk + e * 1024);
                    dma16_soff(v, vof[e], lv + e * 1024);
                }
            } else {
                const int64_t kr = (cached ? a.ps[2] : a.kns[2]) * S::ES, vr = (cached ? a.ps[2] : a.vns[2]) * S::ES;
#pragma unroll
                for (int e = 0; e < S::IPG; ++e) {
                    const int row = e * S::RPI + lane / S::CH;
                    const char* zero = reinterpret_cast<const char*>(zeros);
                    const char* ka = row < n ? k + row * kr + kch[e] : zero;
                    const char* va = row < n ? v + row * vr + vch[e] : zero;
                    dma16_async(ka, smem + (lk - lds0) / 16 + e * 64);
                    dma16_async(va, smem + (lv - lds0) / 16 + e * 64);
                }
            }
        }
        return pack;
    };

    float m[QT], l[QT];
    f32x4 o[QT][S::DT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -INFINITY;
        l[qt] = 0.f;
#pragma unroll
        for (int t = 0; t < S::DT; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // acc += V^T . P^T over the tile's keys, or those of `keep` alone (the others' V taken as 0)
    auto pv = [&](const u32x4* cV, const f32x4 (&p)[QT][S::KG], f32x4 (&acc)[QT][S::DT], auto some, uint64_t keep) {
        constexpr bool SOME = decltype(some)::value;
        if constexpr (F) {
            const float* V = reinterpret_cast<const float*>(cV);
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt)
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int key = kt * 16 + 4 * g + j;
#pragma unroll
                    for (int t = 0; t < S::DT; ++t) {
                        const int c = t * 4 + (l16 >> 2);
                        float v = V[key * D + ((c ^ (((key >> 2) & 3) << 2)) << 2) + (l16 & 3)];
                        if (SOME) v = (keep >> key & 1) ? v : 0.f;
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt)
                            acc[qt][t] = __builtin_amdgcn_mfma_f32_16x16x4f32(v, p[qt][kt][j], acc[qt][t], 0, 0, 0);
                    }
                }
        } else {
#pragma unroll
            for (int kk = 0; kk < S::KG / 2; ++kk) {
                u32x4 pk[QT], km;
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    pk[qt] = u32x4{pack2<T>(p[qt][2 * kk][0], p[qt][2 * kk][1]), pack2<T>(p[qt][2 * kk][2], p[qt][2 * kk][3]),
                                   pack2<T>(p[qt][2 * kk + 1][0], p[qt][2 * kk + 1][1]), pack2<T>(p[qt][2 * kk + 1][2], p[qt][2 * kk + 1][3])};
                if (SOME) {
#pragma unroll
                    for (int e = 0; e < 4; ++e) {
                        const int key = (2 * kk + (e >> 1)) * 16 + 4 * g + (e & 1) * 2;
                        km[e] = (keep >> key & 1 ? 0xffffu : 0u) | (keep >> (key + 1) & 1 ? 0xffff0000u : 0u);
                    }
                }
#pragma unroll
                for (int t = 0; t < S::DT; ++t) {
                    u32x4 vf;
#pragma unroll
                    for (int hh = 0; hh < 2; ++hh) {
                        const int key = (2 * kk + hh) * 16 + g * 4 + (l16 >> 2);
                        const u32x2 w = lds_read_tr16(cV, key * S::ROWB + ((t ^ (key & BMASK)) << 5) + 8 * (l16 & 3));
                        vf[2 * hh] = w[0];
                        vf[2 * hh + 1] = w[1];
                    }
                    if (SOME) vf &= km;
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) acc[qt][t] = mfma_chunk(T{}, vf, pk[qt], acc[qt][t]);
                }
            }
        }
    };

    auto compute = [&](int s, uint32_t pack) {
        const int ti = tile_at(s);
        const u32x4* cK = smem + (s & 1) * 2 * S::STG + wk * S::TILE;
        const u32x4* cV = cK + S::STG;
        const bool cached = ti < nct;
        uint64_t see[QT];
        if (!cached) {
            // the new tokens of this tile on each query's path
            const int u0 = (ti - nct) * KT;
            bool any = false;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                see[qt] = 0;
                if (walk) {
                    while (cur[qt] >= u0) {
                        if (cur[qt] < u0 + KT) see[qt] |= 1ull << (cur[qt] - u0);
                        cur[qt] = s_up[cur[qt]];
                    }
                } else if (tok[qt] >= u0) {
                    see[qt] = tok[qt] - u0 >= 63 ? ~0ull : (2ull << (tok[qt] - u0)) - 1;
                }
                any = any || see[qt] != 0;
            }
            if (__ballot(any) == 0) return;
        }
        f32x4 p[QT][S::KG];
#pragma unroll
        for (int kt = 0; kt < S::KG; ++kt) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt][kt] = f32x4{0.f, 0.f, 0.f, 0.f};
            const int key = kt * 16 + l16;
#pragma unroll
            for (int ks = 0; ks < S::KS; ++ks) {
                const u32x4 kf = cK[key * S::CH + ((ks * 4 + g) ^ (key & KMASK))];
#pragma unroll
                for (int qt = 0; qt < QT; ++qt) p[qt][kt] = mfma_chunk(T{}, kf, qf[qt][ks], p[qt][kt]);
            }
        }
        constexpr uint32_t FULL = S::KG == 1 ? 16u : S::KG == 2 ? 16u | 16u << 5 : 16u | 16u << 5 | 16u << 10 | 16u << 15;
        const bool whole = cached && pack == FULL;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            float mx = -INFINITY;
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    float x = p[qt][kt][r] * a.scale_log2;
                    if (!whole) {
                        const int key = kt * 16 + 4 * g + r;
                        bool vis = 4 * g + r < (int)((pack >> (5 * kt)) & 31);
                        if (!cached) vis = vis && (see[qt] >> key & 1);
                        x = vis ? x : -INFINITY;
                    }
                    p[qt][kt][r] = x;
                    mx = __builtin_elementwise_maximum(mx, x);
                }
            const float top = __builtin_elementwise_maximum(m[qt], max_across_rows(mx));
            const float ref = top == -INFINITY ? 0.f : top;  // nothing seen yet: every weight is 0
            const float corr = __builtin_amdgcn_exp2f(m[qt] - ref);
            m[qt] = top;
            float sum = 0.f;
#pragma unroll
            for (int kt = 0; kt < S::KG; ++kt)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    p[qt][kt][r] = __builtin_amdgcn_exp2f(p[qt][kt][r] - ref);
                    sum += p[qt][kt][r];
                }
            l[qt] = l[qt] * corr + sum;
            if (__ballot(corr != 1.0f) != 0) {
#pragma unroll
                for (int t = 0; t < S::DT; ++t) o[qt][t] *= corr;
            }
        }
        uint64_t odd = 0;
        if (!cached) {
            // 0 . V is NaN for a V that is not finite: such rows of the tile are left out and added
            // for the queries alone that see them
            constexpr uint32_t EXP = std::is_same_v<T, BF16> ? 0x7f80u : 0x7c00u;
#pragma unroll
            for (int i = 0; i < S::TILE / 64; ++i) {
                const u32x4 v = cV[i * 64 + lane];
                bool bad = false;
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    if (F) bad = bad || (v[e] & 0x7f800000u) == 0x7f800000u;
                    else bad = bad || (v[e] & EXP) == EXP || (v[e] >> 16 & EXP) == EXP;
                }
                const uint64_t w = __ballot(bad);
                if (w != 0) {
#pragma unroll
                    for (int r = 0; r < S::RPI; ++r)
                        if (w >> (r * S::CH) & ((S::CH == 64 ? 0ull : 1ull << S::CH) - 1)) odd |= 1ull << (i * S::RPI + r);
                }
            }
        }
        if (odd == 0) {
            pv(cV, p, o, std::false_type{}, 0);
            return;
        }
        pv(cV, p, o, std::true_type{}, ~odd);
        for (uint64_t left = odd; left != 0; left &= left - 1) {
            const int u = __builtin_ctzll(left);
            f32x4 one[QT][S::DT];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                for (int t = 0; t < S::DT; ++t) one[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
            pv(cV, p, one, std::true_type{}, 1ull << u);
#pragma unroll
            for (int qt = 0; qt < QT; ++qt)
#pragma unroll
                for (int t = 0; t < S::DT; ++t)
                    if (see[qt] >> u & 1) o[qt][t] += one[qt][t];
        }
    };

    uint32_t here = nst > 0 ? issue(0) : 0, next = nst > 1 ? issue(1) : 0;
    for (int s = 0; s < nst; ++s) {
        if (next != 0) wait_vmcnt<2 * S::NI>();  // stage s has landed, s + 1 is in flight
        else wait_vmcnt<0>();
        if constexpr (WR > 1) wg_barrier();
        else asm volatile("" ::: "memory");
        if (here != 0) compute(s, here);
        if constexpr (WR > 1) wg_barrier();
        else asm volatile("" ::: "memory");
        here = next;
        next = s + 2 < nst ? issue(s + 2) : 0;
    }
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        l[qt] += __shfl_xor(l[qt], 16, 64);
        l[qt] += __shfl_xor(l[qt], 32, 64);
    }

    // the place of row r's result: O itself, or this item's partial
    auto store4 = [&](int r, int d, f32x4 v, float M, float L) {
        const int t = SPARSE ? t_one : r / a.G, gh = SPARSE ? r : r - t * a.G;
        if (r >= R || t >= tn) return;
        if (nsplit == 1) {
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
            for (int t = 0; t < S::DT; ++t) store4(r0 + wr * 16 * QT + qt * 16 + l16, 16 * t + 4 * g, o[qt][t], m[qt], l[qt]);
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
                sm[2 * row + 1] = l[qt];
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

// Joins the partials of a sequence that several items worked on: a wave per (token, head), in
// the order of the items.
template <class T, int D, bool SPARSE>
__global__ __launch_bounds__(256) void paged_merge_kernel(PagedArgs a, int kt) {
    constexpr int E = D / 64;
    const int lane = threadIdx.x & 63;
    const int r = blockIdx.x * 4 + __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), h = blockIdx.y, b = blockIdx.z;
    const int tn = new_rows(a, b);
    const int t = r / a.G, gh = r - t * a.G;
    if (t >= tn) return;
    int64_t first, step;
    int count;
    if constexpr (SPARSE) {
        const int len = rows_in_use(a, b);
        const int nsel = min(a.top_k, (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift));
        const int nt = (int)((((int64_t)nsel << a.shift) + kt - 1) / kt) + (a.Kn != nullptr ? (t + kt) / kt : 0);
        const int chunk = max((nt + a.target - 1) / a.target, a.min_chunk);
        count = max((nt + chunk - 1) / chunk, 1);
        first = (((int64_t)(b * a.T + t) * a.target) * a.Hkv + h) * a.G + gh;
        step = (int64_t)a.Hkv * a.G;
    } else {
        const Cut c = cut_of(a, kt, -1, b);
        count = c.count;
        first = ((int64_t)c.first * a.Hkv + h) * a.T * a.G + r;
        step = (int64_t)a.Hkv * a.T * a.G;
    }
    if (count == 1) return;
    float M = -INFINITY, L = 0.f, acc[E];
    for (int e = 0; e < E; ++e) acc[e] = 0.f;
    for (int s = lane; s < count; s += 64) M = __builtin_elementwise_maximum(M, a.part_ml[2 * (first + s * step)]);
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) M = __builtin_elementwise_maximum(M, __shfl_xor(M, off, 64));
    const float ref = M == -INFINITY ? 0.f : M;
    for (int s0 = 0; s0 < count; s0 += 64) {
        const int64_t mine = first + (int64_t)min(s0 + lane, count - 1) * step;
        const float w = s0 + lane < count ? __builtin_amdgcn_exp2f(a.part_ml[2 * mine] - ref) : 0.f;
        const float lw = s0 + lane < count ? w * a.part_ml[2 * mine + 1] : 0.f;
        L += wave_sum(lw);
        const int n = min(count - s0, 64);
        const float* src = a.part + (first + (int64_t)s0 * step) * D + lane * E;
        for (int s = 0; s < n; s += 8) {
            float v[8][E];
#pragma unroll
            for (int u = 0; u < 8; ++u)
#pragma unroll
                for (int e = 0; e < E; ++e) v[u][e] = src[(int64_t)min(s + u, n - 1) * step * D + e];
#pragma unroll
            for (int u = 0; u < 8; ++u) {
                const float ws = s + u < n ? __shfl(w, s + u, 64) : 0.f;
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = s + u < n ? fmaf(ws, v[u][e], acc[e]) : acc[e];
            }
        }
    }
    const int64_t at = b * a.os[0] + (int64_t)(h * a.G + gh) * a.os[1] + t * a.os[2] + lane * E;
    for (int e = 0; e < E; ++e) store_from_f32<T>(a.O, at + e, M == -INFINITY ? 0.f : acc[e] / L);
}

// One workgroup per (token, KV head, sequence): every page's score, then the pages that
// fewer than top_k others beat.
template <class T, int D>
__global__ __launch_bounds__(256) void paged_select_simple(PagedArgs a) {
    __shared__ double s_q[D];
    const int t = blockIdx.x, h = blockIdx.y, b = blockIdx.z, tid = threadIdx.x;
    const int64_t row = ((int64_t)b * a.Hkv + h) * a.T + t;
    int32_t* sel = a.sel + row * a.top_k;
    const int len = rows_in_use(a, b), n = t < new_rows(a, b) ? (int)(((int64_t)len + (1 << a.shift) - 1) >> a.shift) : 0;
    if (tid < D) {
        double q = 0.0;
        for (int g = 0; g < a.G; ++g)
            q += (double)load_as_f32<T>(a.Q, b * a.qs[0] + (h * a.G + g) * a.qs[1] + t * a.qs[2] + tid);
        s_q[tid] = q;
    }
    __syncthreads();
    double* score = a.score + row * a.columns;
    for (int i = tid; i < n; i += 256) {
        const int p = a.table[b * a.ld_table + i];
        double s = 0.0;
        if (p >= 0 && p < a.pages)
            for (int e = 0; e < D; ++e) s = fma(s_q[e], (double)a.sums[p * a.ss[0] + h * a.ss[1] + e], s);
        else s = -INFINITY;
        if (s != s) s = -INFINITY;
        score[i] = s;
    }
    for (int i = tid; i < a.top_k; i += 256) sel[i] = -1;
    __threadfence_block();
    __syncthreads();
    for (int i = tid; i < n; i += 256) {
        const double s = score[i];
        int above = i < n - 1 ? 1 : 0;  // the last page
        for (int j = 0; j < n - 1 && i < n - 1; ++j) above += score[j] > s || (score[j] == s && j < i);
        if (above < a.top_k) sel[above] = i;
    }
    __threadfence_block();
    __syncthreads();
    if (tid == 0)  // ascending
        for (int i = 1; i < min(n, a.top_k); ++i) {
            const int v = sel[i];
            int j = i;
            for (; j > 0 && sel[j - 1] > v; --j) sel[j] = sel[j - 1];
            sel[j] = v;
        }
}

// How a call is cut. Both the size of the workspace and the launch come from this alone.
struct Plan {
    int qt, wr, kt;  // the workgroup's shape
    int target, min_chunk, row_tiles;
    int64_t items;
    size_t part_bytes, ml_bytes, score_bytes;
    size_t bytes() const { return part_bytes + ml_bytes + score_bytes; }
};
constexpr int CUS = 256;  // MI355X
Plan plan_of(int dtype, int B, int Hkv, int G, int T, int d, int columns, int page, int top_k) {
    const bool f32 = dtype == YTHIP_F32;
    const int rows = top_k > 0 ? G : (int)std::min<int64_t>((int64_t)T * G, 1 << 20);
    Plan p;
    // 16 rows or 32 leave the keys to the four waves; more share each staged tile between
    // two or four of them
    p.qt = rows <= 16 ? 1 : 2;
    p.wr = rows <= 32 || top_k > 0 ? 1 : rows <= 64 ? 2 : 4;
    p.kt = p.wr == 4 ? 64 : p.wr == 1 && f32 ? 16 : 32;
    const int64_t all_rows = top_k > 0 ? G : (int64_t)T * G;
    const int rw = 16 * p.qt * p.wr;
    p.row_tiles = (int)((all_rows + rw - 1) / rw);
    const int64_t per = (int64_t)Hkv * p.row_tiles;
    p.min_chunk = 4 / p.wr;
    const int64_t new_tiles = ((int64_t)T + p.kt - 1) / p.kt;
    if (top_k > 0) {
        const int64_t tiles = ((int64_t)std::min(top_k, columns) * page + p.kt - 1) / p.kt + new_tiles;
        const int64_t most = (tiles + p.min_chunk - 1) / p.min_chunk, want = (CUS + per * B * T - 1) / (per * B * T);
        p.target = (int)std::max<int64_t>(1, std::min(most, want));
        p.items = (int64_t)B * T * p.target;
    } else {
        const int64_t tiles = ((int64_t)columns * page + p.kt - 1) / p.kt + new_tiles;
        const int64_t most = (tiles + p.min_chunk - 1) / p.min_chunk;
        p.target = (int)std::max<int64_t>(1, CUS / per);
        p.items = std::min<int64_t>((int64_t)p.target + B, B * most);
    }
    const bool parts = top_k > 0 ? p.target > 1 : p.items > B;
    const int64_t part_rows = parts ? p.items * Hkv * all_rows : 0;
    p.part_bytes = (size_t)part_rows * d * sizeof(float);
    p.ml_bytes = ((size_t)part_rows * 2 * sizeof(float) + 15) / 16 * 16;
    p.score_bytes = top_k > 0 ? (size_t)B * Hkv * T * columns * sizeof(double) : 0;
    return p;
}

template <class T, int D, int QT, int WR, int KT, bool SPARSE>
int launch(const PagedArgs& a, const Plan& p, hipStream_t s) {
    const int64_t groups = (p.items * a.Hkv + 7) / 8 * 8;
    if (groups * p.row_tiles > INT_MAX) return fail(YTHIP_EUNSUPPORTED, "paged attention: %lld workgroups", (long long)(groups * p.row_tiles));
    paged_attn_kernel<T, D, QT, WR, KT, SPARSE><<<(int)(groups * p.row_tiles), 256, 0, s>>>(a);
    if (p.part_bytes > 0) paged_merge_kernel<T, D, SPARSE><<<dim3((a.T * a.G + 3) / 4, a.Hkv, a.B), 256, 0, s>>>(a, KT);
    return status_of(hipGetLastError());
}
template <class T, int D, bool SPARSE>
int run_typed(const PagedArgs& a, const Plan& p, hipStream_t s) {
    constexpr int K1 = std::is_same_v<T, F32> ? 16 : 32;
    if constexpr (SPARSE) paged_select_simple<T, D><<<dim3(a.T, a.Hkv, a.B), 256, 0, s>>>(a);
    if (p.qt == 1) return launch<T, D, 1, 1, K1, SPARSE>(a, p, s);
    if constexpr (!SPARSE) {
        if (p.wr == 2) return launch<T, D, 2, 2, 32, SPARSE>(a, p, s);
        if (p.wr == 4) return launch<T, D, 2, 4, 64, SPARSE>(a, p, s);
    }
    return launch<T, D, 2, 1, K1, SPARSE>(a, p, s);
}
template <bool SPARSE>
int run(int dtype, int d, PagedArgs& a, void* ws, hipStream_t s) {
    const Plan p = plan_of(dtype, a.B, a.Hkv, a.G, a.T, d, a.columns, 1 << a.shift, SPARSE ? a.top_k : 0);
    a.target = p.target, a.min_chunk = p.min_chunk, a.items = (int)p.items, a.row_tiles = p.row_tiles;
    char* w = static_cast<char*>(ws);
    a.score = reinterpret_cast<double*>(w);
    a.part = reinterpret_cast<float*>(w + p.score_bytes);
    a.part_ml = reinterpret_cast<float*>(w + p.score_bytes + p.part_bytes);
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
    if (c.columns > 65536 || (int64_t)c.columns * c.page > INT_MAX)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d columns of %d rows (at most 65536 columns, 2^31 - 1 rows)", who, c.columns, c.page);
    if (c.parents != nullptr && c.T > MAX_TREE) return fail(YTHIP_EUNSUPPORTED, "%s: a tree of %d tokens (at most %d)", who, c.T, MAX_TREE);
    if (!c.Q || !c.O || !c.kv_len || !c.q_str || !c.o_str || !c.pool_str) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if ((c.Kn == nullptr) != (c.Vn == nullptr) || (c.Kn && (!c.kn_str || !c.vn_str))) return fail(YTHIP_EINVAL, "%s: Kn and Vn go together, with their strides", who);
    if (c.columns > 0 && (!c.table || (c.pages > 0 && (!c.Kp || !c.Vp)))) return fail(YTHIP_EINVAL, "%s: table or a pool is NULL", who);
    if (c.ld_table < c.columns) return fail(YTHIP_EINVAL, "%s: a table row of %d entries at a stride of %lld", who, c.columns, (long long)c.ld_table);
    if (c.parents && c.ld_par < c.T) return fail(YTHIP_EINVAL, "%s: a parents row of %d entries at a stride of %lld", who, c.T, (long long)c.ld_par);
    const int es = c.dtype == YTHIP_F32 ? 4 : 2;
    int64_t all = (int64_t)(uintptr_t)c.Q | (int64_t)(uintptr_t)c.O | (int64_t)(uintptr_t)c.Kn | (int64_t)(uintptr_t)c.Vn |
                  (int64_t)(uintptr_t)c.Kp | (int64_t)(uintptr_t)c.Vp;
    for (int i = 0; i < 3; ++i) {
        all |= (c.q_str[i] | c.o_str[i] | c.pool_str[i]) * es;
        if (c.Kn) all |= (c.kn_str[i] | c.vn_str[i]) * es;
    }
    if ((all & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
    if (c.pool_str[2] < 0 || c.pool_str[2] >= 1 << 24) return fail(YTHIP_EUNSUPPORTED, "%s: pool rows at a stride of %lld (0 to 2^24 - 1)", who, (long long)c.pool_str[2]);
    a.B = c.B, a.Hq = c.Hq, a.Hkv = c.Hkv, a.G = c.Hq / c.Hkv, a.T = c.T, a.pages = c.pages, a.columns = c.columns;
    a.Q = c.Q, a.Kn = c.Kn, a.Vn = c.Vn, a.Kp = c.Kp, a.Vp = c.Vp;
    for (int i = 0; i < 3; ++i) {
        a.qs[i] = c.q_str[i], a.os[i] = c.o_str[i], a.ps[i] = c.pool_str[i];
        a.kns[i] = c.Kn ? c.kn_str[i] : 0, a.vns[i] = c.Kn ? c.vn_str[i] : 0;
    }
    a.table = c.table, a.kv_len = c.kv_len, a.parents = c.parents, a.new_len = c.new_len;
    a.ld_table = c.ld_table, a.ld_par = c.ld_par, a.O = c.O;
    a.scale_log2 = (c.scale == 0.f ? 1.0f / sqrtf((float)c.d) : c.scale) * 1.4426950408889634f;
    a.sel = nullptr, a.top_k = 0, a.sums = nullptr, a.score = nullptr;
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
    if (top_k < 1 || top_k > 4096) return fail(YTHIP_EINVAL, "%s: top_k %d (1 to 4096)", who, top_k);
    if (!sel || !sums_str || (pages > 0 && !sums)) return fail(YTHIP_EINVAL, "%s: sel or sums is NULL", who);
    if (const int e = check_workspace(who, workspace(dtype, B, Hq, Hkv, T, d, columns, page, top_k), workspace_, ws_bytes)) return e;
    a.sel = sel, a.top_k = top_k, a.sums = sums, a.ss[0] = sums_str[0], a.ss[1] = sums_str[1];
    return run<true>(dtype, d, a, workspace_, static_cast<hipStream_t>(stream));
}

}  // extern "C"
