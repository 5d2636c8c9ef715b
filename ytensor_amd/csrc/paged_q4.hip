// paged_q4.hip — the paged KV cache in 4 bits for gfx950 (include/ythip.h, "4-bit pages"): rows into it
// (ythip_cache_append_q4), its values (ythip_cache_unpack_q4) and attention over it (ythip_paged_attn_q4).
//
// A value is one of the eight magnitudes 0, 0.5, 1, 1.5, 2, 3, 4, 6 with a sign, times its group's 2^e (32 neighbouring
// channels of a row): gfx950 converts two of them at a time, scaled, in one instruction, and with a power of two as the
// scale they are exact in bfloat16, so that the matrix cores take them in that type whatever the queries' type is.

#include "paged.hpp"

namespace ythip {
namespace {

constexpr int E_MIN = -125;  // the scales' exponents: 0.5 2^E_MIN is the smallest normal number
template <class T> constexpr int e_max() { return std::is_same_v<T, F16> ? 13 : 125; }  // 6 2^e_max: within the type

// Bytes of a page and KV head: page codes rows, then the scales.
__host__ __device__ inline int64_t block_bytes(int page, int d) { return (int64_t)page * (d / 2 + d / 32); }
// Where channel group l16 (d / 16 channels) of row r lies in a V block; the 8 rows of r / 8 follow each other.
__device__ __forceinline__ int v_code(int r, int l16, int d) { return ((r >> 3) * 16 + l16) * (8 * (d / 32)) + (r & 7) * (d / 32); }
__device__ __forceinline__ int v_scale(int page, int r, int group, int d) { return page * (d / 2) + ((r >> 3) * (d / 32) + group) * 8 + (r & 7); }

// Two codes (byte SEL of w) times the scale.
template <int SEL>
__device__ __forceinline__ uint32_t to_bf16(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp4(w, scale, SEL));
#else
    return 0;
#endif
}
template <int SEL>
__device__ __forceinline__ f32x2 to_f32(uint32_t w, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_bit_cast(f32x2, __builtin_amdgcn_cvt_scalef32_pk_f32_fp4(w, scale, SEL));
#else
    return f32x2{0.f, 0.f};
#endif
}
// Two values over the scale as the codes nearest to them (of two as near the even one), into byte SEL.
template <int SEL>
__device__ __forceinline__ uint32_t to_codes(uint32_t w, float x, float y, float scale) {
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_cvt_scalef32_pk_fp4_f32(w, x, y, scale, SEL);
#else
    return w;
#endif
}
__device__ __forceinline__ float scale_of(uint32_t byte) { return __uint_as_float(byte << 23); }

// ---------------------------------------------------------------------------
// Rows into the pages
// ---------------------------------------------------------------------------

struct AppendQ4Args {
    int layers, B, Hkv, T, pages, shift, columns, runs;
    const char *Kn, *Vn;
    uint8_t *Kp, *Vp;
    int64_t ns[4];  // bytes
    int64_t ps[3];
    const int32_t *table, *kv_len, *count, *path;
    int64_t ld_table, ld_path;
    bool to;  // count: the lengths afterwards, not the new rows
    int32_t* status;
};

constexpr int APPEND_ROWS = 16;  // of a workgroup at a time

// The group's scale: the power of two 2^e by which its largest magnitude is in [3.5, 7], so that no value is further from
// the nearest code than half a step; NaN (and infinities) leave the group without a value, byte 255.
template <class T>
__device__ __forceinline__ uint32_t scale_byte(float top) {
    if (!(top < INFINITY)) return 255;
    int e = (int)(__float_as_uint(top) >> 23) - 127 - 2;
    e = max(e, E_MIN);
    // (at E_MIN a top is below 8 2^E_MIN, as with any e)
    if (top > 7.f * __uint_as_float((uint32_t)(e + 127) << 23)) ++e;
    return (uint32_t)(min(e, e_max<T>()) + 127);
}

// A thread has 8 channels of a row, four lanes a group; K and V of 16 rows a workgroup of 16 * D / 8 threads. Bound by the
// latency of the lengths, the table and the rows in turn for few rows, by their bytes for many.
template <class T, int D>
__global__ __launch_bounds__(APPEND_ROWS * D / 8) void cache_append_q4_kernel(AppendQ4Args a) {
    constexpr int LPR = D / 8;
    using raw = typename T::raw;
    int w = blockIdx.x;
    const int run = w % a.runs;
    w /= a.runs;
    const int h = w % a.Hkv;
    w /= a.Hkv;
    const int b = w % a.B, l = w / a.B;
    const int page = 1 << a.shift;
    const int len = a.kv_len[b], count = a.count != nullptr ? a.count[b] : a.T;
    const int64_t cap = (int64_t)a.columns << a.shift;
    const int64_t end = a.to ? count : (int64_t)len + min(count, a.T);  // rows in use afterwards
    const bool tells = a.to && l == 0 && h == 0;
    if (tells && run == 0 && threadIdx.x == 0 && end != len && (len < 0 || end < len || end - len > a.T || end > cap) && a.status != nullptr)
        atomicOr(a.status, YTHIP_CACHE_ERR_INDEX);
    if (len < 0 || end <= len) return;
    const int ch = threadIdx.x % LPR;
    // (a sequence may take more rows than the T that are given: zeros)
    for (int64_t i = (int64_t)run * APPEND_ROWS + threadIdx.x / LPR; len + i < min(end, cap); i += (int64_t)a.runs * APPEND_ROWS) {
        const int64_t pos = len + i;
        const int p = a.table[b * a.ld_table + (pos >> a.shift)], r = (int)pos & (page - 1);
        if (p < 0 || p >= a.pages) {
            if (tells && ch == 0 && a.status != nullptr) atomicOr(a.status, YTHIP_CACHE_ERR_INDEX);
            continue;
        }
        const int from = i >= a.T ? -1 : a.path != nullptr ? a.path[b * a.ld_path + i] : (int)i;
        const bool is = from >= 0 && from < a.T;
        const int64_t at = l * a.ns[0] + b * a.ns[1] + h * a.ns[2] + (is ? from : 0) * a.ns[3] + ch * 8 * (int64_t)sizeof(raw);
        uint8_t* pool[2] = {a.Kp, a.Vp};
        const char* src[2] = {a.Kn, a.Vn};
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            float x[8];
            constexpr int W = sizeof(raw) / 2;
            u32x4 v[W];
#pragma unroll
            for (int q = 0; q < W; ++q) {
                v[q] = *reinterpret_cast<const u32x4*>(src[kv] + at + 16 * q);
                if (!is) v[q] = u32x4{0u, 0u, 0u, 0u};
            }
            float top = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                if constexpr (W == 2) x[e] = __uint_as_float(v[e / 4][e % 4]);
                else x[e] = e & 1 ? hi_as_f32(T{}, v[0][e / 2]) : lo_as_f32(T{}, v[0][e / 2]);
                top = __builtin_elementwise_maximum(top, fabsf(x[e]));
            }
            // over the four lanes of the group
            auto quad = [](float f, auto ctrl) { return __int_as_float(__builtin_amdgcn_update_dpp(0, __float_as_int(f), decltype(ctrl)::value, 0xf, 0xf, false)); };
            top = __builtin_elementwise_maximum(top, quad(top, std::integral_constant<int, 0xb1>{}));
            top = __builtin_elementwise_maximum(top, quad(top, std::integral_constant<int, 0x4e>{}));
            const uint32_t byte = scale_byte<T>(top);
            const float scale = scale_of(byte == 255 ? 127 : byte);
            uint32_t codes = 0;
            codes = to_codes<0>(codes, x[0], x[1], scale);
            codes = to_codes<1>(codes, x[2], x[3], scale);
            codes = to_codes<2>(codes, x[4], x[5], scale);
            codes = to_codes<3>(codes, x[6], x[7], scale);
            uint8_t* block = pool[kv] + l * a.ps[0] + p * a.ps[1] + h * a.ps[2];
            if (kv == 0) {
                *reinterpret_cast<uint32_t*>(block + r * (D / 2) + ch * 4) = codes;
                if ((ch & 3) == 0) block[page * (D / 2) + r * (D / 32) + ch / 4] = (uint8_t)byte;
            } else {
                if constexpr (D == 128) {
                    *reinterpret_cast<uint32_t*>(block + v_code(r, ch, D)) = codes;
                } else {
                    *reinterpret_cast<uint16_t*>(block + v_code(r, 2 * ch, D)) = (uint16_t)codes;
                    *reinterpret_cast<uint16_t*>(block + v_code(r, 2 * ch + 1, D)) = (uint16_t)(codes >> 16);
                }
                if ((ch & 3) == 0) block[v_scale(page, r, ch / 4, D)] = (uint8_t)byte;
            }
        }
    }
}

// ---------------------------------------------------------------------------
// The pages' values
// ---------------------------------------------------------------------------

struct UnpackArgs {
    int layers, pages, Hkv, page;
    int64_t first;  // workgroups of earlier launches
    const uint8_t *Kp, *Vp;
    int64_t ps[3];  // bytes
    char *K, *V;    // [layers][pages][Hkv][page][d] in a row
};
// 16 rows of a block a workgroup, 8 channels a thread, so that a wave reads neighbouring codes and writes runs of a row:
// K row by row, V eight rows of eight entries at a time. Bound by the values' bytes.
template <class T, int D>
__global__ __launch_bounds__(16 * D / 8) void cache_unpack_q4_kernel(UnpackArgs a) {
    constexpr int LPR = D / 8;
    using raw = typename T::raw;
    const int runs = a.page / 16;
    int64_t w = a.first + blockIdx.x;
    const int r0 = (int)(w % runs) * 16;
    w /= runs;
    const bool is_v = w % 2;
    w /= 2;
    const int64_t block = w;
    const int h = (int)(w % a.Hkv);
    w /= a.Hkv;
    const int64_t p = w % a.pages, l = w / a.pages;
    const uint8_t* src = (is_v ? a.Vp : a.Kp) + l * a.ps[0] + p * a.ps[1] + h * a.ps[2];
    int r, ch;
    uint32_t codes, byte;
    if (!is_v) {
        r = r0 + threadIdx.x / LPR, ch = threadIdx.x % LPR;
        codes = *reinterpret_cast<const uint32_t*>(src + r * (D / 2) + ch * 4);
        byte = src[a.page * (D / 2) + r * (D / 32) + ch / 4];
    } else {
        r = r0 + threadIdx.x / (8 * LPR) * 8 + threadIdx.x % 8, ch = threadIdx.x / 8 % LPR;
        if constexpr (D == 128) {
            codes = *reinterpret_cast<const uint32_t*>(src + v_code(r, ch, D));
        } else {
            codes = *reinterpret_cast<const uint16_t*>(src + v_code(r, 2 * ch, D));
            codes |= (uint32_t)*reinterpret_cast<const uint16_t*>(src + v_code(r, 2 * ch + 1, D)) << 16;
        }
        byte = src[v_scale(a.page, r, ch / 4, D)];
    }
    const float scale = scale_of(byte);
    float x[8];
    const f32x2 y[4] = {to_f32<0>(codes, scale), to_f32<1>(codes, scale), to_f32<2>(codes, scale), to_f32<3>(codes, scale)};
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = y[e / 2][e % 2];
    char* out = (is_v ? a.V : a.K) + ((block * a.page + r) * D + ch * 8) * (int64_t)sizeof(raw);
    if constexpr (std::is_same_v<T, F32>) {
        *reinterpret_cast<f32x4*>(out) = f32x4{x[0], x[1], x[2], x[3]};
        *reinterpret_cast<f32x4*>(out + 16) = f32x4{x[4], x[5], x[6], x[7]};
    } else {
        *reinterpret_cast<u32x4*>(out) = u32x4{pack2<T>(x[0], x[1]), pack2<T>(x[2], x[3]), pack2<T>(x[4], x[5]), pack2<T>(x[6], x[7])};
    }
}

// ---------------------------------------------------------------------------
// Attention
// ---------------------------------------------------------------------------

// fp32 numbers as NP bfloat16 ones that add up to them (8 bits each; the last one rounded): one for bfloat16, two for
// float16's 11 bits, three for fp32's 24. An infinity is the first one's alone.
template <class T> constexpr int pieces() { return std::is_same_v<T, BF16> ? 1 : std::is_same_v<T, F16> ? 2 : 3; }

__device__ __forceinline__ uint32_t upper2(float x, float y) {  // the first 16 bits of both
#if defined(__HIP_DEVICE_COMPILE__)
    return __builtin_amdgcn_perm(__float_as_uint(y), __float_as_uint(x), 0x07060302);
#else
    return 0;
#endif
}
template <int NP>
__device__ __forceinline__ void split(float x, float y, uint32_t (&out)[NP]) {
#pragma unroll
    for (int i = 0; i < NP - 1; ++i) {
        out[i] = upper2(x, y);
        x = x - lo_as_f32(BF16{}, out[i]);
        y = y - hi_as_f32(BF16{}, out[i]);
    }
    out[NP - 1] = pack2<BF16>(x, y);
}
template <int NP>
__device__ __forceinline__ void split_any(float x, float y, uint32_t (&out)[NP]) {
#pragma unroll
    for (int i = 0; i < NP - 1; ++i) {
        out[i] = upper2(x, y);
        x = fabsf(x) < INFINITY ? x - lo_as_f32(BF16{}, out[i]) : i == 0 && x == x ? 0.f : x;
        y = fabsf(y) < INFINITY ? y - hi_as_f32(BF16{}, out[i]) : i == 0 && y == y ? 0.f : y;
    }
    out[NP - 1] = pack2<BF16>(x, y);
}

__device__ __forceinline__ float sum_across_rows(float v) {
    const uint32_t u = __float_as_uint(v);
    const auto p16 = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    v = __uint_as_float(p16[0]) + __uint_as_float(p16[1]);
    const uint32_t w = __float_as_uint(v);
    const auto p32 = __builtin_amdgcn_permlane32_swap(w, w, false, false);
    return __uint_as_float(p32[0]) + __uint_as_float(p32[1]);
}

// What stands in for a pool that has no pages, or where no sequence has a column: one page of 16 rows, which a tile's
// loads go to.
static __device__ const u32x4 no_pages[16 * (128 / 2 + 128 / 32) / 16] = {};

// (a lambda that is not inlined has its arrays in memory)
#define INLINE __attribute__((always_inline))

template <int D, int QT, int WR>
struct Q4Shape {
    static constexpr bool SHARED = WR == 4;
    static constexpr int KT = SHARED ? 64 : 32, WK = 4 / WR, RW = 16 * QT * WR;
    // Workgroups of a CU: three where 168 registers hold the queries' pieces, else two. Three load the next tile while one is
    // converted, two the next but one (16 sequences, 1 token, up to 32768 rows: 3 and 1 82 us, 2 and 2 88, 2 and 1 98, 3 and
    // 2 85).
    static constexpr int waves(bool bf16) { return QT == 1 && WR == 1 && (bf16 || D == 64) ? 3 : 2; }
    static constexpr int KS = D / 32, DT = D / 16, GROUPS = D / 32, OLD = D + 4;
    static constexpr int KF = 4 * KS, VF = 2 * DT;  // fragments of a tile (a register quadruple of each lane): of 16 rows, of 32
    // (in 16-byte chunks) two converted tiles, or the key groups' results
    static constexpr int LDS = SHARED ? 2 * 64 * (KF + VF) : (WK * RW * (OLD + 2) * 4 + 15) / 16;
};

// One workgroup: RW = 16 QT WR query rows of one KV head (row = token * G + head of the group) over a chunk of its
// sequence's tiles of 32 or 64 rows; its four waves have all its rows and a tile each in turn (WR 1), or its rows by fourths
// and every tile (WR 4). Codes go straight into registers, a tile or two early, and are bfloat16 after one conversion a
// pair; few rows: each wave converts its own tiles, many: each a fourth of every tile, which all read from LDS.
//   S^T = K . Q^T: of 16 rows (subtile j) lane (l16, g) has row 32 (j / 2) + 8 (l16 / 4) + l16 % 4 + 4 (j % 2) of the
//     tile, channels g D / 4 and on (the products' order over channels is free: Q is laid out alike), which is 16 (8) bytes
//     of codes and one scale. Of S^T it has query l16 and of each 32 rows rows 8 g .. 8 g + 7, in the order in which the
//     second product takes its weights.
//   O^T = V^T . P^T: the lane has rows 8 g .. 8 g + 7 of channels l16 D / 16 and on, 32 (16) consecutive bytes of a V block
//     and 8 scales; converted row by row, then paired by row (v_perm), it has each of its channels over 8 rows, which is
//     row l16 of channel tile t. So tile t's row i is channel i D / 16 + t.
//   New tokens are of the queries' type: their scores on its own matrix instruction, so their V, but float32's, which is
//     three bfloat16 pieces.
// Numerics: queries and weights as bfloat16 pieces (split) that hold all bits of the queries and 16 (24 for fp32) of the
//   weights; scores, maxima, sums and O in fp32. (The matrix cores' scaled product would take K's codes as they are, with
//   the queries as e4m3 pieces, but of every 8 products it drops what is 2^13 below the largest: fp32 scores were off by
//   2^-15 of their terms.)
template <class T, int D, int QT, int WR, bool WIN>
__global__ __launch_bounds__(256, (Q4Shape<D, QT, WR>::waves(std::is_same_v<T, BF16>))) void paged_q4_kernel(PagedArgs a) {
    using S = Q4Shape<D, QT, WR>;
    using raw = typename T::raw;
    constexpr bool F = std::is_same_v<T, F32>, SHARED = S::SHARED, HALF = std::is_same_v<T, F16>;
    constexpr int KT = S::KT, SUB = KT / 16, KG = KT / 32, KS = S::KS, DT = S::DT, NQ = pieces<T>(), NW = F ? 3 : 2, GROUPS = S::GROUPS;
    constexpr int ES = sizeof(raw);
    __shared__ u32x4 smem[S::LDS];
    __shared__ int16_t s_up[MAX_TREE];
    __shared__ uint32_t s_odd[SHARED ? 2 * 4 * 2 : 1];  // of a converted tile: bits of rows without a value, by channel group
    __shared__ int s_inf[4];  // of the tiles of new tokens there, by stage: V holds what is not finite
    // New tokens of 16 bits go through LDS too, as they are: a wave reads a quarter of a tile, not all of it (bfloat16, chunk
    // of 2048 after 2048 rows, window 1024: 219 -> 78 us; 4096 after 64, window 2048: 560 -> 221; two chunks of 512 over 8192:
    // 116 -> 96; float16, 2048 after 64: 169 -> 107). A single tile gains nothing, and loses nothing: five trees of 25 39.0 us,
    // each wave by itself 39.2. LDS has no room for float32's.
    constexpr bool SHARED_NEW = SHARED && !F;
    const int tid = threadIdx.x, lane = tid & 63, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int wr = wave % WR, wk = wave / WR;
    const int l16 = lane & 15, g = lane >> 4;

    // (item, KV head, row tile): the row tiles of an item and head read the same rows, so they go to one XCD
    int gi, rt;
    {
        const int w = blockIdx.x, q = w >> 3;
        rt = q % a.row_tiles;
        gi = (q / a.row_tiles) * 8 + (w & 7);
    }
    if (gi >= a.items * a.Hkv) return;
    const int h = gi % a.Hkv, item = a.items - 1 - gi / a.Hkv;
    const int R = a.T * a.G, r0 = rt * S::RW;
    int b, len, tn;
    Cut cut;
    if (a.target == 0) {
        b = item;
        len = rows_in_use(a, b), tn = new_rows(a, b);
    } else {
        cut = cut_of(a, KT, item, -1);
        if (cut.b < 0) return;
        b = cut.b, len = cut.len, tn = cut.tn;
    }
    b = uniform(b), len = uniform(len), tn = uniform(tn);
    const int t_first = r0 / a.G, t_last = min((min(R, r0 + S::RW) - 1) / a.G, tn - 1);
    const int32_t* table = a.table + b * a.ld_table;
    Seen seen = {(len + KT - 1) / KT, 0, 0};
    if constexpr (WIN) seen = seen_rows(a, len, KT);
    const int nct = seen.tiles, nt = nct + (a.Kn != nullptr ? (tn + KT - 1) / KT : 0);
    int c0 = 0, c1 = nt;
    bool whole = true;
    if (a.target != 0) {
        c0 = max(cut.at, 0);
        c1 = min(cut.at + cut.chunk, nt);
        whole = cut.count == 1;
    }
    c0 = uniform(c0), c1 = uniform(c1);
    if (t_first >= tn) return;
    Window win = {c0, c1, c0, 0, 0};
    if constexpr (WIN) win = window_of(a, seen, len, c0, c1, a.parents != nullptr ? 0 : t_first, t_last, KT);
    else win.high = min(c1, nct + t_last / KT + 1);
    const int tiles = WIN ? win.count() : max(win.high - c0, 0);
    const int nst = (tiles + S::WK - 1) / S::WK;

    const bool walk = a.parents != nullptr && (WIN || c1 > nct);
    if (walk) {
        for (int u = tid; u < tn; u += 256) {
            const int p = a.parents[b * a.ld_par + u];
            s_up[u] = (int16_t)(p >= 0 && p < u ? p : -1);
        }
        __syncthreads();
    }

    // ---- tiles of cached rows: lookups and loads
    // (where there is none, no id is one of a page: all loads are within page 0, the stand-in)
    const bool none = a.pages == 0;
    const int page = none ? 16 : 1 << a.shift;
    const int64_t page_str = none ? 0 : a.ps[0], head = none ? 0 : h * a.ps[1];
    const uint8_t* stand_in = reinterpret_cast<const uint8_t*>(no_pages);
    const uint8_t *Kp = (none ? stand_in : static_cast<const uint8_t*>(a.Kp)) + head, *Vp = (none ? stand_in : static_cast<const uint8_t*>(a.Vp)) + head;
    auto tile_at = [&](int s) { return WIN ? win.at(s * S::WK + wk) : win.high - 1 - (s * S::WK + wk); };
    struct Ids {
        int id[SUB];  // of the tile's 16 rows each
    };
    auto ids = [&](int s) INLINE {
        Ids x;
#pragma unroll
        for (int i = 0; i < SUB; ++i) x.id[i] = -1;
        const int ti = tile_at(s);
        if (ti < c0 || ti >= nct) return x;
        const int row = seen.row(ti, KT);
#pragma unroll
        for (int i = 0; i < SUB; ++i)
            if (row + 16 * i < len) x.id[i] = scalar_word(table + ((row + 16 * i) >> a.shift));
        return x;
    };
    // What a wave loads of a tile: K of its subtiles, V of its 32 rows
    constexpr int NK = SHARED ? 1 : SUB, NV = SHARED ? 1 : KG, VW = D / 64;
    struct Raw {
        u32x4 k[NK], v[NV][VW];  // (d 64: the first 8 bytes of k)
        uint32_t ks[NK];
        u32x2 vs[NV];
    };
    const int k_row = 8 * (l16 >> 2) + (l16 & 3), k_group = g * (D / 4) / 32, v_group = l16 * (D / 16) / 32;
    const uint32_t k_at = k_row * (D / 2) + g * (D / 8), ks_at = k_row * (D / 32) + k_group;
    const uint32_t v_at = (g * 16 + l16) * (8 * (D / 32)), vs_at = (g * (D / 32) + v_group) * 8;
    // (rows that a launch reads once stay out of the caches' way; those that row tiles share do not)
    auto fetch = [](auto* p) INLINE {
        if constexpr (SHARED) return *p;
        else return __builtin_nontemporal_load(p);
    };
    // Starts the loads of stage s; the rows of the tile that are in use. The loads are the same in number whatever the tile
    // is (one that is not there, or 16 rows that have no page, read another page and are hidden), so that the wait for one
    // tile's lets the next ones' go on: with a branch around them each waits for all in flight.
    auto load = [&](int s, const Ids& x, Raw& w) INLINE {
        const int ti = tile_at(s), row = seen.row(ti, KT);
        uint64_t use = 0;
        int any = 0;
#pragma unroll
        for (int i = 0; i < SUB; ++i)
            if ((uint32_t)x.id[i] < (uint32_t)a.pages) use |= 0xffffull << (16 * i), any = x.id[i];
        if (len - row < KT) use &= (1ull << max(len - row, 0)) - 1;
        auto page_of = [&](int i) { return (uint32_t)x.id[i] < (uint32_t)a.pages ? x.id[i] : any; };
#pragma unroll
        for (int i = 0; i < NV; ++i) {
            const int q = SHARED ? wave >> 1 : i;
            // where the 32 rows begin in a block, as their two halves have it: with pages of 16 rows those lie in two
            const int first = row + 32 * q, low = first & (page - 1), high = ((first + 16) & (page - 1)) - 16;
            const int64_t p0 = page_of(SHARED ? (wave >> 1 ? 2 : 0) : 2 * i) * page_str, p1 = page_of(SHARED ? (wave >> 1 ? 3 : 1) : 2 * i + 1) * page_str;
            const int64_t codes[2] = {p0 + low * (D / 2), p1 + high * (D / 2)};
            const int64_t scales[2] = {p0 + page * (D / 2) + low * (D / 32), p1 + page * (D / 2) + high * (D / 32)};
            const uint8_t *kc = Kp + (l16 >> 3 ? codes[1] : codes[0]) + k_at, *kx = Kp + (l16 >> 3 ? scales[1] : scales[0]) + ks_at;
            const uint8_t *vc = Vp + (g >> 1 ? codes[1] : codes[0]) + v_at, *vx = Vp + (g >> 1 ? scales[1] : scales[0]) + vs_at;
#pragma unroll
            for (int j = 0; j < NK / NV; ++j) {
                const int sub = SHARED ? wave & 1 : j;
                if constexpr (D == 128) w.k[i * (NK / NV) + j] = fetch(reinterpret_cast<const u32x4*>(kc + sub * 4 * (D / 2)));
                else {
                    const u32x2 y = fetch(reinterpret_cast<const u32x2*>(kc + sub * 4 * (D / 2)));
                    w.k[i * (NK / NV) + j] = u32x4{y[0], y[1], 0u, 0u};
                }
                w.ks[i * (NK / NV) + j] = kx[sub * 4 * (D / 32)];
            }
#pragma unroll
            for (int v = 0; v < VW; ++v) w.v[i][v] = fetch(reinterpret_cast<const u32x4*>(vc + 16 * v));
            w.vs[i] = *reinterpret_cast<const u32x2*>(vx);
        }
        return use;
    };

    // this lane's query rows
    int tok[QT], cur[QT], deep[QT], up[QT], lo[QT];
    const raw* qp[QT];
    u32x4 qf[QT][NQ][KS];
    const float flip = a.scale_log2 < 0.f ? -1.f : 1.f, c = fabsf(a.scale_log2);
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        const int r = r0 + wr * 16 * QT + qt * 16 + l16;
        const int rq = min(r, R - 1), t = rq / a.G, gh = rq - t * a.G;
        tok[qt] = r < R && t < tn ? t : -1;
        cur[qt] = tok[qt];
        deep[qt] = tok[qt];
        up[qt] = 0;
        if constexpr (WIN) {
            if (walk) {
                deep[qt] = -1;
                for (int u = tok[qt]; u >= 0; u = s_up[u]) ++deep[qt];
            }
        }
        lo[qt] = WIN ? (int)max((int64_t)len + deep[qt] + 1 - a.window, (int64_t)0) : 0;
        qp[qt] = static_cast<const raw*>(a.Q) + b * a.qs[0] + (int64_t)(h * a.G + gh) * a.qs[1] + t * a.qs[2] + g * (D / 4);
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) {
            float x[8];
            if constexpr (F) {
                const f32x4 v[2] = {*reinterpret_cast<const f32x4*>(qp[qt] + ks * 8), *reinterpret_cast<const f32x4*>(qp[qt] + ks * 8 + 4)};
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = v[e / 4][e % 4] * flip;
            } else {
                const u32x4 v = *reinterpret_cast<const u32x4*>(qp[qt] + ks * 8);
#pragma unroll
                for (int e = 0; e < 8; ++e) x[e] = (e & 1 ? hi_as_f32(T{}, v[e / 2]) : lo_as_f32(T{}, v[e / 2])) * flip;
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                uint32_t w[NQ];
                split_any<NQ>(x[2 * i], x[2 * i + 1], w);
#pragma unroll
                for (int n = 0; n < NQ; ++n) qf[qt][n][ks][i] = w[n];
            }
        }
    }

    float m[QT], l[QT];  // the largest score so far, before the scale; this lane's rows' share of the weights' sum
    f32x4 o[QT][DT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] = -INFINITY, l[qt] = 0.f;
#pragma unroll
        for (int t = 0; t < DT; ++t) o[qt][t] = f32x4{0.f, 0.f, 0.f, 0.f};
    }

    // The scores p of N 16 rows into weights, m and l anew; o is in the new maximum's unit then.
    auto weigh = [&](auto& p, int qt) INLINE {
        constexpr int N = sizeof(p) / sizeof(f32x4);
        float mx = -INFINITY;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) mx = __builtin_elementwise_maximum(mx, p[j][r]);
        const float top = __builtin_elementwise_maximum(m[qt], max_across_rows(mx));
        const float ref = top == -INFINITY ? 0.f : top;  // nothing seen yet: every weight is 0
        const float corr = __builtin_amdgcn_exp2f((m[qt] - ref) * c);
        m[qt] = top;
        float sum = 0.f;
#pragma unroll
        for (int j = 0; j < N; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                p[j][r] = __builtin_amdgcn_exp2f((p[j][r] - ref) * c);
                sum += p[j][r];
            }
        l[qt] = fmaf(l[qt], corr, sum);
        if (__ballot(corr != 1.0f) != 0) {
#pragma unroll
            for (int t = 0; t < DT; ++t) o[qt][t] *= corr;
        }
    };
    // The weights of 32 rows as the matrix cores take them
    auto split_weights = [&](const f32x4& p0, const f32x4& p1, u32x4 (&pw)[NW]) INLINE {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4& p = i < 2 ? p0 : p1;
            uint32_t w[NW];
            split<NW>(p[2 * (i & 1)], p[2 * (i & 1) + 1], w);
#pragma unroll
            for (int n = 0; n < NW; ++n) pw[n][i] = w[n];
        }
    };
    // (float16's: the first piece in a unit of 2^14, what is left in one of 2^25, below 2^15 as the first is)
    auto half_weights = [&](const f32x4& p0, const f32x4& p1, u32x4 (&pw)[NW]) INLINE {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const f32x4& p = i < 2 ? p0 : p1;
            const float x = p[2 * (i & 1)] * 0x1p14f, y = p[2 * (i & 1) + 1] * 0x1p14f;
#if defined(__HIP_DEVICE_COMPILE__)
            const uint32_t first = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_pkrtz(x, y));
            pw[0][i] = first;
            pw[NW - 1][i] = pack2<F16>((x - lo_as_f32(F16{}, first)) * 0x1p11f, (y - hi_as_f32(F16{}, first)) * 0x1p11f);
#endif
        }
    };
    auto hide_rows = [&](f32x4 (&p)[2], uint32_t see) INLINE {
        const uint32_t mine = see >> (8 * g);
#pragma unroll
        for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) p[j][r] = mine >> (4 * j + r) & 1 ? p[j][r] : -INFINITY;
    };
    // A channel pair of this lane's 8 rows, v[row], as row l16 of two channel tiles
    auto pair_rows = [](const uint32_t (&v)[8], u32x4& even, u32x4& odd) INLINE {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
#if defined(__HIP_DEVICE_COMPILE__)
            even[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x05040100);
            odd[i] = __builtin_amdgcn_perm(v[2 * i + 1], v[2 * i], 0x07060302);
#endif
        }
    };

    // Two 16-bit numbers, 0 in the place of one that is not finite
    auto finite_pair = [](uint32_t w, bool& bad) INLINE {
        constexpr uint32_t ONES = std::is_same_v<T, F16> ? 0x7c007c00u : 0x7f807f80u, LOW = 0x80008000u - ONES;
        const uint32_t none = (((w & ONES) + LOW) >> 15) & 0x00010001u;  // an exponent of ones
        bad = bad || none != 0;
        return w & ~(none * 0xffffu);
    };
    // The sums of one piece of V (two channel tiles) with the weights' two, each in its unit
    auto add_half = [&](int qt, int t, u32x4 even, u32x4 odd, const u32x4 (&pw)[NW]) INLINE {
        static_assert(!HALF || NW == 2);
        f32x4 y[2][NW] = {};
#pragma unroll
        for (int n = 0; n < NW; ++n) y[0][n] = mfma_chunk(T{}, even, pw[n], y[0][n]), y[1][n] = mfma_chunk(T{}, odd, pw[n], y[1][n]);
#pragma unroll
        for (int i = 0; i < 2; ++i)
#pragma unroll
            for (int r = 0; r < 4; ++r) o[qt][t + i][r] = fmaf(y[i][0][r], 0x1p-14f, fmaf(y[i][NW - 1][r], 0x1p-25f, o[qt][t + i][r]));
    };

    // ---- tiles of new tokens, by halves of 32
    const char* Kn = static_cast<const char*>(a.Kn) + (b * a.kns[0] + h * a.kns[1]) * ES;
    const char* Vn = static_cast<const char*>(a.Vn) + (b * a.vns[0] + h * a.vns[1]) * ES;
    auto new_rows_at = [&](int u0) INLINE {
        uint32_t see[QT];
        bool any = false;
        const int n = min(tn - u0, 32);
        if (n <= 0) return;
        const uint32_t there = n >= 32 ? ~0u : (1u << n) - 1;
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            see[qt] = 0;
            if (walk) {
                while (cur[qt] >= u0) {
                    const bool in = !WIN || up[qt] < a.window || deep[qt] - up[qt] < a.sinks - len;
                    if (in && cur[qt] < u0 + 32) see[qt] |= 1u << (cur[qt] - u0);
                    cur[qt] = s_up[cur[qt]];
                    ++up[qt];
                }
            } else if (tok[qt] >= u0) {
                see[qt] = ~from_bit(tok[qt] + 1 - u0);
                if constexpr (WIN) see[qt] &= from_bit((int64_t)tok[qt] + 1 - a.window - u0) | ~from_bit((int64_t)a.sinks - len - u0);
            }
            see[qt] &= there;
            any = any || see[qt] != 0;
        }
        if (__ballot(any) == 0) return;
        // channels l16 D / 16 and on of rows 8 g .. 8 g + 7, a pair at a time
        const char* v = Vn + l16 * (D / 16) * ES;
        int64_t at[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) at[e] = min(u0 + 8 * g + e, tn - 1) * a.vns[2] * ES;
        using Pair = std::conditional_t<F, u32x2, uint32_t>;
        auto pair_at = [&](int e, int q) INLINE { return *reinterpret_cast<const Pair*>(v + at[e] + q * (int)sizeof(Pair)); };
        // (in flight beside K where the registers reach for it, all at once, else a pair at a time: 1024 float32 tokens 153 ->
        // 142 us)
        constexpr bool EARLY = QT == 1 && (SHARED || std::is_same_v<T, BF16> || D == 64);
        Pair ahead[EARLY ? 8 : 1][EARLY ? DT / 2 : 1];
        if constexpr (EARLY) {
#pragma unroll
            for (int e = 0; e < 8; ++e)
#pragma unroll
                for (int q = 0; q < DT / 2; ++q) ahead[e][q] = pair_at(e, q);
        }
        f32x4 p[QT][2];
#pragma unroll
        for (int j = 0; j < 2; ++j) {
            const int u = min(u0 + k_row + 4 * j, tn - 1);
            const char* k = Kn + u * a.kns[2] * ES + g * (D / 4) * ES;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < D / 4 * ES / 16; ++ks) {
                const u32x4 kf = *reinterpret_cast<const u32x4*>(k + ks * 16);
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    p[qt][j] = mfma_chunk(T{}, kf, *reinterpret_cast<const u32x4*>(reinterpret_cast<const char*>(qp[qt]) + ks * 16), p[qt][j]);
            }
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt][j] *= flip;
        }
        // float16's V as it is takes fewer instructions than as two bfloat16 pieces (2048 tokens, each wave by itself: 183 -> 169
        // us); the weights are two float16 numbers then, each in a unit of its own (half_weights): 2^-22 of a weight is lost,
        // or 2^-50 of the largest. (In one unit, of 2^14, a weight below 2^-28 of the largest keeps less than 16 bits.)
        u32x4 pw[QT][NW];
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) {
            hide_rows(p[qt], see[qt]);
            weigh(p[qt], qt);
            if constexpr (HALF) half_weights(p[qt][0], p[qt][1], pw[qt]);
            else split_weights(p[qt][0], p[qt][1], pw[qt]);
        }
        bool bad = false;  // 0 . V is NaN for a V that is not finite: such elements are left out and added to those that see them
#pragma unroll
        for (int q = 0; q < DT / 2; ++q) {
            constexpr int NP = HALF ? 1 : pieces<T>();
            uint32_t part[NP][8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                Pair in;
                if constexpr (EARLY) in = ahead[e][q];
                else in = pair_at(e, q);
                if constexpr (HALF) {
                    part[0][e] = finite_pair(in, bad);
                    continue;
                }
                float x, y;
                if constexpr (F) x = __uint_as_float(in[0]), y = __uint_as_float(in[1]);
                else x = lo_as_f32(T{}, in), y = hi_as_f32(T{}, in);
                const bool fx = fabsf(x) < INFINITY, fy = fabsf(y) < INFINITY;
                bad = bad || !fx || !fy;
                uint32_t w[NP];
                split<NP>(fx ? x : 0.f, fy ? y : 0.f, w);
#pragma unroll
                for (int i = 0; i < NP; ++i) part[i][e] = w[i];
            }
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                u32x4 even, odd;
                pair_rows(part[i], even, odd);
                if constexpr (HALF) {
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt) add_half(qt, 2 * q, even, odd, pw[qt]);
                } else {
#pragma unroll
                    for (int n = 0; n < NW; ++n)
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt) {
                            o[qt][2 * q] = mfma_chunk(BF16{}, even, pw[qt][n], o[qt][2 * q]);
                            o[qt][2 * q + 1] = mfma_chunk(BF16{}, odd, pw[qt][n], o[qt][2 * q + 1]);
                        }
                }
            }
            if constexpr (!EARLY) __builtin_amdgcn_sched_barrier(0);
        }
        if (__ballot(bad) == 0) return;
        for (int u = 0; u < n; ++u) {
            const int64_t row = (u0 + u) * a.vns[2];
#pragma unroll
            for (int t = 0; t < DT; ++t)
#pragma unroll
                for (int r = 0; r < 4; ++r) {
                    const float x = load_as_f32<T>(Vn, row + (4 * g + r) * (D / 16) + t);
#pragma unroll
                    for (int qt = 0; qt < QT; ++qt)
                        if (!(fabsf(x) < INFINITY) && (see[qt] >> u & 1)) o[qt][t][r] += x;
                }
        }
    };

    // ---- tiles of cached rows: values
    constexpr uint64_t FULL = KT == 64 ? ~0ull : (1ull << (KT & 63)) - 1;
    auto k_frag = [&](const Raw& w, int i, int ks) INLINE {
        const float scale = scale_of(w.ks[i]);
        const uint32_t y = w.k[i][ks];
        return u32x4{to_bf16<0>(y, scale), to_bf16<1>(y, scale), to_bf16<2>(y, scale), to_bf16<3>(y, scale)};
    };
    // Rows of 32 that are not in use may hold any scale: 1 in its place. `some`: rows that not every query sees are among
    // them, so that a row without a value gets 1 too; its bit is in the result, a word for the lane's channel group c.
    auto clean_scales = [&](u32x2& vs, uint32_t use, bool some, int c) INLINE {
        const uint32_t mine = use >> (8 * g);
        uint32_t odd = 0;
        // (a byte of 255: bit 7 of it, and of its complement less 1)
        const uint32_t none = vs[0] & (~vs[0] - 0x01010101u) & 0x80808080u, none1 = vs[1] & (~vs[1] - 0x01010101u) & 0x80808080u;
        some = some && __ballot((none | none1) != 0) != 0;
        if (!some && use == ~0u) return odd;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint32_t byte = vs[e / 4] >> (8 * (e % 4)) & 255;
            const bool in = mine >> e & 1;
            if (some) {
                // lane 16 i + l16 has rows 8 i .. of channel group v_group(l16)
                const uint64_t bad = __ballot(in && byte == 255);
                for (int i = 0; i < 4; ++i) odd |= (uint32_t)(bad >> (16 * i + c * (512 / D)) & 1) << (8 * i + e);
            }
            if (!in || (some && byte == 255)) vs[e / 4] = (vs[e / 4] & ~(255u << (8 * (e % 4)))) | 127u << (8 * (e % 4));
        }
        return odd;
    };
    // V fragments of channel tiles 2 q and 2 q + 1 over 32 rows
    auto v_frags = [&](const Raw& w, int i, auto q, u32x4& even, u32x4& odd) INLINE {
        constexpr int Q = decltype(q)::value;
        uint32_t v[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const float scale = scale_of(w.vs[i][e / 4] >> (8 * (e % 4)) & 255);
            // (d 128: a dword a row; d 64: two rows a dword)
            if constexpr (D == 128) v[e] = to_bf16<Q>(w.v[i][e / 4][e % 4], scale);
            else v[e] = e & 1 ? to_bf16<Q + 2>(w.v[i][0][e / 2], scale) : to_bf16<Q>(w.v[i][0][e / 2], scale);
        }
        pair_rows(v, even, odd);
    };
    // A wave's share of a tile into LDS (SHARED): K's subtile `wave`, and every second channel pair of V's 32 rows
    auto convert = [&](int s, uint64_t use, Raw& w) INLINE {
        if (use == 0) return;
        u32x4* to = smem + (s & 1) * 64 * (S::KF + S::VF) + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) to[(wave * KS + ks) * 64] = k_frag(w, 0, ks);
        const int half = wave >> 1;
        if (WIN || use != FULL) {
            const uint32_t odd = clean_scales(w.vs[0], (uint32_t)(use >> (32 * half)), WIN, lane & (GROUPS - 1));
            if (WIN && lane < GROUPS && (wave & 1) == 0) s_odd[((s & 1) * 4 + lane) * 2 + half] = odd;
        }
        to += (S::KF + half * DT) * 64;
        static_for<0, DT / 4>([&](auto i) {
            u32x4 even, odd;
            if (wave & 1) {
                v_frags(w, 0, std::integral_constant<int, 2 * decltype(i)::value + 1>{}, even, odd);
                to[(4 * decltype(i)::value + 2) * 64] = even, to[(4 * decltype(i)::value + 3) * 64] = odd;
            } else {
                v_frags(w, 0, std::integral_constant<int, 2 * decltype(i)::value>{}, even, odd);
                to[(4 * decltype(i)::value) * 64] = even, to[(4 * decltype(i)::value + 1) * 64] = odd;
            }
        });
    };

    // The same for a tile of new tokens: what a wave has of it, and its share into LDS
    struct RawNew {
        u32x4 k[SHARED_NEW ? KS : 1];
        uint32_t v[SHARED_NEW ? 8 : 1][SHARED_NEW ? DT / 4 : 1];
    };
    auto load_new = [&](int s, RawNew& w) INLINE {
        const int u0 = (tile_at(s) - nct) * KT, half = u0 + 32 * (wave >> 1);
        const char* k = Kn + min(half + k_row + 4 * (wave & 1), tn - 1) * a.kns[2] * ES + g * (D / 4) * ES;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) w.k[ks] = *reinterpret_cast<const u32x4*>(k + ks * 16);
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const char* v = Vn + min(half + 8 * g + e, tn - 1) * a.vns[2] * ES + l16 * (D / 16) * ES + 4 * (wave & 1);
#pragma unroll
            for (int i = 0; i < DT / 4; ++i) w.v[e][i] = *reinterpret_cast<const uint32_t*>(v + 8 * i);
        }
    };
    auto convert_new = [&](int s, RawNew& w) INLINE {
        u32x4* to = smem + (s & 1) * 64 * (S::KF + S::VF) + lane;
#pragma unroll
        for (int ks = 0; ks < KS; ++ks) to[(wave * KS + ks) * 64] = w.k[ks];
        to += (S::KF + (wave >> 1) * DT + 2 * (wave & 1)) * 64;
        // 0 . V is NaN for a V that is not finite: such elements are left out, and added for the queries that see them
        bool bad = false;
#pragma unroll
        for (int i = 0; i < DT / 4; ++i) {
            uint32_t v[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                v[e] = finite_pair(w.v[e][i], bad);
            }
            u32x4 even, odd;
            pair_rows(v, even, odd);
            to[4 * i * 64] = even, to[(4 * i + 1) * 64] = odd;
        }
        if (__ballot(bad) != 0 && lane == 0) s_inf[s & 3] = 1;
    };

    // new tokens first, from the last: their paths are walked down once
    const int new_tiles = WIN ? max(win.high - max(win.low, nct), 0) + max(win.sink_end - max(c0, nct), 0) : max(win.high - max(c0, nct), 0);
    // float16's queries as they are, which its new tokens meet
    u32x4 qr[SHARED_NEW && HALF ? KS : 1];
    if constexpr (SHARED_NEW && HALF) {
        static_assert(QT == 1);
        if (new_tiles > 0) {
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) qr[ks] = *reinterpret_cast<const u32x4*>(qp[0] + ks * 8);
        }
    }

    auto compute = [&](int s, uint64_t use, Raw& w, auto masked, auto fresh) INLINE {
        constexpr bool MASKED = decltype(masked)::value, is_new = decltype(fresh)::value;
        uint64_t see[QT];
        bool hide = use != FULL, some = false;  // some: a query sees rows of it that another does not
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) see[qt] = use;
        if constexpr (is_new) {
            const int u0 = (tile_at(s) - nct) * KT;
            bool any = false;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                uint64_t mine = 0;
                if (walk) {
                    while (cur[qt] >= u0) {
                        const bool in = !WIN || up[qt] < a.window || deep[qt] - up[qt] < a.sinks - len;
                        if (in && cur[qt] < u0 + KT) mine |= 1ull << (cur[qt] - u0);
                        cur[qt] = s_up[cur[qt]];
                        ++up[qt];
                    }
                } else if (tok[qt] >= u0) {
                    mine = ~from_bit(tok[qt] + 1 - u0);
                    if constexpr (WIN) mine &= from_bit((int64_t)tok[qt] + 1 - a.window - u0) | ~from_bit((int64_t)a.sinks - len - u0);
                }
                see[qt] &= mine;
                any = any || see[qt] != 0;
                some = some || see[qt] != use;
            }
            if (__ballot(any) == 0) return;
            hide = hide || __ballot(some) != 0;
        } else if constexpr (MASKED && WIN) {
            const int j0 = seen.row(tile_at(s), KT);
            bool any = false;
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                see[qt] &= from_bit((int64_t)lo[qt] - j0) | ~from_bit((int64_t)a.sinks - j0);
                any = any || see[qt] != 0;
                some = some || see[qt] != use;
            }
            if (__ballot(any) == 0) return;
            some = __ballot(some) != 0;
            hide = hide || some;
        }
        const u32x4* from = smem + (s & 1) * 64 * (S::KF + S::VF) + lane;
        f32x4 p[QT][SUB];
#pragma unroll
        for (int j = 0; j < SUB; ++j) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) p[qt][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int ks = 0; ks < KS; ++ks) {
                u32x4 kf;
                if constexpr (SHARED) kf = from[(j * KS + ks) * 64];
                else kf = k_frag(w, j, ks);
                if constexpr (is_new && HALF) {
                    p[0][j] = mfma_chunk(T{}, kf, qr[ks], p[0][j]);
                } else {
#pragma unroll
                    for (int n = 0; n < NQ; ++n)
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt) p[qt][j] = mfma_chunk(BF16{}, kf, qf[qt][n][ks], p[qt][j]);
                }
            }
            if constexpr (is_new && HALF) p[0][j] *= flip;
        }
        uint32_t odd[KG] = {};  // rows without a value in this lane's channels that not every query sees
        if (hide) {
            // (few tiles come here: what is worked out stays behind the branch)
            uint32_t mine[2] = {(uint32_t)use, (uint32_t)(use >> 32)};
            asm volatile("" : "+s"(mine[0]), "+s"(mine[1]));
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
#pragma unroll
                for (int kk = 0; kk < KG; ++kk) {
                    f32x4 y[2] = {p[qt][2 * kk], p[qt][2 * kk + 1]};
                    hide_rows(y, MASKED ? (uint32_t)(see[qt] >> (32 * kk)) & mine[kk] : mine[kk]);
                    p[qt][2 * kk] = y[0], p[qt][2 * kk + 1] = y[1];
                }
            }
            if constexpr (!SHARED) {
#pragma unroll
                for (int kk = 0; kk < KG; ++kk) odd[kk] = clean_scales(w.vs[kk], mine[kk], some, g * (D / 4) / 32);
            }
        }
        if constexpr (SHARED && WIN && !is_new) {
#pragma unroll
            for (int kk = 0; kk < KG; ++kk) odd[kk] = s_odd[((s & 1) * 4 + g * (D / 4) / 32) * 2 + kk];
        }
#pragma unroll
        for (int qt = 0; qt < QT; ++qt) weigh(p[qt], qt);
#pragma unroll
        for (int kk = 0; kk < KG; ++kk) {
            u32x4 pw[QT][NW];
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                if constexpr (is_new && HALF) half_weights(p[qt][2 * kk], p[qt][2 * kk + 1], pw[qt]);
                else split_weights(p[qt][2 * kk], p[qt][2 * kk + 1], pw[qt]);
            }
            static_for<0, DT / 2>([&](auto q) {
                constexpr int Q = decltype(q)::value;
                u32x4 even, odd_;
                if constexpr (SHARED) even = from[(S::KF + kk * DT + 2 * Q) * 64], odd_ = from[(S::KF + kk * DT + 2 * Q + 1) * 64];
                else v_frags(w, kk, q, even, odd_);
                if constexpr (is_new && HALF) {
                    add_half(0, 2 * Q, even, odd_, pw[0]);
                } else {
#pragma unroll
                    for (int n = 0; n < NW; ++n)
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt) {
                            o[qt][2 * Q] = mfma_chunk(BF16{}, even, pw[qt][n], o[qt][2 * Q]);
                            o[qt][2 * Q + 1] = mfma_chunk(BF16{}, odd_, pw[qt][n], o[qt][2 * Q + 1]);
                        }
                }
            });
        }
        if (is_new && s_inf[s & 3] != 0) {  // (of all waves' shares)
            const int u0 = (tile_at(s) - nct) * KT;
            for (int u = 0; u < min(tn - u0, KT); ++u) {
                const int64_t row = (u0 + u) * a.vns[2];
#pragma unroll
                for (int t = 0; t < DT; ++t)
#pragma unroll
                    for (int r = 0; r < 4; ++r) {
                        const float x = load_as_f32<T>(Vn, row + (4 * g + r) * (D / 16) + t);
#pragma unroll
                        for (int qt = 0; qt < QT; ++qt)
                            if (!(fabsf(x) < INFINITY) && (see[qt] >> u & 1)) o[qt][t][r] += x;
                    }
            }
        }
        if constexpr (SHARED ? WIN : MASKED) {
            const uint64_t none = odd[0] | (KG == 2 ? (uint64_t)odd[KG - 1] << 32 : 0);
            if (__ballot(none != 0) != 0) {
#pragma unroll
                for (int qt = 0; qt < QT; ++qt)
                    if (none & see[qt]) {
#pragma unroll
                        for (int t = 0; t < DT; ++t) o[qt][t] = f32x4{NAN, NAN, NAN, NAN};
                    }
            }
        }
    };

    const int s_first = new_tiles / S::WK;  // the first stage with a tile of cached rows (for some wave)
    // the stages whose tiles every query sees whole end there; then those at the window's border and the sinks
    const int s_whole = WIN ? max(s_first, max(win.high - max(win.low, win.clean), 0) / S::WK) : nst;
    auto new_tokens = [&]() INLINE {
        for (int i = wk; i < new_tiles; i += S::WK) {
            const int u0 = ((WIN ? win.at(i) : win.high - 1 - i) - nct) * KT;
#pragma unroll 1
            for (int u = u0 + KT - 32; u >= u0; u -= 32) new_rows_at(u);
        }
    };
    if constexpr (SHARED_NEW) {
        // as below, from the new tokens' tiles on
        if (tid < 4) s_inf[tid] = 0;
        __syncthreads();
        Raw w;
        RawNew fresh;
        uint64_t here, next = 0;
        auto there = [&](int s) { return from_bit(tn - (tile_at(s) - nct) * KT); };  // rows behind the last new token
        Ids x = ids(0);
        uint64_t use = load(0, x, w);
        if (new_tiles > 0) {
            load_new(0, fresh);
            convert_new(0, fresh);
            here = ~there(0);
        } else {
            convert(0, use, w);
            here = use;
        }
        x = ids(1);
        next = load(1, x, w);
        x = ids(2);
        auto stage = [&](int s, auto masked, auto more_new) INLINE {
            __syncthreads();
            const bool fresh_next = decltype(more_new)::value && s + 1 < new_tiles;
            if (fresh_next) load_new(s + 1, fresh);
            if (here != 0) compute(s, here, w, masked, more_new);
            // (read two stages ago, written again in the next)
            if (decltype(more_new)::value && tid == 0) s_inf[(s + 2) & 3] = 0;
            if (fresh_next) {
                convert_new(s + 1, fresh);
                here = ~there(s + 1);
            } else {
                convert(s + 1, next, w);
                here = next;
            }
            next = load(s + 2, x, w);
            x = ids(s + 3);
        };
        for (int s = 0; s < new_tiles; ++s) stage(s, std::true_type{}, std::true_type{});
        for (int s = new_tiles; s < s_whole; ++s) stage(s, std::false_type{}, std::false_type{});
        if constexpr (WIN)
            for (int s = s_whole; s < nst; ++s) stage(s, std::true_type{}, std::false_type{});
    } else if constexpr (SHARED) {
        new_tokens();
        // stage s is computed while s + 1 is converted and s + 2 is on its way: one barrier a stage
        Raw w;
        uint64_t use = load(s_first, ids(s_first), w), here = use, next;
        Ids x = ids(s_first + 1);
        convert(s_first, use, w);
        next = load(s_first + 1, x, w);
        x = ids(s_first + 2);
        auto stage = [&](int s, auto masked) INLINE {
            __syncthreads();
            if (here != 0) compute(s, here, w, masked, std::false_type{});
            convert(s + 1, next, w);
            here = next;
            next = load(s + 2, x, w);
            x = ids(s + 3);
        };
        for (int s = s_first; s < s_whole; ++s) stage(s, std::false_type{});
        if constexpr (WIN)
            for (int s = s_whole; s < nst; ++s) stage(s, std::true_type{});
    } else {
        constexpr int AHEAD = S::waves(std::is_same_v<T, BF16>) == 3 || (WIN && QT == 2) ? 1 : 2;
        Raw w[AHEAD];
        uint64_t use[AHEAD];
        Ids nx;
        auto start = [&]() INLINE {
            Ids x[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) x[i] = ids(s_first + i);
            nx = ids(s_first + AHEAD);
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) use[i] = load(s_first + i, x[i], w[i]);
        };
        // (the cached rows' first loads run beside the new tokens where the registers reach for both)
        if constexpr (QT == 1) start();
        new_tokens();
        if constexpr (QT > 1) start();
        auto stages = [&](int s, int to, auto masked) INLINE {
            while (s < to) {
#pragma unroll
                for (int i = 0; i < AHEAD; ++i) {
                    if (use[i] != 0) compute(s, use[i], w[i], masked, std::false_type{});
                    use[i] = load(s + AHEAD, nx, w[i]);
                    nx = ids(s + AHEAD + 1);
                    ++s;
                }
            }
            return s;
        };
        if constexpr (WIN) {
            // (by whole turns of the registers)
            const int at = stages(s_first, s_first + (s_whole - s_first) / AHEAD * AHEAD, std::false_type{});
            stages(at, nst, std::true_type{});
        } else {
            stages(s_first, nst, std::false_type{});
        }
    }

    float L[QT];
#pragma unroll
    for (int qt = 0; qt < QT; ++qt) {
        m[qt] *= c;
        L[qt] = sum_across_rows(l[qt]);
    }
    auto store4 = [&](int r, int d, f32x4 v, float M, float sum) INLINE {
        const int t = r / a.G, gh = r - t * a.G;
        if (r >= R || t >= tn) return;
        if (whole) {
            raw* op = static_cast<raw*>(a.O) + b * a.os[0] + (int64_t)(h * a.G + gh) * a.os[1] + t * a.os[2] + d;
            const float inv = M == -INFINITY ? 0.f : 1.0f / sum;
            v = M == -INFINITY ? f32x4{0.f, 0.f, 0.f, 0.f} : v * inv;
            if constexpr (F) *reinterpret_cast<f32x4*>(op) = v;
            else *reinterpret_cast<u32x2*>(op) = u32x2{pack2<T>(v[0], v[1]), pack2<T>(v[2], v[3])};
            return;
        }
        const int64_t at = ((int64_t)item * a.Hkv + h) * R + r;
        *reinterpret_cast<f32x4*>(a.part + at * D + d) = v;
        if (d == 0) {
            a.part_ml[2 * at] = M;
            a.part_ml[2 * at + 1] = sum;
        }
    };
    // channels (4 g + r) D / 16 and on of a query, four at a time
    auto each4 = [&](auto f) INLINE {
#pragma unroll
        for (int qt = 0; qt < QT; ++qt)
#pragma unroll
            for (int r = 0; r < 4; ++r)
#pragma unroll
                for (int t = 0; t < DT; t += 4)
                    f(qt, (4 * g + r) * (D / 16) + t, f32x4{o[qt][t][r], o[qt][t + 1][r], o[qt][t + 2][r], o[qt][t + 3][r]});
    };
    if constexpr (S::WK == 1) {
        each4([&](int qt, int d, f32x4 v) { store4(r0 + wr * 16 * QT + qt * 16 + l16, d, v, m[qt], L[qt]); });
    } else {
        // the key groups' results side by side in LDS, then joined
        float *so = reinterpret_cast<float*>(smem), *sm = so + S::WK * S::RW * S::OLD;
        each4([&](int qt, int d, f32x4 v) { *reinterpret_cast<f32x4*>(so + (wk * S::RW + wr * 16 * QT + qt * 16 + l16) * S::OLD + d) = v; });
        if (g == 0) {
#pragma unroll
            for (int qt = 0; qt < QT; ++qt) {
                const int row = wk * S::RW + wr * 16 * QT + qt * 16 + l16;
                sm[2 * row] = m[qt];
                sm[2 * row + 1] = L[qt];
            }
        }
        // (LDS alone: the loads of tiles behind the last are not waited for)
        asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
        for (int i = tid; i < S::RW * D / 4; i += 256) {
            const int row = i / (D / 4), d = i % (D / 4) * 4;
            float M = -INFINITY, sum = 0.f;
#pragma unroll
            for (int k = 0; k < S::WK; ++k) M = __builtin_elementwise_maximum(M, sm[2 * (k * S::RW + row)]);
            const float ref = M == -INFINITY ? 0.f : M;
            f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int k = 0; k < S::WK; ++k) {
                const float f = __builtin_amdgcn_exp2f(sm[2 * (k * S::RW + row)] - ref);
                sum += f * sm[2 * (k * S::RW + row) + 1];
                v += f * *reinterpret_cast<const f32x4*>(so + (k * S::RW + row) * S::OLD + d);
            }
            store4(r0 + row, d, v, M, sum);
        }
    }
}

// How a call is cut (plan_of, for the shapes of paged_q4_kernel).
Plan plan_q4(int dtype, int B, int Hkv, int G, int T, int d, int columns, int page, int window, int sinks) {
    Plan p;
    const int64_t rows = (int64_t)T * G;
    // 16 rows of a wave (bfloat16: 32) leave the tiles to the four; more share them (8 sequences, 32 rows over 8192: 32.9 us,
    // shared 41.1). 32 rows of a wave where there are more than 64 and one piece a query leaves the registers (two chunks of
    // 512 over 8192 rows 101.6 us, with 16 115; 16 x 200 rows over 4096 133 and 146); with a window 16 where that fills the
    // second place of the CUs (chunk of 2048, window 1024: 78.9 us, with 32 96.5; 4 chunks of 512, window 4096 147 and 182)
    const bool few = rows <= (dtype == YTHIP_BF16 ? 32 : 16);
    p.wr = few ? 1 : 4;
    p.qt = few ? (rows <= 16 ? 1 : 2) : rows <= 64 || dtype != YTHIP_BF16 ? 1 : 2;
    if (window > 0 && !few && (int64_t)B * Hkv * ((rows + 127) / 128) < SLOTS) p.qt = 1;
    p.kt = few ? 32 : 64;
    const int rw = 16 * p.qt * p.wr;
    p.row_tiles = (int)((rows + rw - 1) / rw);
    const int64_t per = (int64_t)Hkv * p.row_tiles;
    p.stage = 4 / p.wr;
    const int64_t slots = p.wr == 1 && p.qt == 1 && (dtype == YTHIP_BF16 || d == 64) ? SLOTS / 2 * 3 : SLOTS;
    p.short_run = p.wr > 1 ? 4 : 0;
    int64_t seq_rows = (int64_t)columns * page;
    if (window > 0) seq_rows = std::min(seq_rows, (int64_t)window + sinks + 2 * p.kt);
    const int64_t tiles = (seq_rows + p.kt - 1) / p.kt + ((int64_t)T + p.kt - 1) / p.kt, most = (tiles + p.stage - 1) / p.stage;
    int64_t part_items = 0;
    // (no ranges, as in plan_of: 8 chunks of 256, window 1024 58 us, cut into ranges 78; with a window that is long beside
    // most of the sequences they would be better: chunks of 512 over 4096 and three times 600 rows, window 4096 138 us, cut 91)
    if (most <= WHOLE || (window > 0 && !few && B * per >= SLOTS / 2)) {
        p.target = 0;
        p.items = B;
    } else {
        int64_t ranges = slots / per;
        p.even = B <= EVEN_SEQS && B <= ranges && ranges <= 8 * B;
        if (!p.even && B - 1 <= ranges / 2) ranges -= B - 1;
        p.target = (int)std::min(std::max<int64_t>(1, ranges), B * most);
        p.items = (int64_t)p.target + (p.even ? 0 : B - 1);
        if (p.target > 1) part_items = p.items;
    }
    const int64_t part_rows = part_items * Hkv * rows;
    p.part_bytes = (size_t)part_rows * d * sizeof(float);
    p.ml_bytes = ((size_t)part_rows * 2 * sizeof(float) + 15) / 16 * 16;
    p.rank_bytes = 0;
    return p;
}

template <class T, int D, int QT, int WR, bool WIN>
int launch_q4(const PagedArgs& a, const Plan& p, hipStream_t s) {
    const int64_t groups = (p.items * a.Hkv + 7) / 8 * 8;
    paged_q4_kernel<T, D, QT, WR, WIN><<<(int)(groups * p.row_tiles), 256, 0, s>>>(a);
    if (p.part_bytes > 0) merge_partials<T, D, false>(a, p.kt, s);
    return status_of(hipGetLastError());
}
template <class T, int D, bool WIN>
int run_q4(const PagedArgs& a, const Plan& p, hipStream_t s) {
    if (p.wr == 1 && p.qt == 1) return launch_q4<T, D, 1, 1, WIN>(a, p, s);
    if constexpr (std::is_same_v<T, BF16>) {
        if (p.wr == 1) return launch_q4<T, D, 2, 1, WIN>(a, p, s);
        if (p.qt == 2) return launch_q4<T, D, 2, 4, WIN>(a, p, s);
    }
    return launch_q4<T, D, 1, 4, WIN>(a, p, s);
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------

int page_shift(int page) {
    for (int s = 4; s <= 15; ++s)
        if (page == 1 << s) return s;
    return -1;
}

// Page, head dim and a pool's strides (layer, page, head; bytes) and addresses.
int check_blocks(const char* who, int layers, int pages, int Hkv, int page, int d, const void* Kp, const void* Vp,
                 const int64_t* pool_str, int64_t (&ps)[3]) {
    if (page_shift(page) < 0) return fail(YTHIP_EINVAL, "%s: a page of %d rows (a power of two from 16 to 32768)", who, page);
    if (d != 64 && d != 128) return fail(YTHIP_EUNSUPPORTED, "%s: head dim %d (64 or 128)", who, d);
    if (layers == 0 || pages == 0 || Hkv == 0) return 0;
    if (!Kp || !Vp || !pool_str) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    int64_t all = (int64_t)(uintptr_t)Kp | (int64_t)(uintptr_t)Vp;
    const int dims[3] = {layers, pages, Hkv};
    for (int i = 0; i < 3; ++i) {
        ps[i] = dims[i] > 1 ? pool_str[i] : 0;
        all |= ps[i];
    }
    if ((all & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: pages must be 16-byte aligned", who);
    return 0;
}

}  // namespace
}  // namespace ythip

using namespace ythip;

extern "C" {

__attribute__((visibility("default"))) int64_t ythip_cache_q4_bytes(int page, int d) {
    return page_shift(page) >= 0 && (d == 64 || d == 128) ? block_bytes(page, d) : 0;
}

__attribute__((visibility("default"))) int ythip_cache_append_q4(
    int dtype, int layers, int B, int Hkv, int T, int d, const void* Kn, const void* Vn, const int64_t new_str[4],
    void* Kp, void* Vp, const int64_t pool_str[3], int pages, int page, const int32_t* table, int64_t ld_table,
    int columns, const int32_t* kv_len, const int32_t* n_new, const int32_t* new_len, const int32_t* path,
    int64_t ld_path, int32_t* status, void* stream) {
    const char* who = "ythip_cache_append_q4";
    if (dtype != YTHIP_F32 && dtype != YTHIP_F16 && dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, dtype);
    if (layers < 0 || B < 0 || Hkv < 0 || T < 0 || pages < 0 || columns < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    if (n_new != nullptr && new_len != nullptr) return fail(YTHIP_EINVAL, "%s: n_new and new_len both say how many rows there are", who);
    if (new_len != nullptr && new_len == kv_len) return fail(YTHIP_EINVAL, "%s: kv_len and new_len are one array, so no row is new", who);
    if (columns > 65536 || (int64_t)columns * page > 1 << 30)
        return fail(YTHIP_EUNSUPPORTED, "%s: %d columns of %d rows (at most 65536 columns, 2^30 rows)", who, columns, page);
    AppendQ4Args a;
    if (const int st = check_blocks(who, layers, pages, Hkv, page, d, Kp, Vp, pool_str, a.ps)) return st;
    if (layers == 0 || B == 0 || Hkv == 0 || T == 0 || pages == 0 || columns == 0) return 0;
    if (!Kn || !Vn || !new_str || !table || !kv_len) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if (ld_table < columns) return fail(YTHIP_EINVAL, "%s: a table row of %d entries at a stride of %lld", who, columns, (long long)ld_table);
    if (path && ld_path < T) return fail(YTHIP_EINVAL, "%s: a path of %d entries at a stride of %lld", who, T, (long long)ld_path);
    const int es = dtype == YTHIP_F32 ? 4 : 2;
    int64_t all = (int64_t)(uintptr_t)Kn | (int64_t)(uintptr_t)Vn;
    const int dims[4] = {layers, B, Hkv, T};
    for (int i = 0; i < 4; ++i) {
        a.ns[i] = dims[i] > 1 ? new_str[i] * es : 0;
        all |= a.ns[i];
    }
    if ((all & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
    a.layers = layers, a.B = B, a.Hkv = Hkv, a.T = T, a.pages = pages, a.shift = page_shift(page), a.columns = columns;
    a.runs = (T + APPEND_ROWS - 1) / APPEND_ROWS;
    a.Kn = static_cast<const char*>(Kn), a.Vn = static_cast<const char*>(Vn);
    a.Kp = static_cast<uint8_t*>(Kp), a.Vp = static_cast<uint8_t*>(Vp);
    a.table = table, a.kv_len = kv_len, a.count = new_len ? new_len : n_new, a.path = path, a.ld_table = ld_table, a.ld_path = ld_path;
    a.to = new_len != nullptr, a.status = status;
    const int64_t grid = (int64_t)a.runs * Hkv * B * layers;
    if (!launchable(grid, APPEND_ROWS * d / 8)) return fail(YTHIP_EUNSUPPORTED, "%s: %lld workgroups", who, (long long)grid);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T_ = decltype(t);
        if (d == 64) cache_append_q4_kernel<T_, 64><<<(int)grid, APPEND_ROWS * 8, 0, s>>>(a);
        else cache_append_q4_kernel<T_, 128><<<(int)grid, APPEND_ROWS * 16, 0, s>>>(a);
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) int ythip_cache_unpack_q4(int dtype, int layers, int pages, int Hkv, int page, int d,
                                                                 const void* Kp, const void* Vp, const int64_t pool_str[3],
                                                                 void* K, void* V, void* stream) {
    const char* who = "ythip_cache_unpack_q4";
    if (dtype != YTHIP_F32 && dtype != YTHIP_F16 && dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, dtype);
    if (layers < 0 || pages < 0 || Hkv < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    UnpackArgs a;
    if (const int st = check_blocks(who, layers, pages, Hkv, page, d, Kp, Vp, pool_str, a.ps)) return st;
    if (layers == 0 || pages == 0 || Hkv == 0) return 0;
    if (!K || !V) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if ((((uintptr_t)K | (uintptr_t)V) & 15) != 0) return fail(YTHIP_EUNSUPPORTED, "%s: rows must be 16-byte aligned", who);
    a.layers = layers, a.pages = pages, a.Hkv = Hkv, a.page = page;
    a.Kp = static_cast<const uint8_t*>(Kp), a.Vp = static_cast<const uint8_t*>(Vp);
    a.K = static_cast<char*>(K), a.V = static_cast<char*>(V);
    if (2.0 * layers * pages * Hkv * (page / 16) >= 2147483648.0)
        return fail(YTHIP_EUNSUPPORTED, "%s: %.0f workgroups (2^31 - 1 at most)", who, 2.0 * layers * pages * Hkv * (page / 16));
    const int64_t grid = 2ll * layers * pages * Hkv * (page / 16);
    const int64_t values = (int64_t)layers * pages * Hkv * page * d, es = dtype == YTHIP_F32 ? 4 : 2;
    const Span k = span_of(K, es, {{values, 1}}), v = span_of(V, es, {{values, 1}});
    for (const void* pool : {Kp, Vp}) {
        const Span from = span_of(pool, 1, {{layers, a.ps[0]}, {pages, a.ps[1]}, {Hkv, a.ps[2]}, {block_bytes(page, d), 1}});
        if (overlap(k, from) || overlap(v, from)) return fail(YTHIP_EINVAL, "%s: K or V lies over the pools", who);
    }
    if (overlap(k, v)) return fail(YTHIP_EINVAL, "%s: K and V lie over each other", who);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T_ = decltype(t);
        // (a launch holds fewer than 2^32 threads)
        constexpr int64_t MOST = 1 << 23;
        for (a.first = 0; a.first < grid; a.first += MOST) {
            const int n = (int)std::min(grid - a.first, MOST);
            if (d == 64) cache_unpack_q4_kernel<T_, 64><<<n, 128, 0, s>>>(a);
            else cache_unpack_q4_kernel<T_, 128><<<n, 256, 0, s>>>(a);
        }
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) size_t ythip_paged_attn_q4_workspace_size(int dtype, int B, int Hq, int Hkv, int T,
                                                                                 int d, int columns, int page, int window,
                                                                                 int sinks) {
    if (B <= 0 || Hq <= 0 || Hkv <= 0 || T <= 0 || d <= 0 || columns < 0 || page <= 0 || window < 0 || sinks < 0 || Hq % Hkv != 0) return 0;
    trim_window(T, columns, page, window, sinks);
    return plan_q4(dtype, B, Hkv, Hq / Hkv, T, d, columns, page, window, sinks).bytes();
}

__attribute__((visibility("default"))) int ythip_paged_attn_q4(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[2], int pages, int page, const int32_t* table, int64_t ld_table, int columns,
    const int32_t* kv_len, const int32_t* parents, int64_t ld_parents, const int32_t* new_len, int window, int sinks,
    void* O, const int64_t o_str[3], float scale, void* workspace_, size_t ws_bytes, void* stream) {
    const char* who = "ythip_paged_attn_q4";
    PagedArgs a;
    bool done;
    if (const int e = check_window(who, window, sinks)) return e;
    // (a pool's strides are bytes here: what `prepare` makes of them is replaced below)
    const int64_t none[3] = {0, 0, 0};
    const Call c = {dtype, B, Hq, Hkv, T, d, Q, q_str, Kn, kn_str, Vn, vn_str, Kp, Vp, pool_str ? none : nullptr, pages, page,
                    table, ld_table, columns, kv_len, parents, ld_parents, new_len, O, o_str, scale};
    const int st = prepare(who, c, a, done);
    if (st || done) return st;
    int64_t ps[3] = {0, 0, 0};
    const int64_t str[3] = {0, pool_str[0], pool_str[1]};
    if (columns > 0) {
        if (const int e = check_blocks(who, 1, pages, Hkv, page, d, Kp, Vp, str, ps)) return e;
    } else {
        a.pages = 0;  // the pools may be NULL
    }
    a.ps[0] = ps[1], a.ps[1] = ps[2], a.ps[2] = 0;
    trim_window(T, columns, page, window, sinks);
    a.window = window, a.sinks = sinks;
    const Plan p = plan_q4(dtype, B, Hkv, a.G, T, d, columns, page, window, sinks);
    if (const int e = check_workspace(who, p.bytes(), workspace_, ws_bytes)) return e;
    if (!launchable((p.items * a.Hkv + 8) * p.row_tiles, 256))
        return fail(YTHIP_EUNSUPPORTED, "%s: %lld workgroups (2^24 - 1 at most)", who, (long long)(p.items * a.Hkv * p.row_tiles));
    a.target = p.target, a.stage = p.stage, a.items = (int)p.items, a.row_tiles = p.row_tiles, a.even = p.even, a.short_run = p.short_run;
    char* w = static_cast<char*>(workspace_);
    a.part = reinterpret_cast<float*>(w);
    a.part_ml = reinterpret_cast<float*>(w + p.part_bytes);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T_ = decltype(t);
        if (window > 0) return d == 64 ? run_q4<T_, 64, true>(a, p, s) : run_q4<T_, 128, true>(a, p, s);
        return d == 64 ? run_q4<T_, 64, false>(a, p, s) : run_q4<T_, 128, false>(a, p, s);
    };
    if (dtype == YTHIP_F32) return run(F32{});
    if (dtype == YTHIP_F16) return run(F16{});
    return run(BF16{});
}

}  // extern "C"
