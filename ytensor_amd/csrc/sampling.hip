// sampling.hip — the end of a drafted step for gfx950 (include/ythip.h): probabilities of the vocabulary from
// logits (ythip_token_probs), and which drafted tokens are kept (ythip_verify_drafts).

#include <algorithm>
#include <climits>
#include <cmath>

#include "launch.hpp"

namespace ythip {
namespace {

// ---------------------------------------------------------------------------
// softmax(logits / temperature)
// ---------------------------------------------------------------------------

struct ProbsArgs {
    int rows, n, parts, run;  // columns; workgroups of a row; columns of a workgroup, a multiple of 8
    const void* x;
    int64_t ld, ld_out;
    float scale;  // log2(e) / temperature
    float scale_low;  // what scale lacks to it
    float* p;
    float* part;  // [rows][parts] of (max, sum)
};

// 2^((x - top) scale) with the product's rounding put back: a logit 30 below the largest is else off by 2^-19.
__device__ __forceinline__ float weight(float x, float top, float scale, float low) {
    const float d = x - top, t = d * scale, rest = fmaf(d, scale, -t) + d * low;
    const float w = __builtin_amdgcn_exp2f(t);
    // (below 2^-126 the product has nothing to put back, and -inf has none)
    return t > -126.f ? fmaf(w, rest * 0.6931471805599453f, w) : t == t ? w : t;
}

template <class T>
struct Eight {  // 8 neighbouring logits
    static constexpr int W = std::is_same_v<T, F32> ? 2 : 1;
    u32x4 w[W];
    __device__ __forceinline__ void load(const void* x, int64_t at) {
        const char* p = static_cast<const char*>(x) + at * sizeof(typename T::raw);
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = *reinterpret_cast<const u32x4_any*>(p + 16 * i);
    }
    __device__ __forceinline__ float operator[](int i) const {
        if constexpr (std::is_same_v<T, F32>) return __uint_as_float(w[i / 4][i % 4]);
        else return i & 1 ? hi_as_f32(T{}, w[0][i / 2]) : lo_as_f32(T{}, w[0][i / 2]);
    }
};

// (M, L) of two parts: the larger maximum, and the sums in its unit
__device__ __forceinline__ void join(float& M, float& L, float M2, float L2, float scale, float low) {
    const float top = __builtin_elementwise_maximum(M, M2);
    const float ref = top == -INFINITY ? 0.f : top;
    L = L * weight(M, ref, scale, low) + L2 * weight(M2, ref, scale, low);
    M = top;
}
template <int NT>
__device__ __forceinline__ void join_block(float& M, float& L, float (&lds)[2 * NT / 64], float scale, float low) {
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) {
        const float M2 = __shfl_xor(M, off, 64), L2 = __shfl_xor(L, off, 64);
        join(M, L, M2, L2, scale, low);
    }
    const int wave = threadIdx.x >> 6;
    if ((threadIdx.x & 63) == 0) lds[2 * wave] = M, lds[2 * wave + 1] = L;
    __syncthreads();
    M = lds[0], L = lds[1];
    for (int w = 1; w < NT / 64; ++w) join(M, L, lds[2 * w], lds[2 * w + 1], scale, low);
}

// This thread's maximum and sum over columns [c0, c1) of a row.
template <class T, int NT>
__device__ __forceinline__ void scan_row(const ProbsArgs& a, int64_t row, int c0, int c1, float& M, float& L) {
    constexpr int AHEAD = 4;
    M = -INFINITY, L = 0.f;
    const int whole = c0 + (c1 - c0) / 8 * 8;
    for (int c = c0 + (int)threadIdx.x * 8; c < whole; c += AHEAD * NT * 8) {
        Eight<T> v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u].load(a.x, row * a.ld + (c + u * NT * 8 < whole ? c + u * NT * 8 : c));
        float top = M;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
#pragma unroll
            for (int e = 0; e < 8; ++e) top = __builtin_elementwise_maximum(top, v[u][e]);
        const float ref = top == -INFINITY ? 0.f : top;
        L *= weight(M, ref, a.scale, a.scale_low);
        M = top;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (c + u * NT * 8 < whole) {
#pragma unroll
                for (int e = 0; e < 8; ++e) L += weight(v[u][e], ref, a.scale, a.scale_low);
            }
    }
    const int c = whole + (int)threadIdx.x;
    if (c < c1) join(M, L, load_as_f32<T>(a.x, row * a.ld + c), 1.f, a.scale, a.scale_low);
}
template <class T, int NT>
__device__ __forceinline__ void write_row(const ProbsArgs& a, int64_t row, int c0, int c1, float M, float L) {
    constexpr int AHEAD = 4;
    const float ref = M == -INFINITY ? 0.f : M, inv = M == -INFINITY ? 0.f : 1.0f / L;
    const int whole = c0 + (c1 - c0) / 8 * 8;
    for (int c = c0 + (int)threadIdx.x * 8; c < whole; c += AHEAD * NT * 8) {
        Eight<T> v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u].load(a.x, row * a.ld + (c + u * NT * 8 < whole ? c + u * NT * 8 : c));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (c + u * NT * 8 >= whole) break;
            float* out = a.p + row * a.ld_out + c + u * NT * 8;
#pragma unroll
            for (int q = 0; q < 2; ++q) {
                f32x4 o;
#pragma unroll
                for (int e = 0; e < 4; ++e) o[e] = weight(v[u][4 * q + e], ref, a.scale, a.scale_low) * inv;
                *reinterpret_cast<f32x4_any*>(out + 4 * q) = o;
            }
        }
    }
    const int c = whole + (int)threadIdx.x;
    if (c < c1) a.p[row * a.ld_out + c] = weight(load_as_f32<T>(a.x, row * a.ld + c), ref, a.scale, a.scale_low) * inv;
}

// Many rows: a workgroup has one, and reads it twice (the second time out of the caches).
template <class T>
__global__ __launch_bounds__(1024) void probs_row_kernel(ProbsArgs a) {
    __shared__ float lds[2 * 1024 / 64];
    const int64_t row = blockIdx.x;
    float M, L;
    scan_row<T, 1024>(a, row, 0, a.n, M, L);
    join_block<1024>(M, L, lds, a.scale, a.scale_low);
    write_row<T, 1024>(a, row, 0, a.n, M, L);
}
// Few rows: `parts` workgroups a row, whose maxima and sums the second launch joins, each workgroup for itself.
template <class T>
__global__ __launch_bounds__(256) void probs_part_kernel(ProbsArgs a) {
    __shared__ float lds[2 * 256 / 64];
    const int64_t row = blockIdx.y;
    const int c0 = blockIdx.x * a.run, c1 = min(c0 + a.run, a.n);
    float M, L;
    scan_row<T, 256>(a, row, c0, c1, M, L);
    join_block<256>(M, L, lds, a.scale, a.scale_low);
    if (threadIdx.x == 0) *reinterpret_cast<f32x2*>(a.part + 2 * (row * a.parts + blockIdx.x)) = f32x2{M, L};
}
template <class T>
__global__ __launch_bounds__(256) void probs_write_kernel(ProbsArgs a) {
    __shared__ float lds[2 * 256 / 64];
    const int64_t row = blockIdx.y;
    const int c0 = blockIdx.x * a.run, c1 = min(c0 + a.run, a.n);
    float M = -INFINITY, L = 0.f;
    for (int i = threadIdx.x; i < a.parts; i += 256) {
        const f32x2 v = *reinterpret_cast<const f32x2*>(a.part + 2 * (row * a.parts + i));
        join(M, L, v[0], v[1], a.scale, a.scale_low);
    }
    join_block<256>(M, L, lds, a.scale, a.scale_low);
    write_row<T, 256>(a, row, c0, c1, M, L);
}

constexpr int ROWS_ALONE = 192;  // rows from which a workgroup has one to itself
struct ProbsPlan {
    int parts, run;
};
ProbsPlan probs_plan(int rows, int n) {
    if (rows >= ROWS_ALONE || n <= 4096) return {1, n};
    // 512 workgroups, of at least 1024 columns each
    const int want = std::max(1, std::min((n + 1023) / 1024, (512 + rows - 1) / rows));
    const int run = ((n + want - 1) / want + 7) / 8 * 8;
    return {(n + run - 1) / run, run};
}

// ---------------------------------------------------------------------------
// The verification of drafted tokens
// ---------------------------------------------------------------------------

constexpr int MAX_DRAFTS = 1024;   // tokens of a sequence: their probabilities lie in LDS
constexpr int SLICE = 4096;        // vocabulary entries of a workgroup
constexpr int MAX_SLICES = 1024;

struct VerifyArgs {
    int B, T, V, slices;
    const void *target, *draft;
    int64_t ts[2], ds[2];  // elements
    const int32_t *tokens, *parents, *tree_len;
    int64_t ld_tok, ld_par;
    const float *u, *u_next;
    int64_t ld_u;
    int32_t *path, *kept, *next;
    int64_t ld_path;
    double* sums;  // [B][slices] of (what is left, the row as it is)
};

// What a probability weighs: one that is not a positive number has no weight.
__device__ __forceinline__ double mass(float w) { return w > 0.f && w < INFINITY ? (double)w : 0.0; }

// The tokens that are kept, worked out by one wave for itself; the others wait at the barrier. s_p: p(token | the one
// above it); s_up: the one above it, -1 where it cannot be kept.
struct Walk {
    int n, last;  // kept tokens, the last of them
    int behind;   // the chain's first refused token, whose draft row is taken off the target's (0: none)
};
template <class T>
__device__ __forceinline__ Walk walk_drafts(const VerifyArgs& a, int b, double* s_p, int16_t* s_up, int32_t* s_tok,
                                            int32_t* s_walk, int32_t* path) {
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    for (int t = threadIdx.x; t < tn; t += 256) {
        const int up = a.parents != nullptr ? a.parents[b * a.ld_par + t] : t - 1;
        const int x = a.tokens[b * a.ld_tok + t];
        const bool is = t > 0 && up >= 0 && up < t && x >= 0 && x < a.V;
        s_up[t] = (int16_t)(is ? up : -1);
        s_tok[t] = x;
        double p = is ? mass(load_as_f32<T>(a.target, b * a.ts[0] + up * a.ts[1] + x)) : 0.0;
        if (a.draft != nullptr) {
            // u q < p, in 64 bits without a rounding; 1 for a token that is kept
            const float q = is ? load_as_f32<T>(a.draft, b * a.ds[0] + t * a.ds[1] + x) : 0.f;
            p = is && (double)a.u[b * a.ld_u + t] * (double)q < p ? 1.0 : 0.0;
        }
        s_p[t] = p;
    }
    __syncthreads();
    if (a.draft == nullptr) {
        // of siblings with one token the first has its probability
        for (int t = threadIdx.x; t < tn; t += 256) {
            bool twice = false;
            for (int o = 1; o < t && !twice; ++o) twice = s_up[o] == s_up[t] && s_tok[o] == s_tok[t];
            if (twice && s_up[t] >= 0) s_p[t] = 0.0;
        }
        __syncthreads();
    }
    if (threadIdx.x < 64) {
        const int lane = threadIdx.x;
        int cur = 0, n = tn > 0 ? 1 : 0, behind = 0;
        if (path != nullptr && lane == 0 && tn > 0) path[0] = 0;
        if (a.draft != nullptr) {
            for (int t = 1; t < tn; ++t) {
                if (!(s_p[t] > 0.0)) {
                    behind = t;
                    break;
                }
                cur = t;
                if (path != nullptr && lane == 0) path[n] = t;
                ++n;
            }
        } else {
            double low = 0.0, x = 0.0;
            for (int base = 0; base < tn; base += 64) {
                const int t = base + lane;
                const bool real = t < tn;
                const int up = real ? s_up[t] : -1;
                const double p = real ? s_p[t] : 0.0;
                const float u = real ? a.u[b * a.ld_u + t] : 0.f;
                if (base == 0) x = (double)__shfl(u, 0, 64);
                // a token's children come after it: what is left of these 64, child by child
                uint64_t left = ~0ull;
                for (;;) {
                    const uint64_t is = __ballot(up == cur) & left;
                    if (is == 0) break;
                    const int at = __builtin_ctzll(is);
                    const double high = low + __shfl(p, at, 64);
                    left = at == 63 ? 0 : ~0ull << (at + 1);
                    if (x >= low && x < high) {
                        cur = base + at;
                        if (path != nullptr && lane == 0) path[n] = cur;
                        ++n;
                        low = 0.0;
                        x = (double)__shfl(u, at, 64);
                    } else {
                        low = high;
                    }
                }
            }
        }
        if (lane == 0) s_walk[0] = n, s_walk[1] = cur, s_walk[2] = behind;
        if (path != nullptr)
            for (int t = n + lane; t < a.T; t += 64) path[t] = -1;
    }
    __syncthreads();
    return {s_walk[0], s_walk[1], s_walk[2]};
}

// The weights of eight entries of the row that the next token comes from, as it is and after what was refused.
template <class T>
struct Weights {
    float p[8], q[8];
    __device__ __forceinline__ void load(const VerifyArgs& a, const void* row_p, const void* row_q, int v, int end) {
        if (v + 8 <= end) {
            Eight<T> x;
            x.load(row_p, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) p[e] = x[e], q[e] = 0.f;
            if (row_q != nullptr) {
                Eight<T> y;
                y.load(row_q, v);
#pragma unroll
                for (int e = 0; e < 8; ++e) q[e] = y[e];
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                p[e] = v + e < end ? load_as_f32<T>(row_p, v + e) : 0.f;
                q[e] = v + e < end && row_q != nullptr ? load_as_f32<T>(row_q, v + e) : 0.f;
            }
        }
    }
    __device__ __forceinline__ double whole(int e) const { return mass(p[e]); }
    // `gone`: bit e of an entry that a refused child has taken
    __device__ __forceinline__ double left(int e, uint32_t gone) const {
        if (gone >> e & 1) return 0.0;
        const double w = mass(p[e]) - mass(q[e]);
        return w > 0.0 ? w : 0.0;
    }
};

// Bits of a slice's entries that are children's tokens of the last token that was kept.
__device__ __forceinline__ void mark_children(const Walk& w, int tn, const int16_t* s_up, const int32_t* s_tok, int v0,
                                              uint32_t* s_gone) {
    for (int i = threadIdx.x; i < SLICE / 32; i += 256) s_gone[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < tn; t += 256) {
        const int v = s_tok[t] - v0;
        if (s_up[t] == w.last && v >= 0 && v < SLICE) atomicOr(&s_gone[v / 32], 1u << (v % 32));
    }
    __syncthreads();
}

template <class T>
struct Rows {
    const void *p, *q;
    __device__ __forceinline__ Rows(const VerifyArgs& a, int b, const Walk& w) {
        using raw = typename T::raw;
        p = static_cast<const raw*>(a.target) + b * a.ts[0] + w.last * a.ts[1];
        q = a.draft != nullptr && w.behind > 0 ? static_cast<const raw*>(a.draft) + b * a.ds[0] + w.behind * a.ds[1] : nullptr;
    }
};

// A slice's sums of both weights. Every workgroup of a sequence walks its drafts by itself: the T probabilities are
// loads that lie side by side, and a launch would cost more. Sums are in 64 bits: which entry the random number falls on
// does not depend on how 150000 numbers of 24 bits were added up. Bound by the round trips (lengths, tokens, their
// probabilities, a slice).
template <class T>
__global__ __launch_bounds__(256) void verify_sum_kernel(VerifyArgs a) {
    __shared__ double s_p[MAX_DRAFTS];
    __shared__ int32_t s_tok[MAX_DRAFTS], s_walk[3];
    __shared__ int16_t s_up[MAX_DRAFTS];
    __shared__ uint32_t s_gone[SLICE / 32];
    __shared__ double s_sum[4][2];
    const int b = blockIdx.y, v0 = blockIdx.x * SLICE, end = min(v0 + SLICE, a.V);
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    int32_t* path = blockIdx.x == 0 ? a.path + b * a.ld_path : nullptr;
    const Walk w = walk_drafts<T>(a, b, s_p, s_up, s_tok, s_walk, path);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.kept[b] = w.n;
    if (w.n == 0) {
        if (blockIdx.x == 0 && threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    const Rows<T> rows(a, b, w);
    Weights<T> x[SLICE / 2048];
#pragma unroll
    for (int i = 0; i < SLICE / 2048; ++i) x[i].load(a, rows.p, rows.q, min(v0 + i * 2048 + (int)threadIdx.x * 8, end), end);
    if (a.draft == nullptr) mark_children(w, tn, s_up, s_tok, v0, s_gone);
    double left = 0.0, whole = 0.0;
#pragma unroll
    for (int i = 0; i < SLICE / 2048; ++i) {
        const int at = i * 2048 + threadIdx.x * 8;
        const uint32_t gone = a.draft == nullptr ? s_gone[at / 32] >> (at % 32) : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) left += x[i].left(e, gone), whole += x[i].whole(e);
    }
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) left += __shfl_xor(left, off, 64), whole += __shfl_xor(whole, off, 64);
    if ((threadIdx.x & 63) == 0) s_sum[threadIdx.x >> 6][0] = left, s_sum[threadIdx.x >> 6][1] = whole;
    __syncthreads();
    if (threadIdx.x < 2) {
        double t = 0.0;
        for (int i = 0; i < 4; ++i) t += s_sum[i][threadIdx.x];
        a.sums[2 * ((int64_t)b * a.slices + blockIdx.x) + threadIdx.x] = t;
    }
}

// Sum of v over the threads before this one, and over all 256.
__device__ __forceinline__ double scan256(double v, double* lds, double& total) {
    double inc = v;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double x = __shfl_up(inc, off, 64);
        if (lane >= off) inc += x;
    }
    __syncthreads();  // the last call's totals are read
    if (lane == 63) lds[wave] = inc;
    __syncthreads();
    double before = 0.0;
    for (int w = 0; w < wave; ++w) before += lds[w];
    total = ((lds[0] + lds[1]) + lds[2]) + lds[3];
    return before + (inc - v);
}

// The next token: the slice that the random number falls on by the slices' sums, then the entry. A number that the
// sums' own rounding leaves behind the last entry takes the last with a weight.
template <class T>
__global__ __launch_bounds__(256) void verify_pick_kernel(VerifyArgs a) {
    __shared__ double s_p[MAX_DRAFTS];
    __shared__ int32_t s_tok[MAX_DRAFTS], s_walk[3];
    __shared__ int16_t s_up[MAX_DRAFTS];
    __shared__ uint32_t s_gone[SLICE / 32];
    __shared__ double s_scan[4], s_base;
    __shared__ int s_first, s_last;
    const int b = blockIdx.x;
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    const Walk w = walk_drafts<T>(a, b, s_p, s_up, s_tok, s_walk, nullptr);
    if (w.n == 0) return;
    constexpr int PER = MAX_SLICES / 256;
    const double* sums = a.sums + 2 * (int64_t)b * a.slices;
    double mine[PER][2], left = 0.0, whole = 0.0, total, before;
#pragma unroll
    for (int i = 0; i < PER; ++i) {
        const int at = (int)threadIdx.x * PER + i;
        mine[i][0] = at < a.slices ? sums[2 * at] : 0.0;
        mine[i][1] = at < a.slices ? sums[2 * at + 1] : 0.0;
        left += mine[i][0], whole += mine[i][1];
    }
    int which = 0;
    before = scan256(left, s_scan, total);
    if (!(total > 0.0)) {
        // nothing is left (the draft's row is the target's, up to its rounding): the row as it is
        which = 1;
        before = scan256(whole, s_scan, total);
        if (!(total > 0.0)) {
            if (threadIdx.x == 0) a.next[b] = -1;
            return;
        }
    }
    // the first place where the sum passes x, and the last that adds to it
    const double x = (double)a.u_next[b] * total;
    auto search = [&](double sum, auto weight, int n) {
        if (threadIdx.x == 0) s_first = INT_MAX, s_last = -1;
        __syncthreads();
        int first = INT_MAX, last = -1;
        double at_first = 0.0, at_last = 0.0;
        for (int i = 0; i < n; ++i) {
            const double m = weight(i);
            if (m > 0.0) {
                last = (int)threadIdx.x * n + i, at_last = sum;
                if (first == INT_MAX && sum + m > x) first = last, at_first = sum;
            }
            sum += m;
        }
        if (first != INT_MAX) atomicMin(&s_first, first);
        if (last >= 0) atomicMax(&s_last, last);
        __syncthreads();
        const int at = s_first != INT_MAX ? s_first : s_last;
        if (at == first) s_base = at_first;
        else if (at == last) s_base = at_last;
        __syncthreads();
        return at;
    };
    const int slice = search(before, [&](int i) { return which ? mine[i][1] : mine[i][0]; }, PER);
    const double base = s_base;
    const int v0 = slice * SLICE, end = min(v0 + SLICE, a.V);
    if (a.draft == nullptr) mark_children(w, tn, s_up, s_tok, v0, s_gone);
    const Rows<T> rows(a, b, w);
    constexpr int EACH = SLICE / 256;
    double m[EACH], sum = 0.0;
#pragma unroll
    for (int i = 0; i < EACH / 8; ++i) {
        const int at = (int)threadIdx.x * EACH + i * 8;
        Weights<T> y;
        y.load(a, rows.p, rows.q, min(v0 + at, end), end);
        const uint32_t gone = a.draft == nullptr ? s_gone[at / 32] >> (at % 32) : 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            m[i * 8 + e] = which ? y.whole(e) : y.left(e, gone);
            sum += m[i * 8 + e];
        }
    }
    before = scan256(sum, s_scan, total);
    const int at = search(base + before, [&](int i) { return m[i]; }, EACH);
    if (threadIdx.x == 0) a.next[b] = at >= 0 ? v0 + at : -1;
}

size_t verify_bytes(int B, int V) {
    return B > 0 && V > 0 ? (size_t)B * ((V + SLICE - 1) / SLICE) * 2 * sizeof(double) : 0;
}

}  // namespace
}  // namespace ythip

using namespace ythip;

extern "C" {

__attribute__((visibility("default"))) size_t ythip_token_probs_workspace_size(int rows, int n) {
    if (rows <= 0 || n <= 0) return 0;
    const ProbsPlan p = probs_plan(rows, n);
    return p.parts > 1 ? (size_t)rows * p.parts * 2 * sizeof(float) : 0;
}

__attribute__((visibility("default"))) int ythip_token_probs(int dtype, int rows, int n, const void* logits, int64_t ld,
                                                             float temperature, float* probs, int64_t ld_out,
                                                             void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "ythip_token_probs";
    if (dtype != YTHIP_F32 && dtype != YTHIP_F16 && dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, dtype);
    if (rows < 0 || n < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    if (!(temperature > 0.f) || !(temperature < INFINITY)) return fail(YTHIP_EINVAL, "%s: temperature %g (a positive number)", who, temperature);
    if (rows == 0 || n == 0) return 0;
    if (n > 1 << 30) return fail(YTHIP_EUNSUPPORTED, "%s: %d logits a row (2^30 at most)", who, n);
    if (!logits || !probs) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if (rows > 1 && (ld < n || ld_out < n))
        return fail(YTHIP_EINVAL, "%s: rows of %d at strides of %lld and %lld", who, n, (long long)ld, (long long)ld_out);
    const uintptr_t es = dtype == YTHIP_F32 ? 4 : 2;
    if ((uintptr_t)logits % es != 0 || (uintptr_t)probs % 4 != 0) return fail(YTHIP_EINVAL, "%s: an address within an element", who);
    const ProbsPlan p = probs_plan(rows, n);
    if (!launchable(rows, 1024)) return fail(YTHIP_EUNSUPPORTED, "%s: %d rows (2^22 - 1 at most)", who, rows);
    const size_t need = ythip_token_probs_workspace_size(rows, n);
    if (need > 0 && (workspace == nullptr || ws_bytes < need || ((uintptr_t)workspace & 7) != 0))
        return fail(YTHIP_EINVAL, "%s: needs an 8-byte aligned workspace of %zu bytes, got %zu", who, need, ws_bytes);
    const double scale = 1.4426950408889634 / (double)temperature;
    if (!(scale < 1e38) || !(scale > 1e-37)) return fail(YTHIP_EUNSUPPORTED, "%s: temperature %g", who, temperature);
    const ProbsArgs a = {rows, n, p.parts, p.run, logits, ld, ld_out, (float)scale, (float)(scale - (double)(float)scale), probs,
                         static_cast<float*>(workspace)};
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T = decltype(t);
        if (p.parts == 1) {
            probs_row_kernel<T><<<rows, 1024, 0, s>>>(a);
            return;
        }
        probs_part_kernel<T><<<dim3(p.parts, rows), 256, 0, s>>>(a);
        probs_write_kernel<T><<<dim3(p.parts, rows), 256, 0, s>>>(a);
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

__attribute__((visibility("default"))) size_t ythip_verify_drafts_workspace_size(int B, int V) { return verify_bytes(B, V); }

__attribute__((visibility("default"))) int ythip_verify_drafts(
    int dtype, int B, int T, int V, const void* target, const int64_t target_str[2], const void* draft,
    const int64_t draft_str[2], const int32_t* tokens, int64_t ld_tokens, const int32_t* parents, int64_t ld_parents,
    const int32_t* tree_len, const float* u, int64_t ld_u, const float* u_next, int32_t* path, int64_t ld_path,
    int32_t* kept, int32_t* next, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "ythip_verify_drafts";
    if (dtype != YTHIP_F32 && dtype != YTHIP_F16 && dtype != YTHIP_BF16) return fail(YTHIP_EINVAL, "%s: invalid dtype %d", who, dtype);
    if (B < 0 || T < 0 || V < 0) return fail(YTHIP_EINVAL, "%s: negative size", who);
    if (B == 0) return 0;
    if (T == 0 || V == 0) return fail(YTHIP_EINVAL, "%s: %d tokens, a vocabulary of %d", who, T, V);
    if (T > MAX_DRAFTS) return fail(YTHIP_EUNSUPPORTED, "%s: %d tokens a sequence (at most %d)", who, T, MAX_DRAFTS);
    if (V > MAX_SLICES * SLICE) return fail(YTHIP_EUNSUPPORTED, "%s: a vocabulary of %d (at most %d)", who, V, MAX_SLICES * SLICE);
    if (B > 65535) return fail(YTHIP_EUNSUPPORTED, "%s: %d sequences (at most 65535)", who, B);
    if (!target || !target_str || !tokens || !u || !u_next || !path || !kept || !next) return fail(YTHIP_EINVAL, "%s: NULL argument", who);
    if (draft && parents) return fail(YTHIP_EINVAL, "%s: draft probabilities are those of a chain: no parents", who);
    if (draft && !draft_str) return fail(YTHIP_EINVAL, "%s: draft without strides", who);
    if (ld_tokens < T || ld_u < T || ld_path < T || (parents && ld_parents < T))
        return fail(YTHIP_EINVAL, "%s: rows of %d tokens at strides of %lld, %lld, %lld, %lld", who, T, (long long)ld_tokens,
                    (long long)ld_u, (long long)ld_path, (long long)ld_parents);
    const uintptr_t es = dtype == YTHIP_F32 ? 4 : 2;
    if ((uintptr_t)target % es != 0 || (uintptr_t)draft % es != 0) return fail(YTHIP_EINVAL, "%s: an address within an element", who);
    const size_t need = verify_bytes(B, V);
    if (workspace == nullptr || ws_bytes < need || ((uintptr_t)workspace & 7) != 0)
        return fail(YTHIP_EINVAL, "%s: needs an 8-byte aligned workspace of %zu bytes, got %zu", who, need, ws_bytes);
    VerifyArgs a;
    a.B = B, a.T = T, a.V = V, a.slices = (V + SLICE - 1) / SLICE;
    a.target = target, a.draft = draft;
    for (int i = 0; i < 2; ++i) {
        a.ts[i] = (i == 0 ? B : T) > 1 ? target_str[i] : 0;
        a.ds[i] = draft && (i == 0 ? B : T) > 1 ? draft_str[i] : 0;
    }
    a.tokens = tokens, a.parents = parents, a.tree_len = tree_len, a.ld_tok = ld_tokens, a.ld_par = ld_parents;
    a.u = u, a.u_next = u_next, a.ld_u = ld_u, a.path = path, a.ld_path = ld_path, a.kept = kept, a.next = next;
    a.sums = static_cast<double*>(workspace);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T_ = decltype(t);
        verify_sum_kernel<T_><<<dim3(a.slices, B), 256, 0, s>>>(a);
        verify_pick_kernel<T_><<<B, 256, 0, s>>>(a);
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

}  // extern "C"
