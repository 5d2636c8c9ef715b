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

// A part of a row. Its sum is of up to 2^30 weights: eight are added in 32 bits, those in 64 (256 rows of 151936: 0.8e-7 of a
// probability, that of its own roundings; with sums in 32 bits and parts joined two by two, their lower one brought to the
// other's unit each time, up to 3.4e-7: an exponential's error is not centred).
struct Part {
    double sum;
    float max;
};

struct ProbsArgs {
    int rows, n, parts, run;  // columns; workgroups of a row; columns of a workgroup, a multiple of 8
    const void* x;
    int64_t ld, ld_out;
    float scale;  // log2(e) / temperature
    float scale_low;  // what scale lacks to it
    float least;      // -200 / scale: what lies further below the largest has no weight in 32 bits
    float* p;
    Part* part;  // [rows][parts]
};

// 2^((x - top) scale) with the product's rounding put back: a logit 30 below the largest is else off by 2^-19. 0 for an x
// of -inf; where x or top is NaN or +inf the row is NaN, which its maximum says (see inverse).
__device__ __forceinline__ float weight(const ProbsArgs& a, float x, float top) {
    const float d = __builtin_fmaxf(x - top, a.least), t = d * a.scale;
    const float rest = fmaf(d, a.scale_low, fmaf(d, a.scale, -t));
    const float w = __builtin_amdgcn_exp2f(t);
    return fmaf(w, rest * 0.6931471805599453f, w);
}
__device__ __forceinline__ float finite(float top) { return top == -INFINITY ? 0.f : top; }

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
    // (the compiler keeps no converted logits from one pass for the next: they take twice the registers)
    __device__ __forceinline__ void again() {
#pragma unroll
        for (int i = 0; i < W; ++i) asm volatile("" : "+v"(w[i]));
    }
};

// (M, L) of two parts: the larger maximum, and the sums in its unit
__device__ __forceinline__ void join(const ProbsArgs& a, float& M, double& L, float M2, double L2) {
    const float top = __builtin_elementwise_maximum(M, M2), ref = finite(top);
    L = L * (double)weight(a, M, ref) + L2 * (double)weight(a, M2, ref);
    M = top;
}
// Over a wave, then a workgroup: the largest maximum first, so that a sum is brought to another unit twice.
template <int NT>
__device__ __forceinline__ void join_block(const ProbsArgs& a, float& M, double& L, Part (&lds)[NT / 64]) {
    float top = M;
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) top = __builtin_elementwise_maximum(top, __shfl_xor(top, off, 64));
    L *= (double)weight(a, M, finite(top));
#pragma unroll
    for (int off = 32; off >= 1; off >>= 1) L += __shfl_xor(L, off, 64);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = {L, top};
    __syncthreads();
    // lane l has wave l % (NT / 64)
    const Part mine = lds[threadIdx.x % (NT / 64)];
    M = mine.max;
#pragma unroll
    for (int off = NT / 128; off >= 1; off >>= 1) M = __builtin_elementwise_maximum(M, __shfl_xor(M, off, 64));
    L = mine.sum * (double)weight(a, mine.max, finite(M));
#pragma unroll
    for (int off = NT / 128; off >= 1; off >>= 1) L += __shfl_xor(L, off, 64);
}
// The sum of eight neighbouring logits' weights
template <class T>
__device__ __forceinline__ double sum_eight(const ProbsArgs& a, const Eight<T>& v, float ref) {
    float w[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) w[e] = weight(a, v[e], ref);
    return (double)(((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7])));
}

// This thread's maximum and sum over columns [c0, c1) of a row.
template <class T, int NT>
__device__ __forceinline__ void scan_row(const ProbsArgs& a, int64_t row, int c0, int c1, float& M, double& L) {
    constexpr int AHEAD = 4;
    M = -INFINITY, L = 0.0;
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
        const float ref = finite(top);
        L *= (double)weight(a, M, ref);
        M = top;
#pragma unroll
        for (int u = 0; u < AHEAD; ++u)
            if (c + u * NT * 8 < whole) L += sum_eight<T>(a, v[u], ref);
    }
    const int c = whole + (int)threadIdx.x;
    if (c < c1) join(a, M, L, load_as_f32<T>(a.x, row * a.ld + c), 1.0);
}

// Eight probabilities from their logits.
template <class T>
__device__ __forceinline__ void write_eight(const ProbsArgs& a, const Eight<T>& v, int64_t at, float ref, float inv) {
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        f32x4 o;
#pragma unroll
        for (int e = 0; e < 4; ++e) o[e] = weight(a, v[4 * q + e], ref) * inv;
        *reinterpret_cast<f32x4_any*>(a.p + at + 4 * q) = o;
    }
}
// 1 / the sum; 0 for a row of -inf, NaN for one with a NaN or +inf
__device__ __forceinline__ float inverse(float M, double L) {
    return M == -INFINITY ? 0.f : M < INFINITY ? (float)(1.0 / L) : __builtin_nanf("");
}
template <class T, int NT>
__device__ __forceinline__ void write_row(const ProbsArgs& a, int64_t row, int c0, int c1, float ref, float inv) {
    constexpr int AHEAD = 4;
    const int whole = c0 + (c1 - c0) / 8 * 8;
    for (int c = c0 + (int)threadIdx.x * 8; c < whole; c += AHEAD * NT * 8) {
        Eight<T> v[AHEAD];
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) v[u].load(a.x, row * a.ld + (c + u * NT * 8 < whole ? c + u * NT * 8 : c));
#pragma unroll
        for (int u = 0; u < AHEAD; ++u) {
            if (c + u * NT * 8 >= whole) break;
            write_eight<T>(a, v[u], row * a.ld_out + c + u * NT * 8, ref, inv);
        }
    }
    const int c = whole + (int)threadIdx.x;
    if (c < c1) a.p[row * a.ld_out + c] = weight(a, load_as_f32<T>(a.x, row * a.ld + c), ref) * inv;
}

// Many rows: a workgroup has one. What of it the registers hold is read once (HELD times 8 columns a thread: 155648 columns
// of 16 bits, 73728 of 32), and all of that is on its way before the first maximum; the rest is read twice. Bound by
// memory: 256 rows of 151936 bfloat16 49.6 us, 4.7 TB/s (read twice, and a weight of eleven operations where it has eight:
// 73; with the workgroup's maximum before any sum, a barrier more: 55).
template <class T>
__global__ __launch_bounds__(1024) void probs_row_kernel(ProbsArgs a) {
    constexpr int NT = 1024, HELD = std::is_same_v<T, F32> ? 9 : 19;
    __shared__ Part lds[NT / 64];
    const int64_t row = blockIdx.x;
    const int held = min(a.n / 8, HELD * NT) * 8;
    Eight<T> v[HELD];
    float M;
    double L;
#pragma unroll
    for (int u = 0; u < HELD; ++u)
        if (u * NT * 8 < held) v[u].load(a.x, row * a.ld + min((u * NT + (int)threadIdx.x) * 8, held - 8));
    scan_row<T, NT>(a, row, held, a.n, M, L);
    float top = M;
#pragma unroll
    for (int u = 0; u < HELD; ++u)
        if (u * NT * 8 < held) {
#pragma unroll
            for (int e = 0; e < 8; ++e) top = __builtin_elementwise_maximum(top, v[u][e]);
        }
    float ref = finite(top);
    L *= (double)weight(a, M, ref);
    M = top;
#pragma unroll
    for (int u = 0; u < HELD; ++u)
        if ((u * NT + (int)threadIdx.x) * 8 < held) {
            v[u].again();
            L += sum_eight<T>(a, v[u], ref);
        }
    join_block<NT>(a, M, L, lds);
    ref = finite(M);
    const float inv = inverse(M, L);
#pragma unroll
    for (int u = 0; u < HELD; ++u)
        if ((u * NT + (int)threadIdx.x) * 8 < held) {
            v[u].again();
            write_eight<T>(a, v[u], row * a.ld_out + (u * NT + (int)threadIdx.x) * 8, ref, inv);
        }
    write_row<T, NT>(a, row, held, a.n, ref, inv);
}
// Few rows: `parts` workgroups a row, whose maxima and sums the second launch joins, each workgroup for itself.
template <class T>
__global__ __launch_bounds__(256) void probs_part_kernel(ProbsArgs a) {
    __shared__ Part lds[256 / 64];
    const int64_t row = blockIdx.y;
    const int c0 = blockIdx.x * a.run, c1 = min(c0 + a.run, a.n);
    float M;
    double L;
    scan_row<T, 256>(a, row, c0, c1, M, L);
    join_block<256>(a, M, L, lds);
    if (threadIdx.x == 0) a.part[row * a.parts + blockIdx.x] = {L, M};
}
template <class T>
__global__ __launch_bounds__(256) void probs_write_kernel(ProbsArgs a) {
    __shared__ Part lds[256 / 64];
    const int64_t row = blockIdx.y;
    const int c0 = blockIdx.x * a.run, c1 = min(c0 + a.run, a.n);
    float M = -INFINITY;
    double L = 0.0;
    for (int i = threadIdx.x; i < a.parts; i += 256) {
        const Part v = a.part[row * a.parts + i];
        join(a, M, L, v.max, v.sum);
    }
    join_block<256>(a, M, L, lds);
    write_row<T, 256>(a, row, c0, c1, finite(M), inverse(M, L));
}

// Rows from which a workgroup has one to itself (bfloat16, alone and in parts: 151936 columns, 128 rows 40.4 and 36.5 us,
// 192 50.3 and 55.1, 256 60.1 and 68.8; 32000 columns 14.6 and 12.7, 15.7 and 17.0, 17.2 and 18.9).
constexpr int ROWS_ALONE = 192;
struct ProbsPlan {
    int parts, run;
};
ProbsPlan probs_plan(int rows, int n) {
    if (rows >= ROWS_ALONE || n <= 4096) return {1, n};
    // 512 workgroups, of at least 1024 columns each (64 rows of 151936: 256 workgroups 23.3 us, 512 21.7, 1024 22.4)
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
constexpr int RUN = 512;           // of a wave at a time: what has a sum of its own

struct VerifyArgs {
    int B, T, V, slices, runs;
    const void *target, *draft;
    int64_t ts[2], ds[2];  // elements
    const int32_t *tokens, *parents, *tree_len;
    int64_t ld_tok, ld_par;
    const float *u, *u_next;
    int64_t ld_u;
    int32_t *path, *kept, *next;
    int64_t ld_path;
    double* sums;   // [B][2][runs]: what is left of every RUN entries, then the row as it is
    int32_t* walk;  // [B][2]: last, behind
};

// What a probability weighs: one that is not a positive number has no weight.
__device__ __forceinline__ double mass(float w) { return w > 0.f && w < INFINITY ? (double)w : 0.0; }

// The tokens that are kept, worked out by one wave for itself; the others wait at the barrier. s_p: p(token | the one
// above it); s_up: the one above it, -1 where it cannot be kept.
struct Walk {
    int n, last;  // kept tokens, the last of them
    int behind;   // the chain's first refused token, whose draft row is taken off the target's (0: none)
};
template <class T, int NT>
__device__ __forceinline__ Walk walk_drafts(const VerifyArgs& a, int b, double* s_p, int16_t* s_up, int32_t* s_tok,
                                            int32_t* s_walk, int32_t* path) {
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    for (int t = threadIdx.x; t < tn; t += NT) {
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
        for (int t = threadIdx.x; t < tn; t += NT) {
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

// Bits of `width` entries from v0 on that are children's tokens of the last token that was kept.
template <int NT>
__device__ __forceinline__ void mark_children(const Walk& w, int tn, const int16_t* s_up, const int32_t* s_tok, int v0, int width,
                                              uint32_t* s_gone) {
    for (int i = threadIdx.x; i < width / 32; i += NT) s_gone[i] = 0;
    __syncthreads();
    for (int t = threadIdx.x; t < tn; t += NT) {
        const int v = s_tok[t] - v0;
        if (s_up[t] == w.last && v >= 0 && v < width) atomicOr(&s_gone[v / 32], 1u << (v % 32));
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

// Of n numbers a lane, in the lanes' order, behind `sum`: the first at which the sum passes x, or the last that adds to
// it. `base`: the sum before it.
template <class F>
__device__ __forceinline__ int find_in_wave(F&& number, int n, double sum, double x, double& base) {
    int first = -1, last = -1;
    double at_first = 0.0, at_last = 0.0;
#pragma unroll 8
    for (int i = 0; i < n; ++i) {
        const double m = number(i);
        if (m > 0.0) {
            last = i, at_last = sum;
            if (first < 0 && sum + m > x) first = i, at_first = sum;
        }
        sum += m;
    }
    const uint64_t hit = __ballot(first >= 0), some = __ballot(last >= 0);
    const int lane = hit != 0 ? __builtin_ctzll(hit) : 63 - __builtin_clzll(some | 1);
    base = __shfl(hit != 0 ? at_first : at_last, lane, 64);
    return lane * n + __shfl(hit != 0 ? first : last, lane, 64);
}
__device__ __forceinline__ double before_in_wave(double v, double& total) {
    double inc = v;
    const int lane = threadIdx.x & 63;
#pragma unroll
    for (int off = 1; off < 64; off <<= 1) {
        const double x = __shfl_up(inc, off, 64);
        if (lane >= off) inc += x;
    }
    total = __shfl(inc, 63, 64);
    const double x = __shfl_up(inc, 1, 64);
    return lane > 0 ? x : 0.0;
}

// A slice's sums of both weights. Every workgroup of a sequence walks its drafts by itself: the T probabilities are
// loads that lie side by side, and a launch would cost more. Bound by the round trips (lengths, tokens, their
// probabilities, a slice).
template <class T>
__global__ __launch_bounds__(256) void verify_sum_kernel(VerifyArgs a) {
    __shared__ double s_p[MAX_DRAFTS];
    __shared__ int32_t s_tok[MAX_DRAFTS], s_walk[3];
    __shared__ int16_t s_up[MAX_DRAFTS];
    __shared__ uint32_t s_gone[SLICE / 32];
    const int b = blockIdx.y, v0 = blockIdx.x * SLICE;
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    int32_t* path = blockIdx.x == 0 ? a.path + b * a.ld_path : nullptr;
    const Walk w = walk_drafts<T, 256>(a, b, s_p, s_up, s_tok, s_walk, path);
    if (blockIdx.x == 0 && threadIdx.x == 0) a.kept[b] = w.n;
    if (w.n == 0) {
        if (blockIdx.x == 0 && threadIdx.x == 0) a.next[b] = -1;
        return;
    }
    if (blockIdx.x == 0 && threadIdx.x == 0) {
        a.walk[2 * b] = w.last, a.walk[2 * b + 1] = w.behind;
    }
    const Rows<T> rows(a, b, w);
    constexpr int EACH = SLICE / (4 * RUN);  // runs of a wave
    const int lane = threadIdx.x & 63, run0 = (blockIdx.x * 4 + (threadIdx.x >> 6)) * EACH;
    Weights<T> x[EACH];
#pragma unroll
    for (int i = 0; i < EACH; ++i) x[i].load(a, rows.p, rows.q, min((run0 + i) * RUN + lane * 8, a.V), a.V);
    if (a.draft == nullptr) mark_children<256>(w, tn, s_up, s_tok, v0, SLICE, s_gone);
#pragma unroll
    for (int i = 0; i < EACH; ++i) {
        if (run0 + i >= a.runs) break;
        const int at = (run0 + i) * RUN + lane * 8 - v0;
        const uint32_t gone = a.draft == nullptr ? s_gone[at / 32] >> (at % 32) : 0;
        double left = 0.0, whole = 0.0;
#pragma unroll
        for (int e = 0; e < 8; ++e) left += x[i].left(e, gone), whole += x[i].whole(e);
#pragma unroll
        for (int off = 32; off >= 1; off >>= 1) left += __shfl_xor(left, off, 64), whole += __shfl_xor(whole, off, 64);
        if (lane == 0) {
            double* out = a.sums + (int64_t)b * 2 * a.runs + run0 + i;
            out[0] = left, out[a.runs] = whole;
        }
    }
}

// The next token, by one wave a sequence: the run that the random number falls on by the runs' sums, then the entry, the
// run read again. A number that the sums' own rounding leaves behind the last entry takes the last with a weight. Three
// round trips (the walk's end and the first sums, the row, the token): as a workgroup that walked by itself and searched
// whole slices, 13 us for 16 trees of 16.
template <class T>
__global__ __launch_bounds__(64) void verify_pick_kernel(VerifyArgs a) {
    const int b = blockIdx.x, lane = threadIdx.x;
    const int tn = a.tree_len != nullptr ? min(max(a.tree_len[b], 0), a.T) : a.T;
    if (tn == 0) {
        if (lane == 0) a.next[b] = -1;
        return;
    }
    const Walk w = {1, a.walk[2 * b], a.walk[2 * b + 1]};
    const float u = a.u_next[b];
    // lane l has `per` runs in a row
    const int per = (a.runs + 63) / 64;
    const double* sums = a.sums + (int64_t)b * 2 * a.runs;
    double before, total;
    int which = 0;
    auto sum_of = [&](const double* from) {
        double sum = 0.0;
        for (int i = 0; i < per; ++i) sum += lane * per + i < a.runs ? from[lane * per + i] : 0.0;
        before = before_in_wave(sum, total);
    };
    sum_of(sums);
    if (!(total > 0.0)) {
        // nothing is left (the draft's row is the target's, up to its rounding): the row as it is
        which = 1;
        sums += a.runs;
        sum_of(sums);
        if (!(total > 0.0)) {
            if (lane == 0) a.next[b] = -1;
            return;
        }
    }
    const double x = (double)u * total;
    double base, unused;
    const int run = find_in_wave([&](int i) { return lane * per + i < a.runs ? sums[lane * per + i] : 0.0; }, per, before, x, base);
    const Rows<T> rows(a, b, w);
    const int v = run * RUN + lane * 8;
    Weights<T> y;
    y.load(a, rows.p, rows.q, min(v, a.V), a.V);
    uint32_t gone = 0;
    if (a.draft == nullptr)
        for (int t = w.last + 1; t < tn; ++t) {
            const int up = a.parents != nullptr ? a.parents[b * a.ld_par + t] : t - 1, e = a.tokens[b * a.ld_tok + t] - v;
            if (up == w.last && e >= 0 && e < 8) gone |= 1u << e;
        }
    double m[8], sum = 0.0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        m[e] = which ? y.whole(e) : y.left(e, gone);
        sum += m[e];
    }
    before = before_in_wave(sum, total);
    const int token = run * RUN + find_in_wave([&](int i) { return m[i]; }, 8, base + before, x, unused);
    if (lane == 0) a.next[b] = token;
}

// Rows of `width` bytes at a stride of `ld`; whether two such share a byte (taken to where rows lie side by side at strides
// that differ).
struct Block {
    const void* at;
    int64_t rows, ld, width;
};
bool meet(const Block& a, const Block& b) {
    if (a.at == nullptr || b.at == nullptr || !overlap(span_of(a.at, 1, {{a.rows, a.ld}, {a.width, 1}}), span_of(b.at, 1, {{b.rows, b.ld}, {b.width, 1}}))) return false;
    if (a.rows > 1 && b.rows > 1 && a.ld != b.ld) return true;
    if (a.rows == 1 && b.rows == 1) return true;
    const int64_t ld = a.rows > 1 ? a.ld : b.ld, apart = (int64_t)((uintptr_t)b.at - (uintptr_t)a.at) % ld, off = apart < 0 ? apart + ld : apart;
    return off < a.width || ld - off < b.width;
}

size_t verify_bytes(int B, int V) {
    return B > 0 && V > 0 ? (size_t)B * (((V + RUN - 1) / RUN) * 2 * sizeof(double) + 2 * sizeof(int32_t)) : 0;
}

}  // namespace
}  // namespace ythip

using namespace ythip;

extern "C" {

__attribute__((visibility("default"))) size_t ythip_token_probs_workspace_size(int rows, int n) {
    if (rows <= 0 || n <= 0) return 0;
    const ProbsPlan p = probs_plan(rows, n);
    return p.parts > 1 ? (size_t)rows * p.parts * sizeof(Part) : 0;
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
    if (!(scale < 1e38) || !(scale > 1e-36)) return fail(YTHIP_EUNSUPPORTED, "%s: temperature %g", who, temperature);
    const Block from = {logits, rows, ld * (int64_t)es, n * (int64_t)es}, to = {probs, rows, ld_out * 4, n * 4ll};
    // (in place each element is read before it is written, by one thread)
    if (meet(from, to) && !(logits == probs && dtype == YTHIP_F32 && (rows == 1 || ld == ld_out)))
        return fail(YTHIP_EINVAL, "%s: probs lies over logits (float32 alone, element on element, may)", who);
    const ProbsArgs a = {rows, n, p.parts, p.run, logits, ld, ld_out, (float)scale, (float)(scale - (double)(float)scale), (float)(-200.0 / scale), probs,
                         static_cast<Part*>(workspace)};
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
    const Block row = {nullptr, 1, 0, B * 4ll};
    auto at = [](Block b, const void* p) { return Block{p, b.rows, b.ld, b.width}; };
    auto tokens_at = [&](const void* p, int64_t ld) { return Block{p, B, ld * 4, T * 4ll}; };
    const Block read[] = {tokens_at(tokens, ld_tokens), tokens_at(parents, ld_parents), tokens_at(u, ld_u), at(row, tree_len), at(row, u_next),
                          {workspace, 1, 0, (int64_t)need}};
    const Block written[] = {tokens_at(path, ld_path), at(row, kept), at(row, next)};
    for (const Block& w : written) {
        // (the last launch writes next[b] behind its own reads: it may be the tokens where there is one a sequence)
        const bool same = w.at == next && T == 1 && tokens == next && (B == 1 || ld_tokens == 1);
        for (const Block& x : read)
            if (meet(w, x) && !(same && x.at == tokens)) return fail(YTHIP_EINVAL, "%s: path, kept or next lies over what is read", who);
        for (const Block& x : written)
            if (&x != &w && meet(w, x)) return fail(YTHIP_EINVAL, "%s: path, kept and next lie over each other", who);
    }
    VerifyArgs a;
    a.B = B, a.T = T, a.V = V, a.slices = (V + SLICE - 1) / SLICE, a.runs = (V + RUN - 1) / RUN;
    a.target = target, a.draft = draft;
    for (int i = 0; i < 2; ++i) {
        a.ts[i] = (i == 0 ? B : T) > 1 ? target_str[i] : 0;
        a.ds[i] = draft && (i == 0 ? B : T) > 1 ? draft_str[i] : 0;
    }
    a.tokens = tokens, a.parents = parents, a.tree_len = tree_len, a.ld_tok = ld_tokens, a.ld_par = ld_parents;
    a.u = u, a.u_next = u_next, a.ld_u = ld_u, a.path = path, a.ld_path = ld_path, a.kept = kept, a.next = next;
    a.sums = static_cast<double*>(workspace);
    a.walk = reinterpret_cast<int32_t*>(a.sums + (int64_t)B * 2 * a.runs);
    hipStream_t s = static_cast<hipStream_t>(stream);
    auto run = [&](auto t) {
        using T_ = decltype(t);
        verify_sum_kernel<T_><<<dim3(a.slices, B), 256, 0, s>>>(a);
        verify_pick_kernel<T_><<<B, 64, 0, s>>>(a);
    };
    if (dtype == YTHIP_F32) run(F32{});
    else if (dtype == YTHIP_F16) run(F16{});
    else run(BF16{});
    return status_of(hipGetLastError());
}

}  // extern "C"
