// paged_attn.hip — attention of new tokens over a paged KV cache (include/ythip.h,
// ythip_paged_attn) and over the pages that a score selects (ythip_paged_attn_sparse).

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
};

__device__ __forceinline__ int rows_in_use(const PagedArgs& a, int b) {
    const int64_t cap = (int64_t)a.columns << a.shift;
    return (int)min((int64_t)max(a.kv_len[b], 0), cap);
}
__device__ __forceinline__ int new_rows(const PagedArgs& a, int b) {
    return a.new_len != nullptr ? min(max(a.new_len[b], 0), a.T) : a.T;
}

// One workgroup per (token, query head, sequence): 256 keys at a time, a thread a key for the
// scores and a thread an output element (of 256 / D key groups) for the sums.
template <class T, int D, bool SPARSE>
__global__ __launch_bounds__(256) void paged_attn_simple(PagedArgs a) {
    __shared__ float s_q[D], s_p[256], s_red[256];
    __shared__ int64_t s_v[256];
    __shared__ uint32_t s_path[MAX_TREE / 32];
    const int t = blockIdx.x, hq = blockIdx.y, b = blockIdx.z, tid = threadIdx.x, h = hq / a.G;
    const int len = rows_in_use(a, b), tn = new_rows(a, b);
    if (t >= tn) return;
    if (tid < D) s_q[tid] = load_as_f32<T>(a.Q, b * a.qs[0] + hq * a.qs[1] + t * a.qs[2] + tid);
    if (a.parents != nullptr) {
        for (int i = tid; i < MAX_TREE / 32; i += 256) s_path[i] = 0;
        __syncthreads();
        if (tid == 0)
            for (int u = t, up; u >= 0; u = up) {
                s_path[u >> 5] |= 1u << (u & 31);
                up = a.parents[b * a.ld_par + u];
                if (up < 0 || up >= u) break;
            }
    }
    __syncthreads();
    const int page = 1 << a.shift;
    const int32_t* sel = SPARSE ? a.sel + (((int64_t)b * a.Hkv + h) * a.T + t) * a.top_k : nullptr;
    const int64_t cached = SPARSE ? (int64_t)a.top_k << a.shift : len;
    const int64_t total = cached + (a.Kn != nullptr ? t + 1 : 0);
    float m = -INFINITY, l = 0.f, acc = 0.f;
    constexpr int GROUPS = 256 / D;
    const int d = tid % D, grp = tid / D;
    for (int64_t j0 = 0; j0 < total; j0 += 256) {
        const int64_t j = j0 + tid;
        const void *K = a.Kp, *V = a.Vp;
        int64_t ko = -1, vo = -1;
        if (j < cached) {
            int slot = (int)(j >> a.shift);
            if (SPARSE) slot = sel[slot];
            const int r = (int)(j & (page - 1));
            if (slot >= 0 && ((int64_t)slot << a.shift) + r < len) {
                const int p = a.table[b * a.ld_table + slot];
                if (p >= 0 && p < a.pages) ko = vo = p * a.ps[0] + h * a.ps[1] + r * a.ps[2];
            }
        } else if (j < total) {
            const int u = (int)(j - cached);
            if (a.parents == nullptr || (s_path[u >> 5] >> (u & 31) & 1)) {
                K = a.Kn, V = a.Vn;
                ko = b * a.kns[0] + h * a.kns[1] + u * a.kns[2];
                vo = b * a.vns[0] + h * a.vns[1] + u * a.vns[2];
            }
        }
        float s = -INFINITY;
        if (ko >= 0) {
            s = 0.f;
            for (int e = 0; e < D; ++e) s = fmaf(s_q[e], load_as_f32<T>(K, ko + e), s);
            s *= a.scale_log2;
        }
        s_red[tid] = s;
        __syncthreads();
        float top = m;
        for (int i = 0; i < 256; ++i) top = __builtin_elementwise_maximum(top, s_red[i]);
        const float ref = top == -INFINITY ? 0.f : top;
        const float corr = exp2f(m - ref);
        const float p = ko >= 0 ? exp2f(s - ref) : 0.f;
        s_p[tid] = p;
        s_v[tid] = vo < 0 ? -1 : (vo << 1 | (j < cached ? 0 : 1));
        __syncthreads();
        l *= corr;
        acc *= corr;
        for (int i = 0; i < 256; ++i) l += s_p[i];
        for (int i = grp; i < 256; i += GROUPS)
            if (s_v[i] >= 0) acc = fmaf(s_p[i], load_as_f32<T>(s_v[i] & 1 ? a.Vn : a.Vp, (s_v[i] >> 1) + d), acc);
        m = top;
        __syncthreads();
    }
    s_red[tid] = acc;
    __syncthreads();
    if (tid < D) {
        float o = 0.f;
        for (int g = 0; g < GROUPS; ++g) o += s_red[g * D + tid];
        store_from_f32<T>(a.O, b * a.os[0] + hq * a.os[1] + t * a.os[2] + tid, m == -INFINITY ? 0.f : o / l);
    }
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

template <class T, int D, bool SPARSE>
int run_typed(const PagedArgs& a, hipStream_t s) {
    if constexpr (SPARSE) paged_select_simple<T, D><<<dim3(a.T, a.Hkv, a.B), 256, 0, s>>>(a);
    paged_attn_simple<T, D, SPARSE><<<dim3(a.T, a.Hq, a.B), 256, 0, s>>>(a);
    return status_of(hipGetLastError());
}
template <bool SPARSE>
int run(int dtype, int d, const PagedArgs& a, hipStream_t s) {
    if (dtype == YTHIP_F32) return d == 64 ? run_typed<F32, 64, SPARSE>(a, s) : run_typed<F32, 128, SPARSE>(a, s);
    if (dtype == YTHIP_F16) return d == 64 ? run_typed<F16, 64, SPARSE>(a, s) : run_typed<F16, 128, SPARSE>(a, s);
    return d == 64 ? run_typed<BF16, 64, SPARSE>(a, s) : run_typed<BF16, 128, SPARSE>(a, s);
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
    return 0;
}

__attribute__((visibility("default"))) int ythip_paged_attn(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[3], int pages, int page, const int32_t* table, int64_t ld_table, int columns,
    const int32_t* kv_len, const int32_t* parents, int64_t ld_parents, const int32_t* new_len, void* O,
    const int64_t o_str[3], float scale, void* workspace, size_t ws_bytes, void* stream) {
    const char* who = "ythip_paged_attn";
    PagedArgs a;
    bool done;
    const Call c = {dtype, B, Hq, Hkv, T, d, Q, q_str, Kn, kn_str, Vn, vn_str, Kp, Vp, pool_str, pages, page,
                    table, ld_table, columns, kv_len, parents, ld_parents, new_len, O, o_str, scale};
    const int st = prepare(who, c, a, done);
    if (st || done) return st;
    return run<false>(dtype, d, a, static_cast<hipStream_t>(stream));
}

__attribute__((visibility("default"))) size_t ythip_paged_attn_sparse_workspace_size(int dtype, int B, int Hq, int Hkv,
                                                                                     int T, int d, int columns,
                                                                                     int page, int top_k) {
    if (B <= 0 || Hkv <= 0 || T <= 0 || columns <= 0) return 0;
    return (size_t)B * Hkv * T * columns * sizeof(double);
}

__attribute__((visibility("default"))) int ythip_paged_attn_sparse(
    int dtype, int B, int Hq, int Hkv, int T, int d, const void* Q, const int64_t q_str[3], const void* Kn,
    const int64_t kn_str[3], const void* Vn, const int64_t vn_str[3], const void* Kp, const void* Vp,
    const int64_t pool_str[3], int pages, int page, const float* sums, const int64_t sums_str[2], const int32_t* table,
    int64_t ld_table, int columns, const int32_t* kv_len, const int32_t* parents, int64_t ld_parents,
    const int32_t* new_len, int top_k, int32_t* sel, void* O, const int64_t o_str[3], float scale, void* workspace,
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
    const size_t need = ythip_paged_attn_sparse_workspace_size(dtype, B, Hq, Hkv, T, d, columns, page, top_k);
    if (need > 0 && (workspace == nullptr || ws_bytes < need || ((uintptr_t)workspace & 15) != 0))
        return fail(YTHIP_EINVAL, "%s: needs a 16-byte aligned workspace of %zu bytes, got %zu", who, need, ws_bytes);
    a.sel = sel, a.top_k = top_k, a.sums = sums, a.ss[0] = sums_str[0], a.ss[1] = sums_str[1];
    a.score = static_cast<double*>(workspace);
    return run<true>(dtype, d, a, static_cast<hipStream_t>(stream));
}

}  // extern "C"
