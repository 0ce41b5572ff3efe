// paged.hip — packed tokens of many sequences over a cache in pages: RoPE +
// append, and causal grouped-query attention.
//
// What a call covers is on the device (vva_batch): the kernels find their
// sequence in q_start, its keys in kv_len and their places in the page table,
// so the same launch serves any lengths of the same shapes.
#include "vva_internal.hpp"

namespace vva {

namespace {

#include "wave_ops.hpp"

// A sequence of the batch, kept inside the rows and the table there are.
struct Seq {
    int q0, n;          // first token row, new tokens
    int L;              // keys
};
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int s) {
    Seq r;
    r.q0 = min(max(a.q_start[s], 0), a.n_tok);
    r.n = min(max(a.q_start[s + 1], r.q0), a.n_tok) - r.q0;
    r.L = min(max(a.kv_len[s], 0), a.max_pages << a.page_shift);
    return r;
}

// The sequence whose rows hold token row n, or n_seq.  Called by whole waves.
__device__ __forceinline__ int seq_of_token(const PagedArgs& a, int n) {
    const int lane = threadIdx.x & 63;
    for (int i = 0; i < a.n_seq; i += 64) {
        const int s = min(i + lane, a.n_seq - 1);
        const uint64_t hit = __ballot(a.q_start[s] <= n && n < a.q_start[s + 1]);
        if (hit) return min(i + __ffsll((unsigned long long)hit) - 1, a.n_seq - 1);
    }
    return a.n_seq;
}

// One workgroup per token row.
__global__ void __launch_bounds__(256) paged_append_kernel(PagedAppendArgs a) {
    prefetch_kernargs<sizeof(PagedAppendArgs)>();
    const PagedArgs& p = a.p;
    const int n = blockIdx.x;
    const int s = seq_of_token(p, n);
    if (s >= p.n_seq) return;
    const Seq q = seq_of(p, s);
    if (n < q.q0 || n >= q.q0 + q.n) return;
    const int i = q.L - q.n + (n - q.q0);          // the token's index in the sequence
    const int pos = a.pos ? a.pos[n] : i;
    const int P = p.d >> 1;
    const bool in_table = pos >= 0 && pos < a.n_pos;
    const float* cs = (const float*)(a.rope + (int64_t)(in_table ? pos : 0) * a.rope_nb);
    const int page = i >= 0 ? p.table[s * p.table_stride + (i >> p.page_shift)] : -1;
    const bool live = page >= 0 && page < p.n_pages;
    const int slot = i & ((1 << p.page_shift) - 1);
    const int items = (p.Hq + 2 * p.Hkv) * P;
    for (int w = threadIdx.x; w < items; w += 256) {
        const int h = w / P, e = w - h * P;
        const float c = in_table ? cs[e] : __builtin_nanf(""), sn = in_table ? cs[e + P] : __builtin_nanf("");
        const char* src;
        char* dst;
        int st, dt;
        if (h < p.Hq) {
            src = p.q + n * p.q_nb_t + h * p.q_nb_h; st = a.q_type;
            dst = p.out + n * p.o_nb_t + h * p.o_nb_h; dt = a.qo_type;
        } else if (h < p.Hq + p.Hkv) {
            const int hk = h - p.Hq;
            src = a.k_new + n * a.k_nb_t + hk * a.k_nb_h; st = a.k_type;
            dst = p.k + page * p.k_nb_page + hk * p.k_nb_head + slot * p.k_nb_slot; dt = p.type;
        } else {
            const int hk = h - p.Hq - p.Hkv;
            src = a.v_new + n * a.v_nb_t + hk * a.v_nb_h; st = a.v_type;
            dst = p.v + page * p.v_nb_page + hk * p.v_nb_head + slot * p.v_nb_slot; dt = p.type;
        }
        if (h >= p.Hq && !live) continue;
        const int es = (int)type_elem_bytes(st), ed = (int)type_elem_bytes(dt);
        const float x0 = load_elem(src + e * es, st), x1 = load_elem(src + (e + P) * es, st);
        float y0 = x0, y1 = x1;
        if (h < p.Hq + p.Hkv) {
            y0 = fmaf(x0, c, -(x1 * sn));
            y1 = fmaf(x0, sn, x1 * c);
        }
        store_elem(dst + e * ed, dt, y0);
        store_elem(dst + (e + P) * ed, dt, y1);
    }
}

// One wave per (token row, query head): the keys one after the other, the
// softmax's running maximum and sum beside the output.
template <int D>
__global__ void __launch_bounds__(256) paged_attn_kernel(PagedArgs a) {
    constexpr int E = D / 64;                      // dims per lane
    const int lane = threadIdx.x & 63;
    const int n = blockIdx.x, h = blockIdx.y * 4 + (threadIdx.x >> 6);
    if (h >= a.Hq) return;
    const int s = seq_of_token(a, n);
    if (s >= a.n_seq) return;
    const Seq q = seq_of(a, s);
    const int t = n - q.q0;
    if (t < 0 || t >= min(q.n, a.max_new)) return;
    const int last = q.L - q.n + t, kvh = h / a.G;
    float x[E], o[E] = {};
    for (int e = 0; e < E; ++e) x[e] = load_elem(a.q + n * a.q_nb_t + h * a.q_nb_h + (lane * E + e) * 2, a.type) * a.scale * kLog2e;
    float m = -INFINITY, l = 0.0f;
    for (int j = 0; j <= last; ++j) {
        const int page = a.table[s * a.table_stride + (j >> a.page_shift)];
        const int slot = j & ((1 << a.page_shift) - 1);
        if (page < 0 || page >= a.n_pages) { l = __builtin_nanf(""); continue; }
        const char* kr = a.k + page * a.k_nb_page + kvh * a.k_nb_head + slot * a.k_nb_slot + lane * E * 2;
        const char* vr = a.v + page * a.v_nb_page + kvh * a.v_nb_head + slot * a.v_nb_slot + lane * E * 2;
        float sc = 0.0f;
        for (int e = 0; e < E; ++e) sc = fmaf(x[e], load_elem(kr + e * 2, a.type), sc);
        sc = wave_sum(sc);
        const float mn = fmaxf(m, sc);
        const float base = mn == -INFINITY ? 0.0f : mn;
        const float f = __builtin_amdgcn_exp2f(m - base), p = __builtin_amdgcn_exp2f(sc - base);
        l = l * f + p;
        for (int e = 0; e < E; ++e) o[e] = fmaf(p, load_elem(vr + e * 2, a.type), o[e] * f);
        m = mn;
    }
    const float inv = l == 0.0f ? 0.0f : 1.0f / l;
    for (int e = 0; e < E; ++e) store_elem(a.out + n * a.o_nb_t + h * a.o_nb_h + (lane * E + e) * 2, a.type, o[e] * inv);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(a.p.n_tok), dim3(256), 0, s, a);
    return hipGetLastError();
}

hipError_t launch_paged_attn(const PagedArgs& a, hipStream_t s) {
    const dim3 grid(a.n_tok, (a.Hq + 3) / 4);
    if (a.d == 64) hipLaunchKernelGGL(paged_attn_kernel<64>, grid, dim3(256), 0, s, a);
    else           hipLaunchKernelGGL(paged_attn_kernel<128>, grid, dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace vva
