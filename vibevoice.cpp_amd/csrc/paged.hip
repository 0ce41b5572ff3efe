// paged.hip — RoPE + append of packed tokens of many sequences into a cache in
// pages.
//
// What a call covers is on the device (vva_batch): the kernel finds its
// sequence in q_start, its keys in kv_len and their places in the page table,
// so the same launch serves any lengths of the same shapes.
#include "vva_internal.hpp"

namespace vva {

namespace {

#include "paged_ops.hpp"

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

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(paged_append_kernel, dim3(a.p.n_tok), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace vva
