// paged.hip — RoPE + append of packed tokens of many sequences into a cache in
// pages.
//
// What a call covers is on the device (vva_batch): the kernel finds its
// sequence in q_start, its keys in kv_len and their places in the page table,
// so the same launch serves any lengths of the same shapes.
#include "vva_internal.hpp"

#include <algorithm>

namespace vva {

namespace {

typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));
#include "paged_ops.hpp"

// 8 elements, 16-byte aligned: as loaded, as fp32, and stored
struct Raw8 {
    u32x4 a, b;                                    // b: F32 only
};
__device__ __forceinline__ Raw8 load_raw8(const char* p, int type) {
    Raw8 r;
    r.a = *(const u32x4*)p;
    if (type == VVA_TYPE_F32) r.b = ((const u32x4*)p)[1];
    return r;
}
__device__ __forceinline__ void raw8_to_f32(const Raw8& r, int type, float (&x)[8]) {
#pragma unroll
    for (int e = 0; e < 8; ++e) {
        const uint16_t v = (uint16_t)(r.a[e / 2] >> (16 * (e & 1)));
        x[e] = type == VVA_TYPE_F32 ? __uint_as_float(e < 4 ? r.a[e] : r.b[e - 4])
                                    : (type == VVA_TYPE_F16 ? f16_to_f32(v) : bf16_to_f32(v));
    }
}
__device__ __forceinline__ void store8(char* p, int type, const float (&y)[8]) {
    if (type == VVA_TYPE_F32) {
        ((float4*)p)[0] = make_float4(y[0], y[1], y[2], y[3]);
        ((float4*)p)[1] = make_float4(y[4], y[5], y[6], y[7]);
        return;
    }
    u32x4 w;
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const uint16_t lo = type == VVA_TYPE_F16 ? f32_to_f16(y[2 * e]) : f32_to_bf16(y[2 * e]);
        const uint16_t hi = type == VVA_TYPE_F16 ? f32_to_f16(y[2 * e + 1]) : f32_to_bf16(y[2 * e + 1]);
        w[e] = (uint32_t)lo | ((uint32_t)hi << 16);
    }
    *(u32x4*)p = w;
}

// One workgroup per token row, a thread per 8 rotation pairs (elements i ..
// i + 7 and i + P .. of a head); no head's item crosses a wave's table lookup.
// HBM-bound (4k tokens 78 -> 33 us against one pair per thread); a short call
// is a chain of two round trips: the batch, with the token's own rows under
// way, then the page id and the row of the rope table.
__global__ void __launch_bounds__(512) paged_append_kernel(PagedAppendArgs a) {
    prefetch_kernargs<sizeof(PagedAppendArgs)>();
    const PagedArgs& p = a.p;
    const int n = blockIdx.x, lane = threadIdx.x & 63;
    const int P = p.d >> 1, ph = P / 8;            // items per head
    const int items = (p.Hq + 2 * p.Hkv) * ph;
    // where item w's rows are read, and the loads
    struct Item {
        const char* src;
        int type, h, e;                            // kind of the head: h < Hq: q, then k, then v
    };
    auto item = [&](int w) {
        Item r;
        r.h = ph == 8 ? w >> 3 : w >> 2;
        r.e = (w & (ph - 1)) * 8;
        if (r.h < p.Hq) {
            r.src = p.q + n * p.q_nb_t + r.h * p.q_nb_h;
            r.type = a.q_type;
        } else if (r.h < p.Hq + p.Hkv) {
            r.src = a.k_new + n * a.k_nb_t + (r.h - p.Hq) * a.k_nb_h;
            r.type = a.k_type;
        } else {
            r.src = a.v_new + n * a.v_nb_t + (r.h - p.Hq - p.Hkv) * a.v_nb_h;
            r.type = a.v_type;
        }
        return r;
    };
    int w = threadIdx.x;
    Item it = item(min(w, items - 1));
    auto load = [&](const Item& t, Raw8& lo, Raw8& hi) {
        const int es = t.type == VVA_TYPE_F32 ? 4 : 2;
        lo = load_raw8(t.src + t.e * es, t.type);
        hi = load_raw8(t.src + (t.e + P) * es, t.type);
    };
    Raw8 lo, hi;
    load(it, lo, hi);
    // the token's sequence, its index in it, its slot and its rope row
    int s = -1, i = 0;
    for (int base = 0; base < p.n_seq; base += 64) {
        const Seq q = seq_of(p, min(base + lane, p.n_seq - 1));
        const uint64_t hit = __ballot(n >= q.q0 && n < q.q0 + q.n);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            s = min(base + l, p.n_seq - 1);
            i = lane_of(q.L, l) - lane_of(q.n, l) + (n - lane_of(q.q0, l));
            break;
        }
    }
    if (s < 0) return;
    const int page = i >= 0 ? p.table[s * p.table_stride + (i >> p.page_shift)] : -1;
    const int pos = a.pos ? a.pos[n] : i;
    const bool in_table = pos >= 0 && pos < a.n_pos;
    const float* cs = (const float*)(a.rope + (int64_t)(in_table ? pos : 0) * a.rope_nb);
    const bool live = page >= 0 && page < p.n_pages;
    const int slot = i & ((1 << p.page_shift) - 1);
    while (w < items) {
        float x0[8], x1[8], y0[8], y1[8];
        raw8_to_f32(lo, it.type, x0);
        raw8_to_f32(hi, it.type, x1);
        const Item t = it;
        if (t.h < p.Hq + p.Hkv) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float4 c4 = *(const float4*)(cs + t.e + 4 * v), s4 = *(const float4*)(cs + P + t.e + 4 * v);
                const float c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y0[4 * v + e] = in_table ? fmaf(x0[4 * v + e], c[e], -(x1[4 * v + e] * sn[e])) : __builtin_nanf("");
                    y1[4 * v + e] = in_table ? fmaf(x0[4 * v + e], sn[e], x1[4 * v + e] * c[e]) : __builtin_nanf("");
                }
            }
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                y0[e] = x0[e];
                y1[e] = x1[e];
            }
        }
        w += blockDim.x;
        if (w < items) {                           // heads beyond the workgroup's threads
            it = item(w);
            load(it, lo, hi);
        }
        char* dst;
        int type = p.type;
        if (t.h < p.Hq) {
            type = a.qo_type;
            dst = p.out + n * p.o_nb_t + t.h * p.o_nb_h;
        } else if (!live) {
            continue;
        } else if (t.h < p.Hq + p.Hkv) {
            dst = p.k + page * p.k_nb_page + (t.h - p.Hq) * p.k_nb_head + slot * p.k_nb_slot;
        } else {
            dst = p.v + page * p.v_nb_page + (t.h - p.Hq - p.Hkv) * p.v_nb_head + slot * p.v_nb_slot;
        }
        const int es = type == VVA_TYPE_F32 ? 4 : 2;
        store8(dst + t.e * es, type, y0);
        store8(dst + (t.e + P) * es, type, y1);
    }
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    const int items = (a.p.Hq + 2 * a.p.Hkv) * (a.p.d / 16);
    hipLaunchKernelGGL(paged_append_kernel, dim3(a.p.n_tok), dim3(std::min(512, (items + 63) / 64 * 64)), 0, s, a);
    return hipGetLastError();
}

}  // namespace vva
