// paged.hip — RoPE + append of packed tokens of many sequences into a cache in
// pages, of 16 bits or quantised to Q8_0, and rows read back out of it.
//
// What a call covers is on the device (vva_batch): the kernel finds its
// sequence in q_start, its keys in kv_len and their places in the page table,
// so the same launch serves any lengths of the same shapes.
#include "vva_internal.hpp"

#include <algorithm>

namespace vva {

namespace {

#include "wave_ops.hpp"
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

// 8 elements from i on of a Q8_0 page's row, by 4 lanes per block: the codes are
// d bytes a slot, the scales of a block `page` F16 behind all of them
__device__ __forceinline__ void store8_q8(char* tile, int d, int page_shift, int slot, int i, const float (&y)[8]) {
    const Q8Block b = q8_block(y);
    int c[8];
#pragma unroll
    for (int e = 0; e < 8; ++e) c[e] = b.code(y[e]);
    *(uint2*)(tile + slot * d + i) = make_uint2(q8_pack(c[0], c[1], c[2], c[3]), q8_pack(c[4], c[5], c[6], c[7]));
    if (i % kQK8 == 0) *(uint16_t*)(tile + (d << page_shift) + (((i / kQK8) << page_shift) + slot) * 2) = b.scale;
}

// One workgroup per token row, a thread per 8 rotation pairs (elements i ..
// i + 7 and i + P .. of a head); no head's item crosses a wave's table lookup.
// HBM-bound (4k tokens, F32 rows of 7B heads, three sets of tensors by turns: 27.4 us,
// 4.7 TB/s, 28.2 into Q8_0 pages, 23.3 over one set that the last-level cache holds;
// one pair per thread 78); a short call is a chain of two round trips: the
// batch, with the token's own rows under way, then the page id and the row of the
// rope table.
// IO: the type of q, k and v where it is one, else -1 (types looked up by the lane
// took 32.8 us, BF16 rows into Q8_0 pages 25.4 for 17.4)
template <bool Q8, int IO>
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
        const int type = IO >= 0 ? IO : t.type, es = type == VVA_TYPE_F32 ? 4 : 2;
        lo = load_raw8(t.src + t.e * es, type);
        hi = load_raw8(t.src + (t.e + P) * es, type);
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
    // (uniform: what goes by them are scalar branches and bases)
    const int page = __builtin_amdgcn_readfirstlane(i >= 0 ? p.table[s * p.table_stride + (i >> p.page_shift)] : -1);
    const int pos = __builtin_amdgcn_readfirstlane(a.pos ? a.pos[n] : i);
    const bool in_table = pos >= 0 && pos < a.n_pos;
    const float* cs = (const float*)(a.rope + (int64_t)(in_table ? pos : 0) * a.rope_nb);
    const bool live = page >= 0 && page < p.n_pages;
    const int slot = i & ((1 << p.page_shift) - 1);
    while (w < items) {
        float x0[8], x1[8], y0[8], y1[8];
        raw8_to_f32(lo, IO >= 0 ? IO : it.type, x0);
        raw8_to_f32(hi, IO >= 0 ? IO : it.type, x1);
        const Item t = it;
        if (t.h < p.Hq + p.Hkv) {
#pragma unroll
            for (int v = 0; v < 2; ++v) {
                const float4 c4 = *(const float4*)(cs + t.e + 4 * v), s4 = *(const float4*)(cs + P + t.e + 4 * v);
                const float c[4] = {c4.x, c4.y, c4.z, c4.w}, sn[4] = {s4.x, s4.y, s4.z, s4.w};
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    y0[4 * v + e] = fmaf(x0[4 * v + e], c[e], -(x1[4 * v + e] * sn[e]));
                    y1[4 * v + e] = fmaf(x0[4 * v + e], sn[e], x1[4 * v + e] * c[e]);
                }
            }
            if (!in_table)
#pragma unroll
                for (int e = 0; e < 8; ++e) y0[e] = y1[e] = __builtin_nanf("");
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
            dst = p.k + page * p.k_nb_page + (t.h - p.Hq) * p.k_nb_head + (Q8 ? 0 : slot * p.k_nb_slot);
        } else {
            dst = p.v + page * p.v_nb_page + (t.h - p.Hq - p.Hkv) * p.v_nb_head + (Q8 ? 0 : slot * p.v_nb_slot);
        }
        if constexpr (Q8) {
            if (t.h >= p.Hq) {                     // the same for the 4 lanes of a block
                store8_q8(dst, p.d, p.page_shift, slot, t.e, y0);
                store8_q8(dst, p.d, p.page_shift, slot, t.e + P, y1);
                continue;
            }
        }
        const int es = type == VVA_TYPE_F32 ? 4 : 2;
        store8(dst + t.e * es, type, y0);
        store8(dst + (t.e + P) * es, type, y1);
    }
}

// Rows read back: one workgroup per kReadTokens token rows, a wave for every
// fourth of them, whose loads go out together; a lane takes 8 elements of a K or V
// row at a time.  HBM-bound: 20k tokens of 7B heads to BF16, from Q8_0 pages (63 MB)
// 12.8 us, a copy's 4.9 TB/s, from F16 pages (82 MB) 18.0, 4.6; a short call is the launch and three round trips
// (333 tokens 4.3 us).
constexpr int kReadTokens = 16, kReadWaves = 4;

template <bool Q8>
__global__ void __launch_bounds__(kReadWaves * 64) paged_read_kernel(PagedReadArgs a) {
    prefetch_kernargs<sizeof(PagedReadArgs)>();
    constexpr int NT = kReadTokens / kReadWaves;
    const PagedArgs& p = a.p;
    const int lane = threadIdx.x & 63, w = threadIdx.x >> 6, n0 = blockIdx.x * kReadTokens + w;
    int page[NT], slot[NT];                        // page: -1: NaN, -2: no row
    for (int i = 0; i < NT; ++i) page[i] = -2, slot[i] = 0;
    for (int base = 0; base < p.n_seq; base += 64) {
        const Seq q = seq_of(p, min(base + lane, p.n_seq - 1));
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const int n = n0 + i * kReadWaves;
            const uint64_t hit = __ballot(n < p.n_tok && n >= q.q0 && n < q.q0 + q.n);
            if (!hit || page[i] != -2) continue;
            const int l = __ffsll((unsigned long long)hit) - 1;
            const int at = lane_of(q.L, l) - lane_of(q.n, l) + (n - lane_of(q.q0, l));
            const int id = at >= 0 ? p.table[min(base + l, p.n_seq - 1) * p.table_stride + (at >> p.page_shift)] : -1;
            page[i] = id >= 0 && id < p.n_pages ? id : -1;
            slot[i] = at & ((1 << p.page_shift) - 1);
        }
    }
    const int ph = p.d == 128 ? 16 : 8, each = p.Hkv * ph;   // 8-element parts of a head, of K's row
    for (int k = lane; k < 2 * each; k += 64) {
        const bool v = k >= each;
        char* const out = v ? a.v_out : a.k_out;
        if (!out) continue;
        const int kk = v ? k - each : k, h = p.d == 128 ? kk >> 4 : kk >> 3, e = (kk & (ph - 1)) * 8;
        const char* const pool = (v ? p.v + h * p.v_nb_head : p.k + h * p.k_nb_head);
        const int64_t nb_page = v ? p.v_nb_page : p.k_nb_page, nb_slot = v ? p.v_nb_slot : p.k_nb_slot;
        const int type = v ? a.v_type : a.k_type;
        char* const dst = out + (v ? h * a.v_nb_h : h * a.k_nb_h) + e * (type == VVA_TYPE_F32 ? 4 : 2);
        const int64_t nb_t = v ? a.v_nb_t : a.k_nb_t;
        u32x4 raw[NT];
        uint16_t scale[NT];
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            const char* tile = pool + max(page[i], 0) * nb_page;
            if constexpr (Q8) {
                const uint2 c = *(const uint2*)(tile + slot[i] * p.d + e);
                raw[i] = u32x4{c.x, c.y, 0u, 0u};
                scale[i] = *(const uint16_t*)(tile + (p.d << p.page_shift) + (((e / kQK8) << p.page_shift) + slot[i]) * 2);
            } else {
                raw[i] = *(const u32x4*)(tile + slot[i] * nb_slot + e * 2);
            }
        }
#pragma unroll
        for (int i = 0; i < NT; ++i) {
            if (page[i] == -2) continue;
            float x[8];
            if constexpr (Q8) {
                const float s = f16_to_f32(scale[i]);
#pragma unroll
                for (int b = 0; b < 8; ++b) x[b] = s * (float)(int8_t)(raw[i][b / 4] >> (8 * (b % 4)));
            } else {
                raw8_to_f32(Raw8{raw[i], raw[i]}, p.type, x);
            }
            if (page[i] == -1)
#pragma unroll
                for (int b = 0; b < 8; ++b) x[b] = __builtin_nanf("");
            store8(dst + (n0 + i * kReadWaves) * nb_t, type, x);
        }
    }
}

template <bool Q8>
void launch_append(const PagedAppendArgs& a, dim3 g, dim3 b, hipStream_t s) {
    if (a.q_type != a.k_type || a.k_type != a.v_type) hipLaunchKernelGGL((paged_append_kernel<Q8, -1>), g, b, 0, s, a);
    else if (a.q_type == VVA_TYPE_F32) hipLaunchKernelGGL((paged_append_kernel<Q8, VVA_TYPE_F32>), g, b, 0, s, a);
    else if (a.q_type == VVA_TYPE_F16) hipLaunchKernelGGL((paged_append_kernel<Q8, VVA_TYPE_F16>), g, b, 0, s, a);
    else hipLaunchKernelGGL((paged_append_kernel<Q8, VVA_TYPE_BF16>), g, b, 0, s, a);
}

}  // namespace

hipError_t launch_paged_append(const PagedAppendArgs& a, hipStream_t s) {
    const int items = (a.p.Hq + 2 * a.p.Hkv) * (a.p.d / 16);
    const dim3 g(a.p.n_tok), b(std::min(512, (items + 63) / 64 * 64));
    if (a.p.type == VVA_TYPE_Q8_0) launch_append<true>(a, g, b, s);
    else launch_append<false>(a, g, b, s);
    return hipGetLastError();
}

hipError_t launch_paged_read(const PagedReadArgs& a, hipStream_t s) {
    const dim3 g((a.p.n_tok + kReadTokens - 1) / kReadTokens), b(kReadWaves * 64);
    if (a.p.type == VVA_TYPE_Q8_0) hipLaunchKernelGGL(paged_read_kernel<true>, g, b, 0, s, a);
    else hipLaunchKernelGGL(paged_read_kernel<false>, g, b, 0, s, a);
    return hipGetLastError();
}

}  // namespace vva
