// norm.hip — residual addition and root-mean-square norm before the
// projections (ggml_add, ggml_rms_norm and ggml_mul, src/qwen2.cpp:250-275),
// with the result in 32 or 16 bits or in GGUF Q8_0 blocks.
//
// h = x + add;  y = h / sqrt(mean(h^2) + eps) * w, all in fp32.
//
// One workgroup per row, of as many waves (up to 4) as its 8-element parts
// fill; a thread holds its parts of the row in registers from the one read to
// the one write.  HBM-bound: every input is read once and every output written
// once (8192 BF16 rows of 3584 51 us, 4.6 TB/s; element by element 137); a
// short call is bound by its launch and one round trip (2 rows 3.8 us).  Rows of
// aligned tensors go 8 elements a load; the rest element by element.  The sum
// of squares of a thread runs in fp32 over at most 64 elements, then over the
// lanes and waves.
#include "vva_internal.hpp"

#include <algorithm>

namespace vva {

namespace {

#include "wave_ops.hpp"

// 8 elements from p (VEC: 16-byte aligned and all there; else n of them)
template <bool VEC>
__device__ __forceinline__ void load8(const char* p, int type, int n, float (&x)[8]) {
    if constexpr (VEC) {
        const u32x4 a = *(const u32x4*)p;
        if (type == VVA_TYPE_F32) {
            const u32x4 b = ((const u32x4*)p)[1];
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                x[e] = __uint_as_float(a[e]);
                x[e + 4] = __uint_as_float(b[e]);
            }
            return;
        }
#pragma unroll
        for (int e = 0; e < 8; ++e) {
            const uint16_t v = (uint16_t)(a[e / 2] >> (16 * (e & 1)));
            x[e] = type == VVA_TYPE_F16 ? f16_to_f32(v) : bf16_to_f32(v);
        }
    } else {
        const int es = type == VVA_TYPE_F32 ? 4 : 2;
#pragma unroll
        for (int e = 0; e < 8; ++e) x[e] = e < n ? load_elem(p + e * es, type) : 0.0f;
    }
}
template <bool VEC>
__device__ __forceinline__ void store8(char* p, int type, int n, const float (&x)[8]) {
    if constexpr (VEC) {
        if (type == VVA_TYPE_F32) {
            ((float4*)p)[0] = make_float4(x[0], x[1], x[2], x[3]);
            ((float4*)p)[1] = make_float4(x[4], x[5], x[6], x[7]);
            return;
        }
        u32x4 w;
#pragma unroll
        for (int e = 0; e < 4; ++e) {
            const uint16_t lo = type == VVA_TYPE_F16 ? f32_to_f16(x[2 * e]) : f32_to_bf16(x[2 * e]);
            const uint16_t hi = type == VVA_TYPE_F16 ? f32_to_f16(x[2 * e + 1]) : f32_to_bf16(x[2 * e + 1]);
            w[e] = (uint32_t)lo | ((uint32_t)hi << 16);
        }
        *(u32x4*)p = w;
    } else {
        const int es = type == VVA_TYPE_F32 ? 4 : 2;
#pragma unroll
        for (int e = 0; e < 8; ++e)
            if (e < n) store_elem(p + e * es, type, x[e]);
    }
}

// PARTS: 8-element parts of the row per thread
template <int PARTS, bool VEC>
__global__ void __launch_bounds__(256) norm_kernel(NormArgs a) {
    prefetch_kernargs<sizeof(NormArgs)>();
    const int n = blockIdx.x, tid = threadIdx.x, threads = blockDim.x;
    const int b = n / a.T, t = n - b * a.T;
    const char* x = a.x + b * a.x_nb_b + t * a.x_nb_t;
    const char* ad = a.add ? a.add + b * a.add_nb_b + t * a.add_nb_t : nullptr;
    const int xe = a.x_type == VVA_TYPE_F32 ? 4 : 2, ae = a.add_type == VVA_TYPE_F32 ? 4 : 2;
    float h[PARTS][8], g[PARTS][8];
    float ss = 0.0f;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int k = (i * threads + tid) * 8;
        if (k < a.K) load8<VEC>(x + (int64_t)k * xe, a.x_type, a.K - k, h[i]);
        else for (int e = 0; e < 8; ++e) h[i][e] = 0.0f;
    }
    if (ad) {
#pragma unroll
        for (int i = 0; i < PARTS; ++i) {
            const int k = (i * threads + tid) * 8;
            if (k >= a.K) continue;
            float v[8];
            load8<VEC>(ad + (int64_t)k * ae, a.add_type, a.K - k, v);
#pragma unroll
            for (int e = 0; e < 8; ++e) h[i][e] += v[e];
        }
    }
    // the weights come before the reduction, in the shadow of its latency
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int k = (i * threads + tid) * 8;
        if (k < a.K) load8<VEC>((const char*)(a.w + k), VVA_TYPE_F32, a.K - k, g[i]);
    }
#pragma unroll
    for (int i = 0; i < PARTS; ++i)
#pragma unroll
        for (int e = 0; e < 8; ++e) ss = fmaf(h[i][e], h[i][e], ss);
    ss = wave_sum(ss);
    if (threads > 64) {
        __shared__ float part[4];
        if ((tid & 63) == 0) part[tid >> 6] = ss;
        __syncthreads();
        ss = part[0];
        for (int i = 1; i < threads / 64; ++i) ss += part[i];
    }
    const float r = 1.0f / sqrtf(ss / (float)a.K + a.eps);
    char* y = a.y + b * a.y_nb_b + t * a.y_nb_t;
#pragma unroll
    for (int i = 0; i < PARTS; ++i) {
        const int k = (i * threads + tid) * 8, left = a.K - k;
        if (left <= 0) continue;
        if (a.sum)
            store8<VEC>(a.sum + b * a.sum_nb_b + t * a.sum_nb_t + (int64_t)k * (a.sum_type == VVA_TYPE_F32 ? 4 : 2), a.sum_type, left, h[i]);
        float z[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) z[e] = h[i][e] * r * g[i][e];
        if (a.y_type != VVA_TYPE_Q8_0) {
            store8<VEC>(y + (int64_t)k * (a.y_type == VVA_TYPE_F32 ? 4 : 2), a.y_type, left, z);
            continue;
        }
        // the 4 lanes of a block (K is a multiple of 32: a block's lanes are all here)
        const Q8Block q8 = q8_block(z);
        uint16_t* blk = (uint16_t*)(y + (int64_t)(k / kQK8) * kQ8Bytes);
        const int q = (k % kQK8) / 2;
        if (q == 0) blk[0] = q8.scale;
#pragma unroll
        for (int e = 0; e < 4; ++e) blk[1 + q + e] = (uint16_t)((q8.code(z[2 * e]) & 0xff) | (q8.code(z[2 * e + 1]) << 8));
    }
}

template <bool VEC>
hipError_t launch_parts(const NormArgs& a, hipStream_t s) {
    const int parts = (a.K + 7) / 8;
    const int threads = std::min(256, (parts + 63) / 64 * 64);
    const dim3 g(a.N), b(threads);
    switch ((parts + threads - 1) / threads) {
        case 1: hipLaunchKernelGGL((norm_kernel<1, VEC>), g, b, 0, s, a); break;
        case 2: hipLaunchKernelGGL((norm_kernel<2, VEC>), g, b, 0, s, a); break;
        case 3: case 4: hipLaunchKernelGGL((norm_kernel<4, VEC>), g, b, 0, s, a); break;
        default: hipLaunchKernelGGL((norm_kernel<8, VEC>), g, b, 0, s, a); break;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, hipStream_t s) {
    auto al = [](const void* p, int64_t nb_t, int64_t nb_b) { return !p || ((uintptr_t)p | (uint64_t)nb_t | (uint64_t)nb_b) % 16 == 0; };
    const bool vec = a.K % 8 == 0 && al(a.x, a.x_nb_t, a.x_nb_b) && al(a.add, a.add_nb_t, a.add_nb_b) &&
                     al(a.sum, a.sum_nb_t, a.sum_nb_b) && (a.y_type == VVA_TYPE_Q8_0 || al(a.y, a.y_nb_t, a.y_nb_b)) && al(a.w, 0, 0);
    return vec ? launch_parts<true>(a, s) : launch_parts<false>(a, s);
}

}  // namespace vva
