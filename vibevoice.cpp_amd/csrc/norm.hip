// norm.hip — residual addition and root-mean-square norm before the
// projections (ggml_add, ggml_rms_norm and ggml_mul, src/qwen2.cpp:250-275),
// with the result in 32 or 16 bits or in GGUF Q8_0 blocks.
//
// h = x + add;  y = h / sqrt(mean(h^2) + eps) * w, all in fp32.
//
// One workgroup per row.  HBM-bound: every input is read once and every
// output written once; a short call is bound by its launch and one round trip.
#include "vva_internal.hpp"

namespace vva {

namespace {

__global__ void __launch_bounds__(256) norm_kernel(NormArgs a) {
    prefetch_kernargs<sizeof(NormArgs)>();
    const int n = blockIdx.x, tid = threadIdx.x;
    const int b = n / a.T, t = n - b * a.T;
    const char* x = a.x + b * a.x_nb_b + t * a.x_nb_t;
    const char* ad = a.add ? a.add + b * a.add_nb_b + t * a.add_nb_t : nullptr;
    char* sum = a.sum ? a.sum + b * a.sum_nb_b + t * a.sum_nb_t : nullptr;
    char* y = a.y + b * a.y_nb_b + t * a.y_nb_t;
    const int xe = (int)type_elem_bytes(a.x_type), ae = (int)type_elem_bytes(a.add_type);
    extern __shared__ float h[];                   // the row
    __shared__ float part[4];
    float ss = 0.0f;
    for (int i = tid; i < a.K; i += 256) {
        float v = load_elem(x + (int64_t)i * xe, a.x_type);
        if (ad) v += load_elem(ad + (int64_t)i * ae, a.add_type);
        h[i] = v;
        ss = fmaf(v, v, ss);
    }
    for (int m = 32; m >= 1; m >>= 1) ss += __shfl_xor(ss, m, 64);
    if ((tid & 63) == 0) part[tid >> 6] = ss;
    __syncthreads();
    const float r = 1.0f / sqrtf((part[0] + part[1] + part[2] + part[3]) / (float)a.K + a.eps);
    for (int i = tid; i < a.K; i += 256) {
        const float v = h[i];
        if (sum) store_elem(sum + (int64_t)i * type_elem_bytes(a.sum_type), a.sum_type, v);
        const float z = v * r * a.w[i];
        if (a.y_type != VVA_TYPE_Q8_0) {
            store_elem(y + (int64_t)i * type_elem_bytes(a.y_type), a.y_type, z);
            continue;
        }
        float am = fabsf(z);                       // the 32 lanes of a block: K is a multiple of 32
        for (int m = 16; m >= 1; m >>= 1) am = fmaxf(am, __shfl_xor(am, m, 32));
        const float d = am / 127.0f, id = d != 0.0f ? 1.0f / d : 0.0f;
        char* blk = y + (int64_t)(i / kQK8) * kQ8Bytes;
        if (i % kQK8 == 0) *(uint16_t*)blk = f32_to_f16(d);
        blk[2 + i % kQK8] = (char)(int8_t)roundf(z * id);
    }
}

}  // namespace

hipError_t launch_norm(const NormArgs& a, hipStream_t s) {
    hipLaunchKernelGGL(norm_kernel, dim3(a.N), dim3(256), (size_t)a.K * sizeof(float), s, a);
    return hipGetLastError();
}

}  // namespace vva
