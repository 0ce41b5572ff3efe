// paged_ops.hpp — what the kernels over a cache in pages share: a sequence of
// the batch, kept inside the rows and the table there are, and the lookups by
// whole waves.  Included inside an anonymous namespace of each kernel file.
#pragma once

struct Seq {
    int q0, n;          // first token row, new tokens
    int L;              // keys
    int s;              // its index
};
__device__ __forceinline__ Seq seq_of(const PagedArgs& a, int s) {
    Seq r;
    r.s = s;
    r.q0 = min(max(a.q_start[s], 0), a.n_tok);
    r.n = min(max(a.q_start[s + 1], r.q0), a.n_tok) - r.q0;
    r.L = min(max(a.kv_len[s], 0), a.max_pages << a.page_shift);
    return r;
}

__device__ __forceinline__ int lane_of(int x, int lane) { return __builtin_amdgcn_readlane(x, lane); }
// Sum of x over the lanes up to and with this one (DPP: shifts within rows of
// 16 lanes, then the rows' totals broadcast upwards)
template <int CTRL, int ROWS>
__device__ __forceinline__ int dpp_add(int x) { return x + __builtin_amdgcn_update_dpp(0, x, CTRL, ROWS, 0xf, false); }
__device__ __forceinline__ int wave_scan(int x) {
    x = dpp_add<0x111, 0xf>(x);
    x = dpp_add<0x112, 0xf>(x);
    x = dpp_add<0x114, 0xf>(x);
    x = dpp_add<0x118, 0xf>(x);
    x = dpp_add<0x142, 0xa>(x);                    // row 0's total to row 1, row 2's to row 3
    return dpp_add<0x143, 0xc>(x);                 // the lower half's to the upper
}
// Sum of x over the wave (DPP within rows of 16 lanes, permlane swaps across)
__device__ __forceinline__ int wave_total(int x) {
    x += __builtin_amdgcn_mov_dpp(x, 0xB1, 0xf, 0xf, true);
    x += __builtin_amdgcn_mov_dpp(x, 0x4E, 0xf, 0xf, true);
    x += __builtin_amdgcn_mov_dpp(x, 0x141, 0xf, 0xf, true);
    x += __builtin_amdgcn_mov_dpp(x, 0x140, 0xf, 0xf, true);
    const auto a = __builtin_amdgcn_permlane16_swap((unsigned)x, (unsigned)x, false, false);
    x = (int)(a[0] + a[1]);
    const auto b = __builtin_amdgcn_permlane32_swap((unsigned)x, (unsigned)x, false, false);
    return __builtin_amdgcn_readfirstlane((int)(b[0] + b[1]));
}
// x / G for 0 <= x < 2^31, by the call's multiplier
__device__ __forceinline__ int div_g(const PagedArgs& a, int x) {
    return a.g_mul ? (int)(__umulhi((uint32_t)x, a.g_mul) >> a.g_shift) : x;
}
