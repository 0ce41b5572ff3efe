// Prints the plans of vva_paged_attn calls over single tokens and a few tokens of
// many sequences, one line each: type, head dim, query heads, kv heads, rows of a
// sequence and kv head, sequences, then waves of a workgroup and the workgroups
// that the plan takes to run at once, for a GPU of 256 CUs.  No HIP call.
#include <cstdio>

#include "../../vibevoice.cpp_amd/csrc/vva_internal.hpp"

int main() {
    const int heads[][3] = {{64, 14, 2}, {64, 4, 4}, {64, 32, 1}, {128, 28, 4}, {128, 12, 2}, {128, 32, 1}};
    for (int type : {VVA_TYPE_F16, VVA_TYPE_BF16, VVA_TYPE_Q8_0})
        for (const auto& h : heads)
            for (int n_seq : {1, 2, 7, 48, 64, 65, 130, 256, 1000})
                for (int max_new : {1, 2, 4, 16, 32}) {
                    vva::PagedArgs a{};
                    a.type = type;
                    a.io_type = type == VVA_TYPE_BF16 ? VVA_TYPE_BF16 : VVA_TYPE_F16;
                    a.d = h[0], a.Hq = h[1], a.Hkv = h[2], a.G = h[1] / h[2];
                    a.n_seq = n_seq, a.max_new = max_new, a.n_tok = n_seq * max_new;
                    a.page_shift = 4, a.max_pages = 500;
                    if (max_new * a.G > 32) continue;
                    const vva::PagedPlan p = vva::paged_plan(a, 256);
                    std::printf("%d %d %d %d %d %d %d %d\n", type, a.d, a.Hq, a.Hkv, max_new * a.G, n_seq, p.few_waves, p.few_slots * a.Hkv);
                }
    return 0;
}
