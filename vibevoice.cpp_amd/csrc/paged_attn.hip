// paged_attn.hip — causal grouped-query attention of packed tokens of many
// sequences over a cache in pages, on the matrix cores.
//
// What a call covers is on the device (vva_batch): every kernel finds its
// work in q_start, kv_len and the page table, so the same launch serves any
// lengths of the same shapes and a captured call is replayed while its
// sequences grow.
//
// Query rows are the (token, head) pairs of one kv group, r = t * G + head, so
// the G heads of a group share every K / V row that is read.  Sequences whose
// rows fit one 32-wide matrix operand (n_s * G <= 32: single tokens, a few
// proposed ones) take paged_few_kernel, which is bound by the cache's bytes;
// the others paged_many_kernel, which is bound by the matrix cores.
//
// Both compute, per 32 rows and a tile of keys, with
// v_mfma_f32_32x32x16_{f16,bf16} (layouts in mfma_ops.hpp):
//   S^T[key][row] = K . Q^T    Q^T in registers; a lane owns one query row
//   softmax                    fp32, exp2 domain, scale folded into the exp's
//                              fma; the running max of a row is raised only
//                              when a tile's max passes it by more than 2^8,
//                              so p <= 256 fits f16 and rescales are rare
//   O^T[dim][row] += V^T . P^T P converted in place from the accumulators: the
//                              key order of a step is the one they have
// P is rounded to the pages' type, a relative 2^-11 (F16) or 2^-8 (BF16) at
// most, as the output itself is; the row sum adds the rounded values, so the
// weights of a row sum to one.
//
// K and V rows go from the pages straight into LDS (global_load_lds, 1 KB =
// 4 rows of 128 dims an instruction, no registers), 16-byte chunk c of row r
// at chunk c ^ f(r): with the swizzle chosen by the source address a row needs
// no padding, K is read by 16 lanes on 16 different bank groups, and the
// transposing reads of V (4 rows x 64 B per 32 lanes) on four.  A page id comes
// from the table by scalar loads, once per 16 keys (the smallest page).
//
// Tiles whose last key some row must not see are masked: their scores go to
// -inf by a select, and where such a tile holds a V that is not finite (a
// stale slot behind the sequence, a later token's overflow) its products leave
// those values out and add them to the rows that see them (0 * inf is not 0).
#include "vva_internal.hpp"

#include <algorithm>

namespace vva {

namespace {

#include "wave_ops.hpp"
#include "mfma_ops.hpp"
#include "paged_ops.hpp"

constexpr float kLazy = 8.0f;      // running-max slack in log2 units
constexpr int kFewRows = 32;       // rows of a sequence and kv head that paged_few_kernel takes
// exponent base of a partial whose keys lie in a page outside the pool; handled as
// bits, since this file is compiled for numbers alone
constexpr uint32_t kNanBits = 0x7fc00000u;

typedef const __attribute__((address_space(4))) int32_t* ConstInts;

// 64 lanes' 16 bytes from base + voff to LDS lds .. lds + 1023.  Inline asm so
// that the compiler does not fence LDS reads on it: completion is waited for
// explicitly.  The address is uniform but for the lane's 32-bit offset.
// NT: non-temporal, for rows that the call reads once (64 x 4096 keys 5.4 ->
// 6.0 TB/s, 128 x 4096 5.8 -> 6.5).
template <bool NT>
__device__ __forceinline__ void dma16(uint64_t base, int voff, uint32_t lds) {
    if constexpr (NT)
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2 nt"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(base)
                     : "memory", "m0");
    else
        asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dwordx4 %1, %2"
                     :
                     : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(voff), "s"(base)
                     : "memory", "m0");
}
__device__ __forceinline__ uint64_t uniform64(uint64_t x) {
    return (uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)x) |
           ((uint64_t)(uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(x >> 32)) << 32);
}
template <int N>
__device__ __forceinline__ void wait_vm() {
    asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" : : "n"(N) : "memory");
}
__device__ __forceinline__ const lds_char* lds_at(uint32_t addr) { return (const lds_char*)(uintptr_t)addr; }

// Swizzle of a K / V row of D dims: XORed to the index of a 16-byte chunk
template <int D> __device__ __forceinline__ int k_swz(int row) { return D == 128 ? row & 15 : (row >> 1) & 7; }
template <int D> __device__ __forceinline__ int v_swz(int row) { return D == 128 ? (row & 3) << 2 : ((row >> 1) & 1) << 2; }

// Byte offset, in a 1 KB group of rows that starts at row r0 of its tile, of
// what this lane loads: row lane / chunks, and the chunk that its LDS place
// holds
template <int D, bool V>
__device__ __forceinline__ int dma_off(int lane, int r0, int nb_slot) {
    constexpr int C = D / 8;                       // chunks per row
    const int r = lane / C, c = (lane % C) ^ (V ? v_swz<D>(r0 + r) : k_swz<D>(r0 + r));
    return r * nb_slot + c * 16;
}

// 16-bit types: the pack of two probabilities, and their sum
template <int KT>
__device__ __forceinline__ uint32_t pack2(float x, float y) {
    if constexpr (KT == VVA_TYPE_BF16) {
        const bf2 v = {(__bf16)x, (__bf16)y};
        uint32_t r;
        __builtin_memcpy(&r, &v, 4);
        return r;
    } else {
        const h2 v = {(_Float16)x, (_Float16)y};
        uint32_t r;
        __builtin_memcpy(&r, &v, 4);
        return r;
    }
}
template <int KT>
__device__ __forceinline__ float sum2(uint32_t p, float acc) {
    return KT == VVA_TYPE_BF16 ? dot2_bf16(p, 0x3f803f80u, acc) : dot2_f16(p, 0x3c003c00u, acc);
}
// whether either half of x is infinite or NaN, and x with such halves zeroed
template <int KT>
__device__ __forceinline__ bool not_finite2(uint32_t x) {
    constexpr uint32_t e = KT == VVA_TYPE_BF16 ? 0x7f80u : 0x7c00u;
    return (x & e) == e || ((x >> 16) & e) == e;
}
template <int KT>
__device__ __forceinline__ uint32_t finite2(uint32_t x) {
    constexpr uint32_t e = KT == VVA_TYPE_BF16 ? 0x7f80u : 0x7c00u;
    return ((x & e) == e ? 0u : x & 0xffffu) | (((x >> 16) & e) == e ? 0u : x & 0xffff0000u);
}

// V^T fragment of 16 keys and 32 dims from the lane's two places in the tile
template <int KT>
__device__ __forceinline__ u32x4 v_bits(const lds_char* p0, const lds_char* p1) {
    const s4 lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p0);
    const s4 hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s4*)p1);
    u32x2 a, b;
    __builtin_memcpy(&a, &lo, 8);
    __builtin_memcpy(&b, &hi, 8);
    return u32x4{a.x, a.y, b.x, b.y};
}

// This lane's parts of a tile's LDS addresses: K row l32 (XOR ds << 5 for
// 16-dim step ds), V rows of a 16-key step (XOR dt << 6 for 32-dim tile dt)
template <int D>
__device__ __forceinline__ int k_lane_off(int lane) {
    const int l32 = lane & 31;
    return l32 * 2 * D + (((lane >> 5) ^ k_swz<D>(l32)) << 4);
}
template <int D>
__device__ __forceinline__ int v_lane_off(int lane) {
    const int r = (lane & 15) >> 2;
    const int c = (2 * ((lane >> 4) & 1) + ((lane & 3) >> 1)) ^ v_swz<D>(r);
    return (r + 4 * (lane >> 5)) * 2 * D + (c << 4) + 8 * (lane & 1);
}

// Q^T fragments of the lane's row (zeros where there is none)
template <int D, typename QF>
__device__ __forceinline__ void load_q(const PagedArgs& a, int q0, int kvh, int row, int rows, int half, QF (&qf)[D / 16]) {
    const bool ok = row < rows;
    const int t = ok ? row / a.G : 0, h = ok ? row % a.G : 0;
    const char* p = a.q + (int64_t)(q0 + t) * a.q_nb_t + (int64_t)(kvh * a.G + h) * a.q_nb_h + half * 16;
#pragma unroll
    for (int ds = 0; ds < D / 16; ++ds) {
        const u32x4 r = *(const u32x4*)(p + ds * 32);
        qf[ds] = as_vec<QF>(ok ? r : u32x4{0u, 0u, 0u, 0u});
    }
}

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
__device__ __forceinline__ lds_u32x4* lds_vec(uint32_t addr) { return (lds_u32x4*)(uintptr_t)addr; }
__device__ __forceinline__ u32x4 lds_read(uint32_t addr) { return *lds_vec(addr); }
template <int KT>
__device__ __forceinline__ bool chunk_not_finite(u32x4 x) {
    return not_finite2<KT>(x.x) || not_finite2<KT>(x.y) || not_finite2<KT>(x.z) || not_finite2<KT>(x.w);
}
// Whether some V of a tile of N keys is infinite or NaN (whole wave)
template <int D, int KT, int N>
__device__ __forceinline__ bool tile_not_finite(uint32_t v_lds, int lane) {
    bool bad = false;
#pragma unroll
    for (int i = 0; i < N * 2 * D / 1024; ++i) {
        bad = bad || chunk_not_finite<KT>(lds_read(v_lds + i * 1024 + lane * 16));
    }
    return __any(bad);
}
// O += the infinities and NaNs of a tile's V that this lane's row sees (keys
// k0 .. of the tile up to lim)
template <int D, int KT, int N>
__device__ __forceinline__ void add_not_finite(uint32_t v_lds, int k0, int lim, int half, f32x16 (&o)[D / 32]) {
    for (int j = 0; j < N; ++j) {
        const bool seen = k0 + j <= lim;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const u32x2 x = *(const __attribute__((address_space(3))) u32x2*)lds_at(
                    v_lds + j * 2 * D + (((dt * 4 + q4) ^ v_swz<D>(j)) << 4) + 8 * half);
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t w = (e < 2 ? x.x : x.y) >> (16 * (e & 1)) & 0xffffu;
                    const float v = KT == VVA_TYPE_BF16 ? bf16_to_f32((uint16_t)w) : f16_to_f32((uint16_t)w);
                    if (seen && not_finite2<KT>(w)) o[dt][4 * q4 + e] += v;
                }
            }
    }
}

// ------------------------------------------------------------ few rows

// Workgroups per kv head that paged_few_kernel's work is cut into, and the
// least tiles (32 keys) of one: a tile per wave.
constexpr int kFewWaves = 4;
constexpr int kFewTile = 32;
constexpr int kFewMin = kFewWaves;

// A piece of a sequence's keys: piece `part` of `parts`; n = 0: none
struct FewItem {
    Seq q;
    int s, part, parts, first;      // first: the sequence's piece 0
};
// Tiles of sequence q that paged_few_kernel works on
__device__ __forceinline__ int few_tiles(const PagedArgs& a, const Seq& q) {
    const int n = min(q.n, a.max_new);
    return n > 0 && n * a.G <= kFewRows ? max(1, (q.L + kFewTile - 1) / kFewTile) : 0;
}
// Piece `item` of the call.  All sequences are cut into pieces of at most
// `chunk` tiles, the least for which the pieces are no more than `slots` (the
// workgroups that run at once, per kv head), so a long sequence among short
// ones gets its share of the chip and no piece waits for a second round: tried
// from the even share up in steps of an eighth, for up to 64 sequences; more
// of them leave many pieces, whose rounds even out.  By whole waves.
__device__ __forceinline__ FewItem few_item(const PagedArgs& a, int item, int slots) {
    const int lane = threadIdx.x & 63;
    Seq q = seq_of(a, min(lane, a.n_seq - 1));
    int t = lane < a.n_seq ? few_tiles(a, q) : 0;
    int total = t;
    for (int s = lane + 64; s < a.n_seq; s += 64) total += few_tiles(a, seq_of(a, s));
    total = wave_total(total);
    int chunk = max(kFewMin, (total + slots - 1) / slots);
    if (a.n_seq <= 64)
        for (int i = 0; i < 12 && wave_total((t + chunk - 1) / chunk) > slots; ++i) chunk += (chunk + 7) / 8;
    FewItem r{};
    int base = 0;
    for (int i = 0; i < a.n_seq; i += 64) {
        if (i > 0) {
            q = seq_of(a, min(i + lane, a.n_seq - 1));
            t = i + lane < a.n_seq ? few_tiles(a, q) : 0;
        }
        const int c = (t + chunk - 1) / chunk;
        const int end = wave_scan(c);
        const uint64_t hit = __ballot(item >= base + end - c && item < base + end);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            r.q.q0 = lane_of(q.q0, l);
            r.q.n = lane_of(q.n, l);
            r.q.L = lane_of(q.L, l);
            r.s = i + l;
            r.parts = lane_of(c, l);
            r.first = base + lane_of(end - c, l);
            r.part = item - r.first;
            return r;
        }
        base += lane_of(end, 63);
    }
    return r;
}

constexpr int kSc1 = 16;           // cache policy of the partials: agent scope
// pieces whose partials are loaded together (16: 8 x 1024 keys 9.4 -> 10.0 us, two
// streams of 1k keys 6.8 -> 7.3, 1 x 32768 keys 23.2 -> 22.2)
constexpr int kMergeBatch = 8;

// One workgroup per (piece of a sequence's keys, kv head), two of them (D = 64:
// four) on a CU.  Each wave streams every fourth tile of the piece through LDS of its
// own, without a barrier: the next K goes out when K is read, the next V when V
// is, so 16 KB of the wave's loads fly while it waits and 8 while it computes.
// The waves' sums meet at the end.  Partials in the workspace, per
// piece and kv head: [cap rows][D] sums, then [cap] (exponent base, row sum).
template <int D, int KT>
__global__ void __launch_bounds__(kFewWaves * 64, 2) paged_few_kernel(PagedArgs a, float* __restrict__ ws, unsigned* tickets, int slots, int cap) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    using F = Frag<KT>;
    using QF = typename F::type;
    constexpr int DS = D / 16, DT = D / 32;
    constexpr int NC = kFewTile * 2 * D / 1024;    // loads of a K (V) tile
    constexpr int RC = 1024 / (2 * D);             // rows of a load
    constexpr int TB = kFewTile * 2 * D;           // bytes of a K (V) tile, and of the rows of Q
    constexpr int OP = D + 4;                      // pitch of a row of sums
    constexpr int SUMS = kFewWaves * kFewRows * (OP + 2) * (int)sizeof(float);
    constexpr int RING = (kFewWaves * 2 + 1) * TB;
    __shared__ __attribute__((aligned(1024))) char lds[RING > SUMS ? RING : SUMS];

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.Hkv, piece = blockIdx.x / a.Hkv;
    const FewItem it = few_item(a, piece, slots);
    if (it.parts == 0) return;
    const int n = min(it.q.n, a.max_new), L = it.q.L, rows = n * a.G, past = L - it.q.n;
    const int tiles = (L + kFewTile - 1) / kFewTile;
    const int t0 = (int)((int64_t)it.part * tiles / it.parts), t1 = (int)((int64_t)(it.part + 1) * tiles / it.parts);

    // ---- this wave's tiles: t0 + w, + 4, ...
    const ConstInts table = (ConstInts)(uintptr_t)(a.table + (int64_t)it.s * a.table_stride);
    const int last_page = (L - 1) >> a.page_shift;
    const uint32_t qs = (uint32_t)(uintptr_t)(lds_char*)lds, ks = qs + (1 + 2 * w) * TB, vs = ks + TB;
    int koff[4], voff[4];                          // by row group: the swizzles repeat every 16 rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        koff[i] = dma_off<D, false>(lane, i * RC, (int)a.k_nb_slot);
        voff[i] = dma_off<D, true>(lane, i * RC, (int)a.v_nb_slot);
    }
    bool bad = false;
    int ids[2];                                    // pages of the two 16-key halves of the next tile to load
    auto fetch = [&](int t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) ids[i] = table[min((t * kFewTile + 16 * i) >> a.page_shift, last_page)];
    };
    auto issue = [&](int t, uint32_t dst, const char* pool, int64_t nb_page, int64_t nb_head, int64_t nb_slot, const int (&off)[4]) {
        uint64_t base[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool ok = (uint32_t)ids[i] < (uint32_t)a.n_pages;
            bad = bad || !ok;
            const int64_t id = ok ? ids[i] : 0;
            const int64_t slot = (t * kFewTile + 16 * i) & ((1 << a.page_shift) - 1);
            base[i] = uniform64((uint64_t)(uintptr_t)pool + id * nb_page + kvh * nb_head + slot * nb_slot);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            const int r = c * RC;                  // first row of the load, in its 16-key half r % 16
            dma16<true>(base[r / 16] + (uint64_t)(r % 16) * nb_slot, off[c % 4], dst + c * 1024);
        }
    };
    auto issue_k = [&](int t) { issue(t, ks, a.k, a.k_nb_page, a.k_nb_head, a.k_nb_slot, koff); };
    auto issue_v = [&](int t) { issue(t, vs, a.v, a.v_nb_page, a.v_nb_head, a.v_nb_slot, voff); };
    int t = t0 + w;
    if (t < t1) fetch(t);
    // the rows of Q, a quarter by each wave, laid out as K is; rows that are
    // not there are row 0 again (no one reads their results)
    {
        const uint64_t qb = uniform64((uint64_t)(uintptr_t)a.q + (int64_t)it.q.q0 * a.q_nb_t + (int64_t)kvh * a.G * a.q_nb_h);
#pragma unroll
        for (int i = 0; i < NC / kFewWaves; ++i) {
            const int c = w * (NC / kFewWaves) + i;
            const int r = c * RC + lane / (D / 8), row = r < rows ? r : 0;
            const int off = (row / a.G) * (int)a.q_nb_t + (row % a.G) * (int)a.q_nb_h;
            dma16<false>(qb, off + (((lane % (D / 8)) ^ k_swz<D>(r)) << 4), qs + c * 1024);
        }
    }
    if (t < t1) {
        issue_k(t);
        issue_v(t);
        wait_vm<2 * NC>();                         // Q
    } else {
        wait_vm<0>();
    }
    asm volatile("s_barrier" : : : "memory");
    const int k_off = k_lane_off<D>(lane), v_off = v_lane_off<D>(lane);
    QF qf[DS];
#pragma unroll
    for (int ds = 0; ds < DS; ++ds) qf[ds] = as_vec<QF>(lds_read((qs + k_off) ^ (ds << 5)));
    const int lim = l32 < rows ? min(L - 1, past + l32 / a.G) : -1;   // the last key the lane's row sees
    const float sl2 = a.scale * kLog2e;
    float m = -INFINITY, lsum = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    for (; t < t1; t += kFewWaves) {
        const bool more = t + kFewWaves < t1;
        if (more) fetch(t + kFewWaves);
        wait_vm<NC>();                             // K; V may still fly
        f32x16 s{};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) s = F::mma(as_vec<QF>(lds_read((ks + k_off) ^ (ds << 5))), qf[ds], s);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // K is read
            issue_k(t + kFewWaves);
        }
        const int k0 = t * kFewTile;
        const bool masked = k0 + kFewTile - 1 > min(L - 1, past);      // some row must not see some key
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = k0 + 8 * (r / 4) + 4 * half + r % 4 > lim ? -INFINITY : s[r];
        }
        float mx = fmaxf(s[0], s[1]);
#pragma unroll
        for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
        mx = max_swap32(mx) * sl2;
        if (__any(mx > m + kLazy)) {
            if (mx > m + kLazy) {
                const float alpha = __builtin_amdgcn_exp2f(m - mx);    // 0 while m = -inf
                lsum *= alpha;
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
                m = mx;
            }
        }
        const float nb = m == -INFINITY ? 0.0f : -m;
        uint32_t p[8];
#pragma unroll
        for (int r = 0; r < 8; ++r) {
            p[r] = pack2<KT>(__builtin_amdgcn_exp2f(fmaf(s[2 * r], sl2, nb)), __builtin_amdgcn_exp2f(fmaf(s[2 * r + 1], sl2, nb)));
            lsum = sum2<KT>(p[r], lsum);
        }
        if (more) wait_vm<NC>();                   // V; the next K may still fly
        else wait_vm<0>();
        const bool fix = masked && tile_not_finite<D, KT, kFewTile>(vs, lane);
#pragma unroll
        for (int kk = 0; kk < 2; ++kk) {
            const QF pf = as_vec<QF>(u32x4{p[4 * kk], p[4 * kk + 1], p[4 * kk + 2], p[4 * kk + 3]});
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) {
                const uint32_t v = ((vs + v_off) ^ (dt << 6)) + kk * 16 * 2 * D;
                u32x4 vf = v_bits<KT>(lds_at(v), lds_at(v + 8 * 2 * D));
                if (fix) vf = u32x4{finite2<KT>(vf.x), finite2<KT>(vf.y), finite2<KT>(vf.z), finite2<KT>(vf.w)};
                o[dt] = F::mma(as_vec<QF>(vf), pf, o[dt]);
            }
        }
        if (fix) add_not_finite<D, KT, kFewTile>(vs, k0, lim, half, o);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // V is read
            issue_v(t + kFewWaves);
        }
    }
    // ---- the waves' sums, in LDS, added in wave order
    const float lt = add_swap32(lsum);
    __syncthreads();
    float* const ow = (float*)lds;
    float* const ml = ow + kFewWaves * kFewRows * OP;
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *(float4*)(ow + (w * kFewRows + l32) * OP + dt * 32 + 8 * q4 + 4 * half) =
                make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
    if (half == 0) *(float2*)(ml + (w * kFewRows + l32) * 2) = make_float2(m, lt);
    const bool any_bad = __syncthreads_or(bad);
    auto piece_rsrc = [&](int part) {
        const uint32_t bytes = cap * (D + 2) * sizeof(float);
        return make_rsrc((const char*)ws + ((int64_t)(it.first + part) * a.Hkv + kvh) * bytes, bytes);
    };
    for (int i = tid; i < rows * (D / 4); i += kFewWaves * 64) {
        const int row = i / (D / 4), c = i % (D / 4);
        float M = -INFINITY;
#pragma unroll
        for (int k = 0; k < kFewWaves; ++k) M = fmaxf(M, ml[(k * kFewRows + row) * 2]);
        const float base = M == -INFINITY ? 0.0f : M;
        float den = 0.0f;
        float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll
        for (int k = 0; k < kFewWaves; ++k) {
            const float f = __builtin_amdgcn_exp2f(ml[(k * kFewRows + row) * 2] - base);   // 0 for a wave without keys
            const float4 v = *(const float4*)(ow + (k * kFewRows + row) * OP + 4 * c);
            den = fmaf(f, ml[(k * kFewRows + row) * 2 + 1], den);
            num.x = fmaf(f, v.x, num.x); num.y = fmaf(f, v.y, num.y);
            num.z = fmaf(f, v.z, num.z); num.w = fmaf(f, v.w, num.w);
        }
        if (it.parts > 1) {
            // agent-scope stores: coherent across the XCDs' L2 caches
            __builtin_amdgcn_raw_buffer_store_b128(
                u32x4{__float_as_uint(num.x), __float_as_uint(num.y), __float_as_uint(num.z), __float_as_uint(num.w)},
                piece_rsrc(it.part), (row * D + 4 * c) * 4, 0, kSc1);
            if (c == 0)
                __builtin_amdgcn_raw_buffer_store_b64(u32x2{any_bad ? kNanBits : __float_as_uint(M), __float_as_uint(den)},
                                                      piece_rsrc(it.part), (cap * D + row * 2) * 4, 0, kSc1);
            continue;
        }
        const float inv = den > 0.0f ? 1.0f / den : 0.0f;
        uint2 y = {pack2<KT>(num.x * inv, num.y * inv), pack2<KT>(num.z * inv, num.w * inv)};
        if (any_bad) y.x = y.y = 0x7fff7fffu;
        *(uint2*)(a.out + (int64_t)(it.q.q0 + row / a.G) * a.o_nb_t + (int64_t)(kvh * a.G + row % a.G) * a.o_nb_h + 8 * c) = y;
    }
    if (it.parts == 1) return;
    // ---- the last of the sequence's pieces adds their partials, in order:
    // every store of this workgroup is done before its ticket
    __builtin_amdgcn_s_waitcnt(0);
    __syncthreads();
    int* const last = (int*)lds;
    if (tid == 0) {
        unsigned* tk = tickets + it.s * a.Hkv + kvh;
        const unsigned old = __hip_atomic_fetch_add(tk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        *last = old == (unsigned)(it.parts - 1);
        if (*last) __hip_atomic_store(tk, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
    }
    __syncthreads();
    if (!*last) return;
    for (int i = tid; i < rows * (D / 4); i += kFewWaves * 64) {
        const int row = i / (D / 4), c = i % (D / 4);
        float M = -INFINITY, den = 0.0f;
        float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        bool nan = false;
        for (int p0 = 0; p0 < it.parts; p0 += kMergeBatch) {
            // a batch's loads go out together, one round trip each; those past
            // the last piece lie outside their buffer and read nothing
            u32x2 e[kMergeBatch];
            u32x4 v[kMergeBatch];
#pragma unroll
            for (int u = 0; u < kMergeBatch; ++u) {
                const bool in = p0 + u < it.parts;
                const BufRsrc rs = piece_rsrc(in ? p0 + u : 0);
                e[u] = __builtin_amdgcn_raw_buffer_load_b64(rs, in ? (cap * D + row * 2) * 4 : 0x7ffffff0, 0, kSc1);
                v[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, in ? (row * D + 4 * c) * 4 : 0x7ffffff0, 0, kSc1);
            }
#pragma unroll
            for (int u = 0; u < kMergeBatch; ++u) asm volatile("" : "+v"(e[u]), "+v"(v[u]));
            float mb = M;
#pragma unroll
            for (int u = 0; u < kMergeBatch; ++u) {
                const bool hit = e[u].x == kNanBits;
                nan = nan || hit;
                if (hit || p0 + u >= it.parts) {              // nothing to add
                    e[u] = u32x2{0xff800000u, 0u};
                    v[u] = u32x4{0u, 0u, 0u, 0u};
                }
                mb = fmaxf(mb, __uint_as_float(e[u].x));
            }
            const float base = mb == -INFINITY ? 0.0f : mb;
            const float f0 = __builtin_amdgcn_exp2f(M - base);
            M = mb;
            den *= f0;
            num.x *= f0; num.y *= f0; num.z *= f0; num.w *= f0;
#pragma unroll
            for (int u = 0; u < kMergeBatch; ++u) {
                const float f = __builtin_amdgcn_exp2f(__uint_as_float(e[u].x) - base);
                den = fmaf(f, __uint_as_float(e[u].y), den);
                num.x = fmaf(f, __uint_as_float(v[u].x), num.x);
                num.y = fmaf(f, __uint_as_float(v[u].y), num.y);
                num.z = fmaf(f, __uint_as_float(v[u].z), num.z);
                num.w = fmaf(f, __uint_as_float(v[u].w), num.w);
            }
        }
        const float inv = den > 0.0f ? 1.0f / den : 0.0f;
        uint2 y = {pack2<KT>(num.x * inv, num.y * inv), pack2<KT>(num.z * inv, num.w * inv)};
        if (nan) y.x = y.y = 0x7fff7fffu;
        *(uint2*)(a.out + (int64_t)(it.q.q0 + row / a.G) * a.o_nb_t + (int64_t)(kvh * a.G + row % a.G) * a.o_nb_h + 8 * c) = y;
    }
}

// ----------------------------------------------------------- many rows

constexpr int kBN = 64;            // keys per tile
constexpr int kRowsWave = 32;
constexpr int kWaves = 8;          // two per SIMD
constexpr int kRowsWG = kRowsWave * kWaves;
constexpr int kStages = 4;         // LDS ring: tile j + 3 loads while tile j is computed
constexpr int kMaxKs = 16;         // key splits per row tile
constexpr int kMinPiece = 8;       // key tiles of a piece at least

// A piece of a row tile's keys: row tile rt of the sequence, piece `ks` of
// `n_ks`; n_ks = 0: none.  first: the row tile's piece 0 of the call.
struct ManyItem {
    Seq q;
    int s, rt, ks, n_ks, first;
};
__device__ __forceinline__ int many_row_tiles(const PagedArgs& a, const Seq& q) {
    const int n = min(q.n, a.max_new);
    return n * a.G > kFewRows ? (n * a.G + kRowsWG - 1) / kRowsWG : 0;
}
// Key tiles that row tile rt of a sequence sees
__device__ __forceinline__ int many_key_tiles(const PagedArgs& a, const Seq& q, int rt) {
    const int n = min(q.n, a.max_new);
    const int t_hi = min(n * a.G, (rt + 1) * kRowsWG) - 1;
    return (max(0, min(q.L, q.L - q.n + t_hi / a.G + 1)) + kBN - 1) / kBN;
}
// Item `item` of the call: a row tile (TILE) or a piece of one; the last row
// tiles of a sequence (the longest) come first.  Every row tile is cut into the same number of
// pieces, the one that leaves the least for the fullest CU (one workgroup at a
// time each): rounds of workgroups times their share of the keys and what a
// piece costs beside them, about kMinPiece tiles.  max_wgs: the most workgroups
// that the launch's grid and workspace hold of split row tiles (0: none is
// split).  By whole waves.
template <bool TILE>
__device__ __forceinline__ ManyItem many_item(const PagedArgs& a, int item, int n_cu, int max_wgs) {
    const int lane = threadIdx.x & 63;
    int rts = 0;
    float work = 0.0f;
    for (int i = 0; i < a.n_seq; i += 64) {
        const int s = i + lane;
        const Seq q = seq_of(a, min(s, a.n_seq - 1));
        const int r = s < a.n_seq ? many_row_tiles(a, q) : 0;
        rts += r;
        work += r > 0 ? (float)r * (float)many_key_tiles(a, q, r - 1) : 0.0f;
    }
#pragma unroll
    for (int m = 32; m >= 1; m >>= 1) {
        rts += __shfl_xor(rts, m, 64);
        work += __shfl_xor(work, m, 64);
    }
    ManyItem it{};
    if (rts == 0) return it;
    const int kt = (int)(work / (float)rts);       // key tiles of a row tile
    const int wgs = rts * a.Hkv;
    // lane x: x + 1 pieces
    const int x = min(lane, kMaxKs - 1) + 1;
    int cost = 0x7fffffff;
    if (x == 1 || (wgs * x <= max_wgs && kt >= kMinPiece * x))
        cost = ((wgs * x + n_cu - 1) / n_cu) * ((kt + x - 1) / x + (x > 1 ? kMinPiece : 0));
    int best = cost;
#pragma unroll
    for (int m = 8; m >= 1; m >>= 1) best = min(best, __shfl_xor(best, m, 64));
    const int sp = __ffsll((unsigned long long)__ballot(cost == best));
    const int tile = TILE ? item : item / sp;
    it.ks = TILE ? 0 : item - tile * sp;
    int base = 0;
    for (int i = 0; i < a.n_seq; i += 64) {
        const int s = i + lane;
        const Seq q = seq_of(a, min(s, a.n_seq - 1));
        const int r = s < a.n_seq ? many_row_tiles(a, q) : 0;
        const int end = wave_scan(r);
        const uint64_t hit = __ballot(tile >= base + end - r && tile < base + end);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            it.q.q0 = lane_of(q.q0, l);
            it.q.n = lane_of(q.n, l);
            it.q.L = lane_of(q.L, l);
            it.s = i + l;
            it.rt = base + lane_of(end, l) - 1 - tile;
            it.first = tile * sp;
            it.n_ks = sp;
            return it;
        }
        base += lane_of(end, 63);
    }
    return it;
}

// One workgroup per (piece of a row tile's keys, kv head): 8 waves x 32 rows
// that share every K / V tile.
template <int D, int KT>
__global__ void __launch_bounds__(kWaves * 64) paged_many_kernel(PagedArgs a, float* __restrict__ ws, int n_cu, int max_wgs) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    using F = Frag<KT>;
    using QF = typename F::type;
    constexpr int DS = D / 16, DT = D / 32;
    constexpr int ROW = 2 * D;
    constexpr int TB = kBN * ROW;                  // bytes of a K (V) tile
    constexpr int NI = TB / 1024 / kWaves;         // loads of a K (V) tile per wave
    constexpr int RC = 1024 / ROW;                 // rows of a load
    constexpr int STAGE = 2 * TB;
    constexpr int NLD = 2 * NI;
    __shared__ __attribute__((aligned(1024))) char lds[kStages * STAGE];
    __shared__ int fix;                            // the last tile found to hold a V that is not finite

    const int tid = threadIdx.x, lane = tid & 63, half = lane >> 5, l32 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int kvh = blockIdx.x % a.Hkv;
    if (tid == 0) fix = -1;                        // before the first tile's barrier
    const ManyItem it = many_item<false>(a, blockIdx.x / a.Hkv, n_cu, max_wgs);
    if (it.n_ks == 0) return;
    const int L = it.q.L, past = L - it.q.n, G = a.G;
    const int rows = min(it.q.n, a.max_new) * G;
    const int wr0 = it.rt * kRowsWG + w * kRowsWave;
    const int n_tiles_rt = many_key_tiles(a, it.q, it.rt);
    const int j_lo = (int)((int64_t)it.ks * n_tiles_rt / it.n_ks);
    const int n_tiles = (int)((int64_t)(it.ks + 1) * n_tiles_rt / it.n_ks) - j_lo;
    const int kb0 = j_lo * kBN;
    // keys [0, kend_w) are seen by some row of the wave, keys up to lim_w by every row
    const bool wave_live = wr0 < rows;
    const int kend_w = wave_live ? max(0, min(L, past + (min(wr0 + kRowsWave, rows) - 1) / G + 1)) : 0;
    const int lim_w = min(L - 1, past + min(wr0, rows - 1) / G);

    // ---- tile loads: load i of K (V) covers rows RC * (i * 8 + w) .. of the
    // tile, inside one 16-key group
    const ConstInts table = (ConstInts)(uintptr_t)(a.table + (int64_t)it.s * a.table_stride);
    const int last_page = max(0, (L - 1) >> a.page_shift);
    const int r0w = RC * w;                                   // first row of the wave's loads, + i * 8 * RC
    const int koff = dma_off<D, false>(lane, r0w, (int)a.k_nb_slot);
    const int voff = dma_off<D, true>(lane, r0w, (int)a.v_nb_slot);
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds;
    bool bad = false;
    int ids[NI];
    auto fetch = [&](int j) {
#pragma unroll
        for (int i = 0; i < NI; ++i) ids[i] = table[min((kb0 + j * kBN + i * kWaves * RC + r0w) >> a.page_shift, last_page)];
    };
    // the loads of tile j (K, then V); past the last tile the last one's again,
    // to a stage that nobody reads any more, so that every tile counts the same
    auto issue = [&](int j) {
        const uint32_t st = lds0 + (j % kStages) * STAGE + w * 1024;
        uint64_t kb[NI], vb[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const bool ok = (uint32_t)ids[i] < (uint32_t)a.n_pages;
            bad = bad || !ok;
            const int64_t id = ok ? ids[i] : 0;
            const int64_t slot = (kb0 + j * kBN + i * kWaves * RC + r0w) & ((1 << a.page_shift) - 1);
            kb[i] = uniform64((uint64_t)(uintptr_t)a.k + id * a.k_nb_page + kvh * a.k_nb_head + slot * a.k_nb_slot);
            vb[i] = uniform64((uint64_t)(uintptr_t)a.v + id * a.v_nb_page + kvh * a.v_nb_head + slot * a.v_nb_slot);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) dma16<false>(kb[i], koff, st + i * kWaves * 1024);
#pragma unroll
        for (int i = 0; i < NI; ++i) dma16<false>(vb[i], voff, st + TB + i * kWaves * 1024);
    };
    const int row = wr0 + l32;
    const bool qok = row < rows;
    const int tcol = (qok ? row : rows - 1) / G;
    QF qf[DS];
    float m = -INFINITY, lsum = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    if (n_tiles > 0) {                                        // uniform
        fetch(0);
        issue(0);
        load_q<D>(a, it.q.q0, kvh, row, rows, half, qf);
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) asm volatile("" : "+v"(qf[ds]));   // Q has landed, and tile 0
        fetch(1);
        issue(1);
        fetch(2);
        issue(2);
        fetch(3);
        const float sl2 = a.scale * kLog2e;
        const int k_off = k_lane_off<D>(lane), v_off = v_lane_off<D>(lane);
        const int lim = min(L - 1, past + tcol);              // the last key the lane's row sees
        auto stage = [&](int j) { return lds0 + (j % kStages) * STAGE; };
        auto read_k128 = [&](uint32_t ka, int ds, int kt) {
            return lds_read((ka ^ (ds << 5)) + kt * 32 * ROW);
        };
        auto scores = [&](uint32_t ka, f32x16 (&s)[2]) {
#pragma unroll
            for (int ds = 0; ds < DS; ++ds)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt)
                    s[kt] = F::mma(as_vec<QF>(read_k128(ka, ds, kt)), qf[ds], ds == 0 ? f32x16{} : s[kt]);
        };
        auto apply_mask = [&](f32x16 (&s)[2], int k0) {
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[kt][r] = k0 + kt * 32 + 8 * (r / 4) + 4 * half + r % 4 > lim ? -INFINITY : s[kt][r];
        };
        auto rowmax = [&](const f32x16 (&s)[2]) {
            float mr = fmaxf(fmaxf(s[0][0], s[0][1]), s[0][2]);
#pragma unroll
            for (int r = 3; r < 15; r += 2) mr = fmaxf(fmaxf(mr, s[0][r]), s[0][r + 1]);
            mr = fmaxf(mr, s[0][15]);
#pragma unroll
            for (int r = 0; r < 16; r += 2) mr = fmaxf(fmaxf(mr, s[1][r]), s[1][r + 1]);
            return max_swap32(mr) * sl2;
        };
        auto rescale = [&](float mx) {
            if (__any(mx > m + kLazy)) {
                if (mx > m + kLazy) {
                    const float alpha = __builtin_amdgcn_exp2f(m - mx);   // 0 while m = -inf
                    lsum *= alpha;
#pragma unroll
                    for (int dt = 0; dt < DT; ++dt) o[dt] *= alpha;
                    m = mx;
                }
            }
        };
        // Software pipeline over the key tiles: a step raises the running max
        // to tile j's, then runs one straight line of matrix-core slots, the
        // scores of tile j + 1, then P.V of tile j, with the softmax of tile j
        // and the operand reads placed between them by scheduling fences so
        // that the VALU issues while the matrix cores run.
        const int n_live = max(0, min(n_tiles, (kend_w - kb0 + kBN - 1) / kBN));   // the wave's tiles
        auto needs_mask = [&](int j) { return kb0 + j * kBN + kBN - 1 > lim_w; };
        constexpr int NQ = 2 * DS, NP = 4 * DT, NS = NQ + NP;
        constexpr int KAHEAD = 2, VAHEAD = 2;                 // operand reads ahead of their slot
        auto block = [&](const f32x16 (&cur)[2], f32x16 (&nxt)[2], uint32_t ka, uint32_t va) {
            const float nb = m == -INFINITY ? 0.0f : -m;      // no visible key yet: every s is -inf
            u32x4 kf[NQ], vf[NP];
            float pe[32];
            uint32_t pp[16];
            float ps = lsum;
            auto read_k = [&](int i) { kf[i] = read_k128(ka, i >> 1, i & 1); };
            auto read_v = [&](int p) {
                const uint32_t v = (va ^ ((p % DT) << 6)) + (p / DT) * 16 * ROW;
                vf[p] = v_bits<KT>(lds_at(v), lds_at(v + 8 * ROW));
            };
            // score v: its fma in slot fslot(v), the exp2 a slot later, the pack
            // of a pair three slots after its second fma, its sum one later
            auto fslot = [](int v) { return v * (NS - 8) / 32; };
            auto pair_slot = [&](int i) { return fslot(2 * i + 1) + 3; };
            static_assert(((31 * (NS - 8)) / 32) + 3 < NQ + 3 * DT, "chunk 3 packed before its P.V");
            auto valu_slot = [&](int sl) {
#pragma unroll
                for (int v = 0; v < 32; ++v) {
                    if (fslot(v) == sl) pe[v] = fmaf(cur[v >> 4][v & 15], sl2, nb);
                    if (fslot(v) + 1 == sl) pe[v] = __builtin_amdgcn_exp2f(pe[v]);
                }
#pragma unroll
                for (int i = 0; i < 16; ++i) {
                    if (pair_slot(i) == sl) pp[i] = pack2<KT>(pe[2 * i], pe[2 * i + 1]);
                    if (pair_slot(i) + 1 == sl) ps = sum2<KT>(pp[i], ps);
                }
            };
#pragma unroll
            for (int i = 0; i < KAHEAD; ++i) read_k(i);
#pragma unroll
            for (int sl = 0; sl < NS; ++sl) {
                if (sl < NQ) {
                    const int ds = sl >> 1, kt = sl & 1;
                    nxt[kt] = F::mma(as_vec<QF>(kf[sl]), qf[ds], ds == 0 ? f32x16{} : nxt[kt]);
                    if (sl + KAHEAD < NQ) read_k(sl + KAHEAD);
                } else {
                    const int p = sl - NQ, c = p / DT;
                    const QF pf = as_vec<QF>(u32x4{pp[4 * c], pp[4 * c + 1], pp[4 * c + 2], pp[4 * c + 3]});
                    o[p % DT] = F::mma(as_vec<QF>(vf[p]), pf, o[p % DT]);
                }
                if (sl - NQ + VAHEAD >= 0 && sl - NQ + VAHEAD < NP) read_v(sl - NQ + VAHEAD);
                valu_slot(sl);
                __builtin_amdgcn_sched_barrier(0);
            }
            lsum = ps;
        };
        // A tile that some row of the workgroup must not see all of: each wave
        // looks at its share of V, and where a value is not finite every row adds
        // the ones that it sees and the tile goes on with zeros in their places
        // (the order of the barriers is the workgroup's; seen by no other tile).
        const int lim_wg = min(L - 1, past + min(it.rt * kRowsWG, rows - 1) / G);
        auto fix_tile = [&](int j) {
            const uint32_t vs = stage(j) + TB;
            constexpr int NF = TB / 1024 / kWaves;
            bool nf = false;
#pragma unroll
            for (int i = 0; i < NF; ++i) nf = nf || chunk_not_finite<KT>(lds_read(vs + (i * kWaves + w) * 1024 + lane * 16));
            if (__any(nf)) *(volatile __attribute__((address_space(3))) int*)&fix = j;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
            if (*(volatile __attribute__((address_space(3))) int*)&fix != j) return;
            add_not_finite<D, KT, kBN>(vs, kb0 + j * kBN, qok ? lim : -1, half, o);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                auto* p = lds_vec(vs + (i * kWaves + w) * 1024 + lane * 16);
                const u32x4 x = *p;
                *p = u32x4{finite2<KT>(x.x), finite2<KT>(x.y), finite2<KT>(x.z), finite2<KT>(x.w)};
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
        };
        // K of tile 0 has landed (its V and tiles 1, 2 may still fly)
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(NI + 2 * NLD) : "memory");
        f32x16 sa[2], sb[2];
        float mx = 0.0f;
        if (n_live > 0) {
            scores(stage(0) + k_off, sa);
            if (needs_mask(0)) apply_mask(sa, kb0);
            mx = rowmax(sa);
        }
        auto step = [&](int j, const f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
            // K of tile j + 1 and V of tile j have landed, and every wave is done
            // with tile j - 1, whose stage tile j + 3 now takes
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(NI + NLD) : "memory");
            issue(j + 3);
            fetch(j + 4);
            if (j < n_live) rescale(mx);                      // wave-uniform
            if (kb0 + j * kBN + kBN - 1 > lim_wg) fix_tile(j);
            if (j < n_live) {
                uint32_t va = stage(j) + TB + v_off, ka = stage(j + 1) + k_off;
                asm volatile("" : "+v"(va), "+v"(ka));
                // tile j + 1's scores are computed whether or not the wave sees
                // it: past its last tile no step reads them
                block(cur, nxt, ka, va);
                if (needs_mask(j + 1)) apply_mask(nxt, kb0 + (j + 1) * kBN);
                mx = rowmax(nxt);
            }
        };
        int j = 0;
        for (; j + 1 < n_tiles; j += 2) {
            step(j, sa, sb);
            step(j + 1, sb, sa);
        }
        if (j < n_tiles) step(j, sa, sb);
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");   // the padding tiles' loads
    }
    // ---- normalize and write (lanes l and l ^ 32 summed different keys), or
    // the piece's partial: sums, and (exponent base, row sum)
    const float lt = add_swap32(lsum);
    const bool any_bad = __syncthreads_or(bad);
    if (!qok) return;
    if (it.n_ks == 1) {
        char* const orow = a.out + (int64_t)(it.q.q0 + row / G) * a.o_nb_t + (int64_t)(kvh * G + row % G) * a.o_nb_h;
        const float inv = lt > 0.0f ? 1.0f / lt : 0.0f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                uint2 y = {pack2<KT>(o[dt][4 * q4] * inv, o[dt][4 * q4 + 1] * inv),
                           pack2<KT>(o[dt][4 * q4 + 2] * inv, o[dt][4 * q4 + 3] * inv)};
                if (any_bad) y.x = y.y = 0x7fff7fffu;
                *(uint2*)(orow + (dt * 32 + 8 * q4 + 4 * half) * 2) = y;
            }
        return;
    }
    float* const pr = ws + ((int64_t)(it.first + it.ks) * a.Hkv + kvh) * kRowsWG * (D + 2);
    const int r = w * kRowsWave + l32;
    if (half == 0) *(uint2*)(pr + kRowsWG * D + 2 * r) = make_uint2(any_bad ? kNanBits : __float_as_uint(m), __float_as_uint(lt));
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int q4 = 0; q4 < 4; ++q4)
            *(float4*)(pr + r * D + dt * 32 + 8 * q4 + 4 * half) =
                make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
}

// The pieces' sums of a row tile's rows: D / 4 threads a row.
template <int D, int KT>
__global__ void __launch_bounds__(256) paged_many_merge_kernel(PagedArgs a, const float* __restrict__ ws, int n_cu, int max_wgs) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    constexpr int C = D / 4, R = 256 / C;          // rows of a workgroup
    const int kvh = blockIdx.x % a.Hkv;
    const ManyItem it = many_item<true>(a, blockIdx.x / a.Hkv, n_cu, max_wgs);
    if (it.n_ks <= 1) return;
    const int r = blockIdx.y * R + threadIdx.x / C, c = threadIdx.x % C;
    const int row = it.rt * kRowsWG + r;
    if (row >= min(it.q.n, a.max_new) * a.G) return;
    constexpr int64_t PS = kRowsWG * (D + 2);
    const float* pr = ws + ((int64_t)it.first * a.Hkv + kvh) * PS;
    float2 e[kMaxKs];
#pragma unroll
    for (int k = 0; k < kMaxKs; ++k) e[k] = *(const float2*)(pr + (int64_t)min(k, it.n_ks - 1) * a.Hkv * PS + kRowsWG * D + 2 * r);
    float M = -INFINITY;
    bool bad = false;
#pragma unroll
    for (int k = 0; k < kMaxKs; ++k) {
        const bool b = __float_as_uint(e[k].x) == kNanBits;
        bad = bad || b;
        M = fmaxf(M, b ? -INFINITY : e[k].x);
    }
    const float base = M == -INFINITY ? 0.0f : M;
    float den = 0.0f;
    float4 num = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
    for (int k = 0; k < it.n_ks; ++k) {
        const float2 ek = *(const float2*)(pr + (int64_t)k * a.Hkv * PS + kRowsWG * D + 2 * r);
        const float f = __builtin_amdgcn_exp2f(ek.x - base);
        const float4 v = *(const float4*)(pr + (int64_t)k * a.Hkv * PS + r * D + 4 * c);
        den = fmaf(f, ek.y, den);
        num.x = fmaf(f, v.x, num.x); num.y = fmaf(f, v.y, num.y);
        num.z = fmaf(f, v.z, num.z); num.w = fmaf(f, v.w, num.w);
    }
    const float inv = den > 0.0f ? 1.0f / den : 0.0f;
    uint2 y = {pack2<KT>(num.x * inv, num.y * inv), pack2<KT>(num.z * inv, num.w * inv)};
    if (bad) y.x = y.y = 0x7fff7fffu;
    *(uint2*)(a.out + (int64_t)(it.q.q0 + row / a.G) * a.o_nb_t + (int64_t)(kvh * a.G + row % a.G) * a.o_nb_h + 8 * c) = y;
}

template <int D, int KT>
hipError_t launch_paged(const PagedArgs& a, const PagedPlan& p, float* ws, unsigned* tickets, hipStream_t s) {
    hipError_t e = hipSuccess;
    if (p.many_tiles > 0) {
        hipLaunchKernelGGL((paged_many_kernel<D, KT>), dim3(p.many_pieces * a.Hkv), dim3(kWaves * 64), 0, s, a, ws, p.n_cu, p.max_wgs);
        if ((e = hipGetLastError()) != hipSuccess) return e;
        if (p.many_split) {
            hipLaunchKernelGGL((paged_many_merge_kernel<D, KT>), dim3(p.many_tiles * a.Hkv, kRowsWG * D / 4 / 256), dim3(256), 0, s, a, ws, p.n_cu, p.max_wgs);
            if ((e = hipGetLastError()) != hipSuccess) return e;
        }
    }
    if (p.few_pieces > 0) {
        hipLaunchKernelGGL((paged_few_kernel<D, KT>), dim3(p.few_pieces * a.Hkv), dim3(kFewWaves * 64), 0, s, a, ws, tickets, p.few_slots, p.few_cap);
        e = hipGetLastError();
    }
    return e;
}

}  // namespace

// What a call of these shapes may need: the lengths are on the device, so
// every count here is the most there can be, and workgroups beyond the work
// there is end at once.
PagedPlan paged_plan(const PagedArgs& a, int n_cu) {
    PagedPlan p{};
    p.n_cu = n_cu;
    const int64_t rows = (int64_t)a.max_new * a.G, all = (int64_t)a.n_tok * a.G;
    const int64_t max_keys = (int64_t)a.max_pages << a.page_shift;
    // every sequence brings max_new tokens where their number says so
    const bool even = (int64_t)a.n_seq * a.max_new == a.n_tok;
    if (rows > kFewRows) {
        const int64_t seqs = std::min<int64_t>(a.n_seq, all / (kFewRows + 1));
        const int64_t tiles = even ? (int64_t)a.n_seq * ((rows + kRowsWG - 1) / kRowsWG) : all / kRowsWG + seqs;
        const int64_t key_tiles = (max_keys + kBN - 1) / kBN;
        p.many_tiles = (int)tiles;
        // at most four workgroups per CU in all where row tiles are split
        p.many_split = key_tiles >= 2 * kMinPiece && (!even || 2 * tiles * a.Hkv <= 4 * n_cu);
        p.max_wgs = p.many_split ? 4 * n_cu : 0;
        p.many_pieces = (int)std::max<int64_t>(tiles, p.max_wgs / a.Hkv);
    }
    if (rows <= kFewRows || !even) {
        p.few_cap = (int)std::min<int64_t>(rows, kFewRows);
        // Half the workgroups that fit a CU, so that fewer partials are added and
        // no CU's share of the bytes is less (1 x 32768 keys 29.3 -> 22.3 us, 64 x 4096
        // 88.8 -> 83.8); all of them where the sequences are too many to be cut evenly
        // into that few (48 of 500 to 8000 keys: 94.2 -> 79.3)
        const int slots = n_cu * (a.d == 64 ? 2 : 1);
        p.few_slots = std::max(1, (2 * a.n_seq * a.Hkv > slots ? 2 : 1) * slots / a.Hkv);
        const int64_t seq_tiles = (max_keys + kFewTile - 1) / kFewTile;
        p.few_split = seq_tiles > kFewMin;
        p.few_pieces = (int)std::min<int64_t>(p.few_slots + (int64_t)a.n_seq, a.n_seq * ((seq_tiles + kFewMin - 1) / kFewMin));
    }
    return p;
}
size_t paged_ws_bytes(const PagedArgs& a, const PagedPlan& p) {
    const size_t many = p.many_split ? (size_t)p.many_pieces * a.Hkv * kRowsWG * (a.d + 2) * sizeof(float) : 0;
    const size_t few = p.few_split ? (size_t)p.few_pieces * a.Hkv * p.few_cap * (a.d + 2) * sizeof(float) : 0;
    return std::max(many, few);                    // one after the other on the stream
}

hipError_t launch_paged_attn(const PagedArgs& a, const PagedPlan& p, float* ws, unsigned* tickets, hipStream_t s) {
    if (a.d == 64)
        return a.type == VVA_TYPE_F16 ? launch_paged<64, VVA_TYPE_F16>(a, p, ws, tickets, s) : launch_paged<64, VVA_TYPE_BF16>(a, p, ws, tickets, s);
    return a.type == VVA_TYPE_F16 ? launch_paged<128, VVA_TYPE_F16>(a, p, ws, tickets, s) : launch_paged<128, VVA_TYPE_BF16>(a, p, ws, tickets, s);
}

}  // namespace vva
