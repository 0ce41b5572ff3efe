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
// proposed ones) go through few_piece, which is bound by the cache's bytes, the
// others through many_share, which is bound by the matrix cores.  A call whose
// max_new tokens are few rows is paged_few_kernel; one of n_seq * max_new tokens
// paged_many_kernel, which then takes short sequences too; any other may bring
// both kinds and is paged_mixed_kernel, which runs them side by side.
//
// Reached, of a copy's 4.9 TB/s and a large product's 1175 TFLOP/s: single
// tokens 5.5 TB/s (48 sequences of 500 to 8000 keys, 405 MB, 73 us); 2048 tokens
// behind 28672 keys 976 to 1026 TFLOP/s from GPU to GPU (893 to 850 us), 512 behind
// 15872 829 to 868 (143 to 136).  Over Q8_0 pages: the 48 sequences (216 MB) 46.4 us,
// one of 30k keys 14.5 (16-bit pages 17.4); the chunks 880 to 922 and 142 to 147 us.
//
// Both compute, per 32 rows and a tile of keys, with
// v_mfma_f32_32x32x16_{f16,bf16} (layouts in mfma_ops.hpp):
//   S^T[key][row] = K . Q^T    Q^T in registers; a lane owns one query row
//   softmax                    fp32, exp2 domain, scale folded into the exp's
//                              fma; the running max of a row is raised only
//                              when a tile's max passes it by more than 2^8
//                              (rescales are rare), so p <= 2^8
//   O^T[dim][row] += V^T . P^T P converted in place from the accumulators: the
//                              key order of a step is the one they have
// P is rounded to the pages' type, as the output itself is: a relative 2^-8 at
// most in BF16.  F16 has fewer exponents than a long row has sizes of weights,
// so its P carry a factor of 2^7 (p <= 2^15), which leaves with the row sum:
// weights down to 2^-21 of the row's largest are rounded by a relative 2^-11,
// smaller ones by 2^-32 of it (without the factor a weight of e^-17 is 44 % off,
// and a long cache has many).  The row sum adds the rounded values, so the weights
// of a row sum to one.  Few rows of BF16 pages, which wait for the cache's bytes,
// multiply what the rounding leaves as well, in a second product with the same V:
// their P are within 2^-15 (48 sequences of 500 to 8000 keys 72.1 -> 72.9 us).
// Many rows, with 250 of 256 registers in use and the arithmetic their bound,
// round once.
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
//
// Q8_0 pages (paged_q8.hpp) take the F16 products.  Few rows keep the codes in LDS
// and convert them as operands; many rows convert each tile once, into the LDS tile
// that F16 pages are loaded into, so K and V are rounded to F16 there (a relative
// 2^-11 at most; with the probabilities' and the result's rounding an F16 result is
// off by 4.2e-4 of its size, of which the last alone is 2.1e-4).
#include "vva_internal.hpp"

#include <algorithm>
#include <type_traits>

namespace vva {

namespace {

#include "wave_ops.hpp"
#include "mfma_ops.hpp"
#include "paged_ops.hpp"

typedef float f32x4 __attribute__((ext_vector_type(4)));

constexpr float kLazy = 8.0f;      // running-max slack in log2 units
// The type that the products take: the pages' own, F16 for Q8_0
template <int KT> constexpr int kComp = KT == VVA_TYPE_Q8_0 ? VVA_TYPE_F16 : KT;
// log2 of the factor that P carries
template <int KT> constexpr float kLift = KT == VVA_TYPE_F16 ? 7.0f : 0.0f;
constexpr int kFewRows = 32;       // rows of a sequence and kv head that paged_few_kernel takes
// Exponent base of a partial whose keys lie in a page outside the pool, compared as
// bits.  No sums' own base is one: a running max is raised only where a score is
// greater, which none is to or from a NaN.
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
// this lane, from the hardware: no register holds it meanwhile
__device__ __forceinline__ int lane_id() {
    int x;
    asm volatile("v_mbcnt_lo_u32_b32 %0, -1, 0\n\tv_mbcnt_hi_u32_b32 %0, -1, %0" : "=v"(x));
    return x;
}
__device__ __forceinline__ int uni(int x) { return __builtin_amdgcn_readfirstlane(x); }
__device__ __forceinline__ float uni(float x) { return __int_as_float(__builtin_amdgcn_readfirstlane(__float_as_int(x))); }
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
// Two probabilities x, y >= 0 in two BF16 parts each: the upper half of the
// float's bits, and the rest.  The rest is above 0 wherever x is (x goes into it
// a step of 2^-23 larger, as into the row sum), so that the products with an
// infinite V have its sign alone.
__device__ __forceinline__ void split2_bf16(float x, float y, uint32_t& p, uint32_t& rest) {
    const uint32_t hx = __float_as_uint(x) & 0xffff0000u, hy = __float_as_uint(y) & 0xffff0000u;
    constexpr float up = 1.0f + 0x1p-23f;
    p = (hx >> 16) | hy;
    rest = pack2<VVA_TYPE_BF16>(fmaf(x, up, -__uint_as_float(hx)), fmaf(y, up, -__uint_as_float(hy)));
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

// Q fragment as the products take it, from the 16 bytes of a row
template <int KT, int OT>
__device__ __forceinline__ typename Frag<KT>::type q_frag(u32x4 x) {
    if constexpr (OT != KT) {                      // BF16 rows over Q8_0 pages: F16 holds their 8 bits
#pragma unroll
        for (int e = 0; e < 4; ++e) x[e] = pack2<KT>(__uint_as_float(x[e] << 16), __uint_as_float(x[e] & 0xffff0000u));
    }
    return as_vec<typename Frag<KT>::type>(x);
}
// The kernel's arguments, read again from their segment: each phase loads the
// few that it needs (they hit the scalar cache), so that not all of them are
// held, and spilled, through the key tiles.
__device__ __forceinline__ const PagedArgs& fresh_args() {
    uint64_t p = (uint64_t)(uintptr_t)(const char*)__builtin_amdgcn_kernarg_segment_ptr();
    asm volatile("" : "+s"(p));
    return *(const PagedArgs*)(const __attribute__((address_space(4))) PagedArgs*)(uintptr_t)p;
}

// ------------------------------------------------------------ few rows

constexpr int kFewWaves = 4;       // of a workgroup of paged_few_kernel (Q8_0 pages, 16 rows: 8)
constexpr int kFewTile = 32;
constexpr int kMaxWgs = 256;       // workgroups of the many rows at most
constexpr int kFewCost = 4;        // what a piece costs beside its keys, in tiles
constexpr int kFewSnap = 8;        // cuts this near an end of a sequence, in tiles, are moved there

// Tiles of sequence q that few_piece works on
__device__ __forceinline__ int few_tiles(const PagedArgs& a, const Seq& q) {
    const int n = min(q.n, a.max_new);
    return n > 0 && n * a.G <= kFewRows ? max(1, (q.L + kFewTile - 1) / kFewTile) : 0;
}
__device__ __forceinline__ int few_weight(const PagedArgs& a, const Seq& q) {
    const int t = few_tiles(a, q);
    return t > 0 ? t + kFewCost : 0;
}
// Length of the axis on which a kv head's sequences lie one after the other,
// each as long as its tiles and what a piece costs beside them.  `mine`: the
// lane's own of the first 64.  By whole waves.
__device__ __forceinline__ int few_axis(const PagedArgs& a, const Seq& mine) {
    const int lane = threadIdx.x & 63;
    int total = lane < a.n_seq ? few_weight(a, mine) : 0;
    for (int s = lane + 64; s < a.n_seq; s += 64) total += few_weight(a, seq_of(a, s));
    return wave_total(total);
}

// x / n for a uniform p >= 0 whose quotient a float holds
__device__ __forceinline__ int part_of(int p, int n) {
    int k = uni((int)((float)p * __builtin_amdgcn_rcpf((float)n))), r = p - k * n;   // within one or two of it
    while (r < 0) --k, r += n;
    while (r >= n) ++k, r -= n;
    return k;
}
// An axis cut into n equal shares, a workgroup's each.  A cut at place b inside
// the item [x, x + len) that is near one of its ends is moved there.
struct Shares {
    int share, n, snap;
    __device__ __forceinline__ int cut(int b, int x, int len) const {
        const int l = b - x, r = x + len - b;
        return l < snap && l <= r ? x : (r < snap ? x + len : b);
    }
    // the first and the last workgroup of the item [x, x + len)
    __device__ __forceinline__ int first_of(int x, int len) const {
        const int k = part_of(x, share), b = (k + 1) * share;
        return min(n - 1, b < x + len && cut(b, x, len) == x ? k + 1 : k);
    }
    __device__ __forceinline__ int final_of(int x, int len) const {
        const int k = part_of(x + len - 1, share), b = k * share;
        return min(n - 1, b > x && cut(b, x, len) == x + len ? k - 1 : k);
    }
};

// A piece of a sequence's keys: piece `part` of `parts`, tiles [t0, t1)
struct FewItem {
    Seq q;
    int part, parts, t0, t1;
    int first;                      // piece 0's number, or workgroup
};
// Piece `item` of a call of few rows alone.  All sequences are cut into pieces
// of at most `chunk` tiles, the least for which the pieces are no more than
// `slots` (the workgroups that run at once, per kv head), so a long sequence
// among short ones gets its share of the chip and no piece waits for a second
// round: tried from the even share up in steps of an eighth, for up to 64
// sequences; more of them leave many pieces, whose rounds even out.  Against
// equal shares of the axis, which cross the sequences' ends, the workgroups find
// their work sooner (8 x 1024 keys 8.4 us against 11.4, 64 x 4096 88 against 89).
// By whole waves.
__device__ __forceinline__ FewItem few_item(const PagedArgs& a, int item, int slots, int least) {
    const int lane = threadIdx.x & 63;
    Seq q = seq_of(a, min(lane, a.n_seq - 1));
    int t = lane < a.n_seq ? few_tiles(a, q) : 0;
    int total = t;
    for (int s = lane + 64; s < a.n_seq; s += 64) total += few_tiles(a, seq_of(a, s));
    total = wave_total(total);
    int chunk = max(least, (total + slots - 1) / slots);
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
            r.q.s = i + l;
            r.parts = lane_of(c, l);
            r.first = base + lane_of(end - c, l);
            r.part = item - r.first;
            const int tiles = (r.q.L + kFewTile - 1) / kFewTile;
            r.t0 = (int)((int64_t)r.part * tiles / r.parts);
            r.t1 = (int)((int64_t)(r.part + 1) * tiles / r.parts);
            return r;
        }
        base += lane_of(end, 63);
    }
    return r;
}
constexpr int kSc1 = 16;           // cache policy of the partials: agent scope
// a ticket per piece (or partial's place) and kv head, and one per sequence's
// first; pieces are at most n_seq and the workgroups at once, per kv head
constexpr int kFewTickets = kMaxPagedSeqHeads + 4 * kMaxWgs;
// pieces whose partials are loaded together (16: 8 x 1024 keys 9.4 -> 10.0 us, two
// streams of 1k keys 6.8 -> 7.3, 1 x 32768 keys 23.2 -> 22.2)
constexpr int kMergeBatch = 8;

// How few_piece goes over pages of type PT with up to ROWS rows: tiles that a wave
// has under way, and its LDS: the rows of Q and the waves' tiles (16-bit pages: a K
// and a V tile, Q8_0: codes and scales of each), then the waves' sums
template <int D, int PT, int WAVES, int ROWS>
struct FewLds {
    static constexpr bool Q8 = PT == VVA_TYPE_Q8_0;
    static constexpr int STAGES = Q8 && !(ROWS == 16 && D == 128) ? 2 : 1;
    static constexpr int TILE = Q8 ? kFewTile * (D + D / 16) : kFewTile * 2 * D;   // bytes of a K (V) tile
    static constexpr int OP = D + 4;               // pitch of a row of sums
    static constexpr int SUMS = WAVES * ROWS * (OP + 2) * (int)sizeof(float), RING = ROWS * 2 * D + WAVES * STAGES * 2 * TILE;
    static constexpr int BYTES = RING > SUMS ? RING : SUMS;
};

// What a wave's walk over the tiles of a piece leaves, for up to ROWS rows
template <int D, int ROWS> struct FewSums;
template <int D>
struct FewSums<D, 32> {
    f32x16 o[D / 32] = {};
    float m = -INFINITY, lsum = 0.0f;
    bool bad = false;               // a page outside the pool
    // dims of row `lane % 32` into its row of sums; the row sum over the lanes
    __device__ __forceinline__ void store(float* row, int lane) const {
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt)
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4)
                *(float4*)(row + dt * 32 + 8 * q4 + 4 * (lane >> 5)) =
                    make_float4(o[dt][4 * q4], o[dt][4 * q4 + 1], o[dt][4 * q4 + 2], o[dt][4 * q4 + 3]);
    }
    __device__ __forceinline__ float row_sum() const { return add_swap32(lsum); }
};
template <int D>
struct FewSums<D, 16> {
    f32x4 o[D / 16] = {};
    float m = -INFINITY, lsum = 0.0f;
    bool bad = false;
    __device__ __forceinline__ void store(float* row, int lane) const {
#pragma unroll
        for (int i = 0; i < D / 16; ++i) *(float4*)(row + i * 16 + 4 * (lane >> 4)) = make_float4(o[i][0], o[i][1], o[i][2], o[i][3]);
    }
    __device__ __forceinline__ float row_sum() const { return add_swap32(add_swap16(lsum)); }
};
// The rows of Q into LDS, a part by each wave, laid out as 16-bit K is; rows that
// are not there are row 0 again (no one reads their results)
template <int D, int WAVES, int ROWS>
__device__ __forceinline__ void few_load_q(const PagedArgs& a, const FewItem& it, int kvh, int rows, uint32_t qs) {
    constexpr int NC = ROWS * 2 * D / 1024, RC = 1024 / (2 * D);
    const int lane = threadIdx.x & 63, w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint64_t qb = uniform64((uint64_t)(uintptr_t)a.q + (int64_t)it.q.q0 * a.q_nb_t + (int64_t)kvh * a.G * a.q_nb_h);
#pragma unroll
    for (int i = 0; i < (NC + WAVES - 1) / WAVES; ++i) {
        const int c = w + i * WAVES;
        if (NC % WAVES && c >= NC) break;
        const int r = c * RC + lane / (D / 8), row = r < rows ? r : 0;
        const int rt = div_g(a, row), off = rt * (int)a.q_nb_t + (row - rt * a.G) * (int)a.q_nb_h;
        dma16<false>(qb, off + (((lane % (D / 8)) ^ k_swz<D>(r)) << 4), qs + c * 1024);
    }
}
// The softmax of a tile's scores: the running max and the sums raised to it, the
// probabilities packed (BF16: with what their rounding leaves), their sum
template <int D, int KT>
__device__ __forceinline__ void few_probs(const f32x16& s, float sl2, FewSums<D, 32>& f, uint32_t (&p)[8], uint32_t (&rest)[8]) {
    float mx = fmaxf(s[0], s[1]);
#pragma unroll
    for (int r = 2; r < 16; r += 2) mx = fmaxf(fmaxf(mx, s[r]), s[r + 1]);
    mx = max_swap32(mx) * sl2;
    if (__any(mx > f.m + kLazy)) {
        if (mx > f.m + kLazy) {
            const float alpha = __builtin_amdgcn_exp2f(f.m - mx);  // 0 while m = -inf
            f.lsum *= alpha;
#pragma unroll
            for (int dt = 0; dt < D / 32; ++dt) f.o[dt] *= alpha;
            f.m = mx;
        }
    }
    const float nb = kLift<KT> - (f.m == -INFINITY ? 0.0f : f.m);
#pragma unroll
    for (int r = 0; r < 8; ++r) {
        const float x = __builtin_amdgcn_exp2f(fmaf(s[2 * r], sl2, nb)), y = __builtin_amdgcn_exp2f(fmaf(s[2 * r + 1], sl2, nb));
        if constexpr (KT == VVA_TYPE_BF16) {
            split2_bf16(x, y, p[r], rest[r]);
            f.lsum = sum2<KT>(rest[r], f.lsum);
        } else {
            p[r] = pack2<KT>(x, y);
        }
        f.lsum = sum2<KT>(p[r], f.lsum);
    }
}

// Each wave streams every WAVES-th tile of a piece through LDS of its own, without
// a barrier: the next K goes out when K is read, the next V when V is, so 16 KB of
// the wave's loads fly while it waits and 8 while it computes.
template <int D, int KT, int WAVES>
__device__ __forceinline__ void few_stream(const PagedArgs& a, const FewItem& it, int kvh, char* lds, FewSums<D, 32>& f) {
    using F = Frag<KT>;
    using QF = typename F::type;
    constexpr int DS = D / 16, DT = D / 32;
    constexpr int NC = kFewTile * 2 * D / 1024;    // loads of a K (V) tile
    constexpr int RC = 1024 / (2 * D);             // rows of a load
    constexpr int TB = kFewTile * 2 * D;           // bytes of a K (V) tile, and of the rows of Q

    const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = min(it.q.n, a.max_new), L = it.q.L, rows = n * a.G, past = L - it.q.n;
    const int t0 = it.t0, t1 = it.t1;

    // ---- this wave's tiles: t0 + w, + 4, ...
    const ConstInts table = (ConstInts)(uintptr_t)(a.table + (int64_t)it.q.s * a.table_stride);
    const int last_page = (L - 1) >> a.page_shift;
    const uint32_t qs = (uint32_t)(uintptr_t)(lds_char*)lds, ks = qs + (1 + 2 * w) * TB, vs = ks + TB;
    int koff[4], voff[4];                          // by row group: the swizzles repeat every 16 rows
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        koff[i] = dma_off<D, false>(lane, i * RC, (int)a.k_nb_slot);
        voff[i] = dma_off<D, true>(lane, i * RC, (int)a.v_nb_slot);
    }
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
            f.bad = f.bad || !ok;
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
    few_load_q<D, WAVES, 32>(a, it, kvh, rows, qs);
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
    const int lim = l32 < rows ? min(L - 1, past + div_g(a, l32)) : -1;   // the last key the lane's row sees
    const float sl2 = a.scale * kLog2e;
    for (; t < t1; t += WAVES) {
        const bool more = t + WAVES < t1;
        if (more) fetch(t + WAVES);
        wait_vm<NC>();                             // K; V may still fly
        f32x16 s{};
#pragma unroll
        for (int ds = 0; ds < DS; ++ds) s = F::mma(as_vec<QF>(lds_read((ks + k_off) ^ (ds << 5))), qf[ds], s);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // K is read
            issue_k(t + WAVES);
        }
        const int k0 = t * kFewTile;
        const bool masked = k0 + kFewTile - 1 > min(L - 1, past);      // some row must not see some key
        if (masked) {
#pragma unroll
            for (int r = 0; r < 16; ++r) s[r] = 8 * (r / 4) + r % 4 > lim - k0 - 4 * half ? -INFINITY : s[r];
        }
        uint32_t p[8];
        [[maybe_unused]] uint32_t rest[8];
        few_probs<D, KT>(s, sl2, f, p, rest);
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
                f.o[dt] = F::mma(as_vec<QF>(vf), pf, f.o[dt]);
                if constexpr (KT == VVA_TYPE_BF16)
                    f.o[dt] = F::mma(as_vec<QF>(vf), as_vec<QF>(u32x4{rest[4 * kk], rest[4 * kk + 1], rest[4 * kk + 2], rest[4 * kk + 3]}), f.o[dt]);
            }
        }
        if (fix) add_not_finite<D, KT, kFewTile>(vs, k0, lim, half, f.o);
        if (more) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // V is read
            issue_v(t + WAVES);
        }
    }
}

#include "paged_q8.hpp"

// A workgroup's piece of a sequence's keys, for one kv head.  The waves' sums
// meet at the end.  Partials in the workspace, per piece and kv head: [cap
// rows][D] sums, then [cap] (exponent base, row sum).
template <int D, int PT, int OT, int WAVES, int ROWS, bool SHARES>
__device__ __forceinline__ void few_piece(const PagedArgs& a, float* __restrict__ ws, unsigned* tickets, int cap, const FewItem& it, int kvh, char* lds) {
    using Lds = FewLds<D, PT, WAVES, ROWS>;
    constexpr int OP = Lds::OP;
    const int tid = threadIdx.x, lane = tid & 63;
    const int w = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int rows = min(it.q.n, a.max_new) * a.G;
    FewSums<D, ROWS> f;
    if constexpr (ROWS == 16) few_stream16_q8<D, OT, WAVES, Lds::STAGES>(a, it, kvh, lds, f);
    else if constexpr (Lds::Q8) few_stream_q8<D, OT, WAVES>(a, it, kvh, lds, f);
    else few_stream<D, PT, WAVES>(a, it, kvh, lds, f);
    // ---- the waves' sums, in LDS, added in wave order
    const float lt = f.row_sum();
    __syncthreads();
    float* const ow = (float*)lds;
    float* const ml = ow + WAVES * ROWS * OP;
    if (lane % ROWS < rows) {
        f.store(ow + (w * ROWS + lane % ROWS) * OP, lane);
        if (lane < ROWS) *(float2*)(ml + (w * ROWS + lane) * 2) = make_float2(f.m, lt);
    }
    const bool bad_page = __syncthreads_or(f.bad);
    const PagedArgs& args = fresh_args();
    // thread i's part of the sums: 4 dims of a row
    struct Sum {
        float4 num;
        float M, den;
    };
    // nan: the row is to answer NaN
    auto write = [&](int row, int c, const Sum& x, bool nan) {
        const int rt = div_g(args, row);
        // zeros where the row sees no key; all scores -inf: 0 * (1 / 0), the softmax's NaN
        const float inv = min(it.q.L - 1, it.q.L - it.q.n + rt) >= 0 ? 1.0f / x.den : 0.0f;
        uint2 y = {pack2<OT>(x.num.x * inv, x.num.y * inv), pack2<OT>(x.num.z * inv, x.num.w * inv)};
        if (nan) y.x = y.y = 0x7fff7fffu;
        *(uint2*)(args.out + (int64_t)(it.q.q0 + rt) * args.o_nb_t + (int64_t)(kvh * args.G + row - rt * args.G) * args.o_nb_h + 8 * c) = y;
    };
    // A piece's place for its partial, by its number; in shares, where a
    // workgroup may end one sequence and begin another, the workgroup's first, for
    // a sequence's first piece its second
    auto place = [&](int part) { return (SHARES ? 2 * (it.first + part) + (part == 0) : it.first + part) * args.Hkv + kvh; };
    auto piece_rsrc = [&](int part) {
        const uint32_t bytes = cap * (D + 2) * sizeof(float);
        return make_rsrc((const char*)ws + (int64_t)place(part) * bytes, bytes);
    };
    // agent-scope stores: coherent across the XCDs' L2 caches
    auto store = [&](int part, int row, int c, const Sum& x, bool nan) {
        const BufRsrc rs = piece_rsrc(part);
        __builtin_amdgcn_raw_buffer_store_b128(u32x4{__float_as_uint(x.num.x), __float_as_uint(x.num.y), __float_as_uint(x.num.z), __float_as_uint(x.num.w)},
                                               rs, (row * D + 4 * c) * 4, 0, kSc1);
        if (c == 0)
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{nan ? kNanBits : __float_as_uint(x.M), __float_as_uint(x.den)}, rs,
                                                  (cap * D + row * 2) * 4, 0, kSc1);
    };
    for (int i = tid; i < rows * (D / 4); i += WAVES * 64) {
        const int row = i / (D / 4), c = i % (D / 4);
        Sum x{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
#pragma unroll
        for (int k = 0; k < WAVES; ++k) x.M = fmaxf(x.M, ml[(k * ROWS + row) * 2]);
        const float base = x.M == -INFINITY ? 0.0f : x.M;
#pragma unroll
        for (int k = 0; k < WAVES; ++k) {
            const float e = __builtin_amdgcn_exp2f(ml[(k * ROWS + row) * 2] - base);   // 0 for a wave without keys
            const float4 v = *(const float4*)(ow + (k * ROWS + row) * OP + 4 * c);
            x.den = fmaf(e, ml[(k * ROWS + row) * 2 + 1], x.den);
            x.num.x = fmaf(e, v.x, x.num.x); x.num.y = fmaf(e, v.y, x.num.y);
            x.num.z = fmaf(e, v.z, x.num.z); x.num.w = fmaf(e, v.w, x.num.w);
        }
        if (it.parts > 1) store(it.part, row, c, x, bad_page);
        else write(row, c, x, bad_page);
    }
    if (it.parts == 1) return;
    // ---- the last of a group of pieces adds their partials, in order, and the
    // last of more groups adds the groups (one group of up to 16 pieces, more
    // of 8: two batches of loads in a row cost less than a second ticket).
    // The group's sums take the place of its first piece's, which a thread
    // overwrites where it alone has read them (a row's exponent: its wave).
    const int size = it.parts <= 2 * kMergeBatch ? 2 * kMergeBatch : kMergeBatch, grp = it.part / size;
    const int groups = (it.parts + size - 1) / size;
    unsigned* tk = tickets + kFewTickets + place(grp * size);
    int first = grp * size, by = 1, n_add = min(size, it.parts - first);
#pragma unroll 1
    for (int level = 0; level < 2; ++level) {
        const bool final = level > 0 || groups == 1;
        if (n_add > 1) {
            __builtin_amdgcn_s_waitcnt(0);             // every store of this workgroup is done before its ticket
            __syncthreads();
            int* const last = (int*)lds;
            if (tid == 0) {
                const unsigned old = __hip_atomic_fetch_add(tk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                *last = old == (unsigned)(n_add - 1);
                if (*last) __hip_atomic_store(tk, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            __syncthreads();
            if (!*last) return;
#pragma unroll 1
            for (int i = tid; i < rows * (D / 4); i += WAVES * 64) {
                const int row = i / (D / 4), c = i % (D / 4);
                Sum x{make_float4(0.0f, 0.0f, 0.0f, 0.0f), -INFINITY, 0.0f};
                bool nan = false;
#pragma unroll 1
                for (int p0 = 0; p0 < n_add; p0 += kMergeBatch) {
                    // a batch's loads go out together, one round trip each; those
                    // past the last piece lie outside their buffer and read nothing
                    u32x2 e[kMergeBatch];
                    u32x4 v[kMergeBatch];
#pragma unroll
                    for (int u = 0; u < kMergeBatch; ++u) {
                        const bool in = p0 + u < n_add;
                        const BufRsrc rs = piece_rsrc(first + (in ? p0 + u : 0) * by);
                        e[u] = __builtin_amdgcn_raw_buffer_load_b64(rs, in ? (cap * D + row * 2) * 4 : 0x7ffffff0, 0, kSc1);
                        v[u] = __builtin_amdgcn_raw_buffer_load_b128(rs, in ? (row * D + 4 * c) * 4 : 0x7ffffff0, 0, kSc1);
                    }
#pragma unroll
                    for (int u = 0; u < kMergeBatch; ++u) asm volatile("" : "+v"(e[u]), "+v"(v[u]));
                    float mb = x.M;
#pragma unroll
                    for (int u = 0; u < kMergeBatch; ++u) {
                        const bool hit = e[u].x == kNanBits;
                        nan = nan || hit;
                        if (hit || p0 + u >= n_add) {          // nothing to add
                            e[u] = u32x2{0xff800000u, 0u};
                            v[u] = u32x4{0u, 0u, 0u, 0u};
                        }
                        mb = fmaxf(mb, __uint_as_float(e[u].x));
                    }
                    const float base = mb == -INFINITY ? 0.0f : mb;
                    const float f0 = __builtin_amdgcn_exp2f(x.M - base);
                    x.M = mb;
                    x.den *= f0;
                    x.num.x *= f0; x.num.y *= f0; x.num.z *= f0; x.num.w *= f0;
#pragma unroll
                    for (int u = 0; u < kMergeBatch; ++u) {
                        const float f = __builtin_amdgcn_exp2f(__uint_as_float(e[u].x) - base);
                        x.den = fmaf(f, __uint_as_float(e[u].y), x.den);
                        x.num.x = fmaf(f, __uint_as_float(v[u].x), x.num.x);
                        x.num.y = fmaf(f, __uint_as_float(v[u].y), x.num.y);
                        x.num.z = fmaf(f, __uint_as_float(v[u].z), x.num.z);
                        x.num.w = fmaf(f, __uint_as_float(v[u].w), x.num.w);
                    }
                }
                if (final) write(row, c, x, nan);
                else store(first, row, c, x, nan);
            }
        }
        if (final) return;
        tk = tickets + place(0);
        first = 0;
        by = size;
        n_add = groups;
    }
}

// One workgroup per (piece, kv head), two of them on a CU (D = 64, 4 waves: four over
// 16-bit pages, three over Q8_0 ones).
template <int D, int PT, int OT, int WAVES, int ROWS>
__global__ void __launch_bounds__(WAVES * 64, WAVES == 8 ? 4 : 2) paged_few_kernel(PagedArgs a, float* __restrict__ ws, unsigned* tickets, int slots, int cap) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    __shared__ __attribute__((aligned(1024))) char lds[FewLds<D, PT, WAVES, ROWS>::BYTES];
    const FewItem it = few_item(a, blockIdx.x / a.Hkv, slots, WAVES);
    if (it.parts > 0) few_piece<D, PT, OT, WAVES, ROWS, false>(a, ws, tickets, cap, it, blockIdx.x % a.Hkv, lds);
}

// ----------------------------------------------------------- many rows

constexpr int kBN = 64;            // keys per tile
constexpr int kRowsWave = 32;
constexpr int kWaves = 8;          // two per SIMD
constexpr int kRowsWG = kRowsWave * kWaves;
constexpr int kStages = 4;         // LDS ring: tile j + 3 loads while tile j is computed
constexpr int kRowTileCost = 4;    // what a row tile costs beside its keys, in key tiles
constexpr int kSnap = 3;           // cuts this near an end of a row tile, in key tiles, are moved there
constexpr int kGroup = 8;          // pieces whose partials are added at once
constexpr int kManyTickets = kMaxWgs * kWaves * (1 + kMaxWgs / kGroup);

// Row tiles of a sequence (few_rows: what paged_few_kernel takes, 0 where it is
// not launched), and the key tiles that one sees
__device__ __forceinline__ int many_row_tiles(const PagedArgs& a, const Seq& q) {
    const int n = min(q.n, a.max_new);
    return n * a.G > a.few_rows ? (n * a.G + kRowsWG - 1) / kRowsWG : 0;
}
__device__ __forceinline__ int many_key_tiles(const PagedArgs& a, const Seq& q, int rt) {
    const int n = min(q.n, a.max_new);
    const int t_hi = min(n * a.G, (rt + 1) * kRowsWG) - 1;
    return (max(0, min(q.L, q.L - q.n + div_g(a, t_hi) + 1)) + kBN - 1) / kBN;
}

// The call's work on one axis: kv heads, in them the sequences, in them the
// row tiles, each as long as the keys that it sees: first + slope * (rt + 1)
// sixteenths of a key tile (more, where 2^30 of them would not hold the call).
// The axis is cut into equal shares, one per workgroup, wherever that falls in
// a row tile: a chunk over a long cache, prompts of unlike lengths and a few
// row tiles all leave every CU the same work.
struct ManyWeight {
    int r, first, slope;
    __device__ __forceinline__ int before(int rt) const { return rt * first + (int)((int64_t)slope * rt * (rt + 1) / 2); }
    __device__ __forceinline__ int of(int rt) const { return first + slope * (rt + 1); }
};
__device__ __forceinline__ ManyWeight many_weight(const PagedArgs& a, const Seq& q, int slope, int shift) {
    ManyWeight w;
    w.r = many_row_tiles(a, q);
    w.first = max((max(q.L - q.n, 0) / (kBN / 16) + 16 * kRowTileCost) >> shift, 1);
    w.slope = slope >> shift;
    return w;
}
struct ManyAxis {
    int slope;              // of a row tile, in sixteenths
    int shift;              // the unit's power of two above a sixteenth
    int head;               // length of a kv head's part (0: no work)
    int row_tiles;          // in it
};
// `mine`: the lane's own of the first 64 sequences.  By whole waves.
__device__ __forceinline__ ManyAxis many_axis(const PagedArgs& a, const Seq& mine) {
    const int lane = threadIdx.x & 63;
    ManyAxis x;
    x.slope = div_g(a, kRowsWG * 16 / kBN);
    float all = 0.0f;
    for (int s = lane; s < a.n_seq; s += 64) {
        const ManyWeight w = many_weight(a, s == lane ? mine : seq_of(a, s), x.slope, 0);
        all += (float)w.r * ((float)w.first + 0.5f * (float)w.slope * (float)(w.r + 1));
    }
    all = wave_sum(all) * (float)a.Hkv;
    int shift = 0;
    for (; all > 1.0e9f; all *= 0.5f) ++shift;
    x.shift = uni(shift);
    int total = 0, r = 0;
    for (int s = lane; s < a.n_seq; s += 64) {
        const ManyWeight w = many_weight(a, s == lane ? mine : seq_of(a, s), x.slope, x.shift);
        total += w.before(w.r);
        r += w.r;
    }
    x.head = wave_total(total);
    x.row_tiles = wave_total(r);
    return x;
}
// The sequence at place p of a kv head's part, and where it starts and ends
struct ManySeq {
    Seq q;
    int start, end;
};
__device__ __forceinline__ ManySeq many_seq(const PagedArgs& a, const ManyAxis& x, const Seq& mine, int p) {
    const int lane = threadIdx.x & 63;
    ManySeq r{};
    Seq q = mine;
    int base = 0;
    for (int i = 0; i < a.n_seq; i += 64) {
        if (i > 0) q = seq_of(a, min(i + lane, a.n_seq - 1));
        const ManyWeight w = many_weight(a, q, x.slope, x.shift);
        const int len = i + lane < a.n_seq ? w.before(w.r) : 0;
        const int end = base + wave_scan(len);
        const uint64_t hit = __ballot(p >= end - len && p < end);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            r.q.q0 = lane_of(q.q0, l);
            r.q.n = lane_of(q.n, l);
            r.q.L = lane_of(q.L, l);
            r.q.s = i + l;
            r.end = lane_of(end, l);
            r.start = r.end - lane_of(len, l);
            return r;
        }
        base = lane_of(end, 63);
    }
    return r;
}

// The shares of the work, n at most.  A row tile of t key tiles cut into n
// parts takes about t / n of them, and a part of one more per piece to add:
// shares are not below 0.6 times the square root of the average t and what a
// row tile costs (256 tokens behind 4096 keys, 28 row tiles: 51.6 us with
// shares of 4 tiles, 47.8 with 8).
__device__ __forceinline__ int many_shares(const PagedArgs& a, const ManyAxis& axis, int n) {
    const float tile = 16.0f * __builtin_amdgcn_rcpf((float)(1 << axis.shift));
    const float mean = fmaxf((float)axis.head * __builtin_amdgcn_rcpf((float)axis.row_tiles * tile) - (float)kRowTileCost, 1.0f);
    const float least = ((float)kRowTileCost + 0.6f * __builtin_amdgcn_sqrtf(mean)) * tile;
    return uni(max(1, min(n, (int)((float)(axis.head * a.Hkv) * __builtin_amdgcn_rcpf(least)))));
}

// The share of a workgroup: neighbouring shares on one XCD (workgroups go round
// its 8), since they read the same keys (252 shares of 256 tokens behind 4096
// keys 44 us by turns, 38 so).
__device__ __forceinline__ int on_xcds(int block, int wgs) {
    const int x = block % 8;
    return x * (wgs / 8) + min(x, wgs % 8) + block / 8;
}

// The other way to cut, for calls of few row tiles: each into equal parts of at
// most S key tiles, a part per workgroup.
struct ManyPieces {
    int head;               // parts of a kv head, 0: equal shares
    Seq q;                  // the workgroup's row tile
    int rt, kvh, first, parts;  // its parts are `first` .. of all; how many
};
// Where the row tiles are no more than the workgroups (n), S is the least for
// which the parts are not either: tried up in steps of an eighth from the even
// length or, where that is longer, what a cut is worth (kPieceLeast, and
// kPieceRoot times the root of the longest row tile, as each part is one more to
// add).  A share that crosses a row tile's end costs its workgroup a second
// opening and more sums, about kPieceGain key tiles of time; against it stand
// the workgroups that parts of one length leave idle, so that parts longer by
// more than that are left to the shares.  Shares against parts, us: 1.5B heads,
// a prompt of 700 tokens 29.6 and 22.4; 7B, 4 prompts of up to 1000 38.3 and 33.9, 64
// tokens behind 4096 keys 42 and 34, 128 behind 8192 51 and 40; 0.5B, 4096 tokens
// (28 key tiles a share) 51.1 and 52.6.  By whole waves.
constexpr int kPieceGain = 9;
constexpr int kPieceMost = 16;     // shares longer than this, in key tiles, are not worth the look
constexpr float kPieceLeast = 4.0f, kPieceRoot = 1.1f;
__device__ __forceinline__ ManyPieces many_pieces(const PagedArgs& a, const ManyAxis& axis, const Seq& mine, int n, int block) {
    constexpr int CH = 4;   // row tiles of a lane
    const int lane = threadIdx.x & 63;
    const int slots = part_of(n, a.Hkv);
    ManyPieces m{};
    // (key tiles of a share)
    const float mean = (float)axis.head * (float)(1 << axis.shift) * (1.0f / 16) - (float)kRowTileCost * (float)axis.row_tiles;
    if (a.n_seq > 64 || axis.row_tiles > min(slots, 64 * CH) || mean > (float)kPieceMost * (float)slots) return m;
    const int r = lane < a.n_seq ? many_row_tiles(a, mine) : 0;
    const int end = wave_scan(r);
    int tiles[CH] = {}, total = 0;
    for (uint64_t left = __ballot(r > 0); left; left &= left - 1) {
        const int l = __ffsll((unsigned long long)left) - 1;
        const Seq q{lane_of(mine.q0, l), lane_of(mine.n, l), lane_of(mine.L, l), l};
        const int e = lane_of(end, l), b = e - lane_of(r, l);
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            if (64 * k >= e || 64 * (k + 1) <= b) continue;
            const int i = 64 * k + lane;
            if (i >= b && i < e) tiles[k] = max(1, many_key_tiles(a, q, i - b));
        }
    }
    float most = 0.0f;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        total += tiles[k];
        most = fmaxf(most, (float)tiles[k]);
    }
    total = wave_total(total);
    most = fmaxf(most, dpp<kDppXor1>(most));
    most = fmaxf(most, dpp<kDppXor2>(most));
    most = fmaxf(most, dpp<kDppHalfMirror>(most));
    most = fmaxf(most, dpp<kDppMirror>(most));
    most = uni(max_swap32(max_swap16(most)));
    const int even = part_of(total + slots - 1, slots);
    const int floor = uni((int)fmaxf(kPieceLeast, kPieceRoot * __builtin_amdgcn_sqrtf(most)));
    int S = max(even, floor);
    int parts[CH];
    auto count = [&] {
        const float inv = __builtin_amdgcn_rcpf((float)S);
        int c = 0;
#pragma unroll
        for (int k = 0; k < CH; ++k) {
            parts[k] = 0;
            if (k > 0 && axis.row_tiles <= 64 * k) continue;
            parts[k] = tiles[k] > 0 ? max(1, (int)__builtin_ceilf((float)tiles[k] * inv - 0.01f)) : 0;
            c += parts[k];
        }
        return wave_total(c);
    };
    int c = count();
    for (const int limit = S + kPieceGain; c > slots;) {
        S += (S + 7) / 8;
        if (S > limit) return m;
        c = count();
    }
    m.head = c;
    const int wgs = c * a.Hkv;
    if (block >= wgs) return m;
    const int g = on_xcds(block, wgs);
    m.kvh = part_of(g, c);
    const int p = g - m.kvh * c;
    int base = 0, i = 0;
#pragma unroll
    for (int k = 0; k < CH; ++k) {
        const int to = base + wave_scan(parts[k]);
        const uint64_t hit = __ballot(p >= to - parts[k] && p < to);
        if (hit) {
            const int l = __ffsll((unsigned long long)hit) - 1;
            m.parts = lane_of(parts[k], l);
            m.first = m.kvh * c + lane_of(to, l) - m.parts;
            i = 64 * k + l;
        }
        base = lane_of(to, 63);
    }
    const int l = __ffsll((unsigned long long)__ballot(r > 0 && i < end && i >= end - r)) - 1;
    m.q = Seq{lane_of(mine.q0, l), lane_of(mine.n, l), lane_of(mine.L, l), l};
    m.rt = i - lane_of(end - r, l);
    return m;
}

// Share `block` of `wgs`, or a part (parts.head > 0), by one workgroup: 8 waves x 32 rows that share every
// K / V tile.  A row tile that lies in one share is written at once; of one that
// several workgroups share, each leaves its rows' sums in the workspace, wave
// by wave ([wave][16-byte group][lane], then (exponent base, row sum)), and
// takes the wave's ticket: the last of up to kGroup pieces adds them, and of
// more groups the last adds the groups, in the order of the keys whoever it is
// (its own sums are read back too, so that they need no registers meanwhile).
template <int D, int PT>
struct ManyLds {
    // Q8_0: tile j + 2 is stored while tile j is computed.  The last two stages of
    // the 16-bit ring, one of three here, take the rows of Q first.
    static constexpr int STAGES = PT == VVA_TYPE_Q8_0 ? 3 : kStages;
    static constexpr int Q_AT = PT == VVA_TYPE_Q8_0 ? 1 : 2;
    static constexpr int BYTES = STAGES * 2 * kBN * 2 * D;
};
template <int D, int PT, int OT>
__device__ __forceinline__ void many_share(const PagedArgs& a, float* __restrict__ ws, unsigned* tickets, const ManyAxis& axis, const ManyPieces& pc, const Seq& mine, int block, int wgs, char* lds, int* marks) {
    constexpr int KT = kComp<PT>;
    constexpr bool Q8 = PT == VVA_TYPE_Q8_0;
    using F = Frag<KT>;
    using QF = typename F::type;
    constexpr int DS = D / 16, DT = D / 32;
    constexpr int ROW = 2 * D;
    constexpr int TB = kBN * ROW;                  // bytes of a K (V) tile
    constexpr int NI = TB / 1024 / kWaves;         // loads of a K (V) tile per wave
    constexpr int RC = 1024 / ROW;                 // rows of a load
    constexpr int STAGE = 2 * TB, STAGES = ManyLds<D, PT>::STAGES, Q_AT = ManyLds<D, PT>::Q_AT;
    constexpr int NLD = 2 * NI;
    constexpr int NID = Q8 ? 1 : NI;               // page ids of a wave's loads of a tile
    constexpr int WAVE_O = DT * 16 * 64 * 4;       // bytes of a wave's sums
    constexpr int WAVE = WAVE_O + 64 * 8;
    int& fix = marks[0];                           // the last tile with a V that is not finite
    int& bad_seg = marks[1];                       // the last share with a bad page

    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    if (threadIdx.x == 0) fix = bad_seg = -1;      // before the first tile's barrier
    ManySeq sq{};                                  // the sequence at hand, and its end on the axis
    int sq_kvh = 0, sq_end = -1;
    // parts lie on an axis of their own, a unit each, in shares of one
    const bool whole_parts = pc.head > 0;
    const int head = whole_parts ? pc.head : axis.head, axis_shift = axis.shift, axis_slope = axis.slope, total = head * a.Hkv;
    const int g = on_xcds(block, wgs);
    const int share = whole_parts ? 1 : uni((int)((float)total * 1.000001f * __builtin_amdgcn_rcpf((float)wgs)) + 1);      // share * wgs >= total
    if (whole_parts) {
        sq.q = pc.q;
        sq_kvh = pc.kvh;
        sq_end = total;
    } else {
        const int p = min(g * share, total - 1);
        sq_kvh = part_of(p, head);
        sq = many_seq(a, axis, mine, p - sq_kvh * head);
        sq_end = sq_kvh * head + sq.end;
    }
    const Shares cuts{share, wgs, whole_parts ? 0 : max(1, min(share / 2, (16 * kSnap) >> axis_shift))};
    const int p_end = min(total, (g + 1) * share);
    const float inv_g = uni(1.0f / (float)a.G);

    // ---- the row tile at place p of the axis, and this workgroup's keys of it
    struct Cut {
        int s, kvh, q0, rows, L, past;             // the sequence; rows of its kv group
        int rt, n_tiles, kb0;                      // row tile, key tiles from key kb0 on
        int place, len;                            // the row tile on the axis
        bool whole, empty;
        int next;                                  // the place after this part
    };
    auto find = [&](int p, bool begin) {           // begin: p is the share's own, yet to be moved
        const PagedArgs& a = fresh_args();
        const int G = a.G;
        Cut c;
        if (p >= sq_end) {
            sq_kvh = part_of(p, head);
            sq = many_seq(a, ManyAxis{axis_slope, axis_shift, head}, seq_of(a, min((int)threadIdx.x & 63, a.n_seq - 1)), p - sq_kvh * head);
            sq_end = sq.end > sq.start ? sq_kvh * head + sq.end : p_end;   // no sequence: a batch that changed meanwhile
        }
        int rt = pc.rt;
        c.len = pc.parts;
        c.place = pc.first;
        if (!whole_parts) {
        ManyWeight wt = many_weight(a, sq.q, axis_slope, axis_shift);
        wt.r = uni(wt.r);
        const int ps = p - sq_kvh * head - sq.start;           // place in the sequence
        const float s2 = 0.5f * (float)wt.slope, f1 = (float)wt.first + s2;
        rt = (int)(wt.slope > 0 ? (__builtin_amdgcn_sqrtf(f1 * f1 + 4.0f * s2 * (float)ps) - f1) * __builtin_amdgcn_rcpf(2.0f * s2)
                                    : (float)ps * __builtin_amdgcn_rcpf((float)wt.first));
        rt = uni(max(0, min(rt, wt.r - 1)));
        while (rt > 0 && wt.before(rt) > ps) --rt;
        while (rt + 1 < wt.r && wt.before(rt + 1) <= ps) ++rt;
        c.len = wt.of(rt);
        c.place = p - (ps - wt.before(rt));
        }
        c.rt = rt;
        c.s = sq.q.s;
        c.kvh = sq_kvh;
        c.q0 = sq.q.q0;
        c.rows = min(sq.q.n, a.max_new) * G;
        c.L = sq.q.L;
        c.past = sq.q.L - sq.q.n;
        const int off = (begin ? cuts.cut(p, c.place, c.len) : p) - c.place;
        const int off_end = (p_end < c.place + c.len ? cuts.cut(p_end, c.place, c.len) : c.place + c.len) - c.place;
        c.whole = off <= 0 && off_end == c.len;
        c.empty = off_end <= off;                  // the share begins with the next row tile, or ended with the last
        c.next = c.place + max(c.empty ? off : off_end, 1);
        // keys in proportion: a function of the place alone, so that a part ends where the next begins
        const int tiles = uni(many_key_tiles(a, sq.q, rt));
        const float r = (float)tiles * __builtin_amdgcn_rcpf((float)c.len);
        const int lo = uni(min(tiles, (int)((float)max(off, 0) * r)));
        c.n_tiles = (off_end == c.len ? tiles : uni(min(tiles, (int)((float)off_end * r)))) - lo;
        c.kb0 = lo * kBN;
        return c;
    };

    // ---- tile loads: load i of K (V) covers rows RC * (i * 8 + w) .. of the
    // tile, inside one 16-key group
    const int r0w = RC * w;                        // first row of the wave's loads, + i * 8 * RC
    const int koff = dma_off<D, false>(lane_id(), r0w, (int)a.k_nb_slot);
    const int voff = dma_off<D, true>(lane_id(), r0w, (int)a.v_nb_slot);
    const int k_off = k_lane_off<D>(lane_id()), v_off = v_lane_off<D>(lane_id());
    const uint32_t lds0 = (uint32_t)(uintptr_t)(lds_char*)lds;
    const float sl2 = uni(a.scale * kLog2e);
    bool bad = false;
    int ids[NID];
    // where a part's K and V come from
    struct Source {
        uint64_t k, v;                             // the pools' kv head
        int64_t k_page, v_page;
        int k_slot, v_slot, n_pages, shift, last;  // last: the sequence's last page
        ConstInts table;
    };
    auto source = [&](const Cut& c) {
        const PagedArgs& a = fresh_args();
        return Source{uniform64((uint64_t)(uintptr_t)a.k + c.kvh * a.k_nb_head), uniform64((uint64_t)(uintptr_t)a.v + c.kvh * a.v_nb_head),
                      a.k_nb_page, a.v_nb_page, (int)a.k_nb_slot, (int)a.v_nb_slot, a.n_pages, a.page_shift,
                      max(0, (c.L - 1) >> a.page_shift), (ConstInts)(uintptr_t)(a.table + (int64_t)c.s * a.table_stride)};
    };
    auto fetch = [&](const Source& t, int key, int (&id)[NID]) {
#pragma unroll
        for (int i = 0; i < NID; ++i) id[i] = t.table[min((key + (Q8 ? 8 * w : i * kWaves * RC + r0w)) >> t.shift, t.last)];
    };
    // the loads of tile j, from key `key` on (K, then V); past the last tile
    // further ones of the sequence, to a stage that nobody reads any more, so
    // that every tile counts the same
    auto issue = [&](const Source& t, int j, int key, const int (&id)[NID]) {
        const uint32_t st = lds0 + (j % STAGES) * STAGE + w * 1024;
        uint64_t kb[NI], vb[NI];
#pragma unroll
        for (int i = 0; i < NI; ++i) {
            const bool ok = (uint32_t)id[i] < (uint32_t)t.n_pages;
            bad = bad || !ok;
            const int64_t page = ok ? id[i] : 0;
            const int slot = (key + i * kWaves * RC + r0w) & ((1 << t.shift) - 1);
            kb[i] = uniform64(t.k + page * t.k_page + slot * t.k_slot);
            vb[i] = uniform64(t.v + page * t.v_page + slot * t.v_slot);
        }
#pragma unroll
        for (int i = 0; i < NI; ++i) dma16<false>(kb[i], koff, st + i * kWaves * 1024);
#pragma unroll
        for (int i = 0; i < NI; ++i) dma16<false>(vb[i], voff, st + TB + i * kWaves * 1024);
    };
    // Q8_0: a wave takes 8 rows of a tile (D = 64: K by the lower lanes, V by the
    // upper), a lane 16 dims of one of K and one of V: loaded a step before they are
    // converted to F16 and stored, at the start of a step.  On one GPU, 2048 tokens
    // behind 28672 keys: 915 us so (F16 pages, whose rows go into LDS by themselves,
    // 870); by half of the waves at the end of the step 934, between the products 960, rows of
    // 8 dims a lane, whose stores meet on no banks but take two loads each, 928.
    constexpr int QC = D / 16, QN = D == 128 ? 2 : 1;
    u32x4 codes[QN];
    uint16_t scales[QN];
    auto load_q8 = [&](const Source& t, int key, const int (&id)[NID]) {
        const uint32_t ln = lane_id(), shift = t.shift;
        const bool ok = (uint32_t)id[0] < (uint32_t)t.n_pages;
        bad = bad || !ok;
        const int64_t at = ok ? id[0] : 0;
        const uint32_t slot = (uint32_t)(key + 8 * w) & ((1u << shift) - 1);
        // 8 rows of codes are one run of memory, 16 bytes a lane
        const uint32_t co = slot * D, so = ((uint32_t)D << shift) + 2 * slot;
        const uint32_t cl = ln % (8 * QC) * 16, sl = ((ln % QC / 2 << shift) + ln / QC % 8) * 2;
        const uint64_t kp = uniform64(t.k + at * t.k_page), vp = uniform64(t.v + at * t.v_page);
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const uint64_t p = QN == 2 ? (i == 0 ? kp : vp) : (ln < 32 ? kp : vp);
            codes[i] = global_load<u32x4>(p + co, cl);
            scales[i] = global_load<uint16_t>(p + so, sl);
        }
    };
    auto put_q8 = [&](int j) {
        const uint32_t ln = lane_id(), r = 8 * w + ln / QC % 8, c = 2 * (ln % QC);
        const uint32_t row = lds0 + (j % STAGES) * STAGE + r * ROW;
#pragma unroll
        for (int i = 0; i < QN; ++i) {
            const bool v = QN == 2 ? i == 1 : ln >= 32;
            const uint32_t to = row + (v ? TB : 0) + ((c ^ (uint32_t)(v ? v_swz<D>(r) : k_swz<D>(r))) << 4);
            const h2 x = q8_scale(scales[i]);
            const h2 x4[4] = {x, x, x, x};
            *lds_vec(to) = q8_frag<false>(codes[i].x, codes[i].y, x4).hi;
            *lds_vec(to ^ 16) = q8_frag<false>(codes[i].z, codes[i].w, x4).hi;
        }
    };
    // x = t * G + h for small x (below G + 32): one product
    auto small_divide = [&](int x, int G, int& t, int& h) {
        t = (int)(((float)x + 0.5f) * inv_g);
        h = x - t * G;
    };
    // a part's first loads: the wave's rows of Q (laid out as K is, in the
    // stages of tiles 2 and 3; rows past the last: one that is there), two tiles
    auto start = [&](const Cut& c, const Source& src) {
        const PagedArgs& a = fresh_args();
        const int G = a.G;
        bad = false;
        const int ln = lane_id();                  // offsets made here, not held from one part to the next
        int id0[NID];
        [[maybe_unused]] int id1[NID];
        fetch(src, c.kb0, id0);
        if constexpr (!Q8) fetch(src, c.kb0 + kBN, id1);
        fetch(src, c.kb0 + (Q8 ? 1 : 2) * kBN, ids);
        const int wr0 = min(c.rt * kRowsWG + w * kRowsWave, c.rows - 1), live = min(kRowsWave, c.rows - wr0);
        const int t0 = div_g(a, wr0), h0 = wr0 - t0 * G;
        const uint64_t qb = uniform64((uint64_t)(uintptr_t)a.q + (int64_t)(c.q0 + t0) * a.q_nb_t + (int64_t)c.kvh * G * a.q_nb_h);
#pragma unroll
        for (int i = 0; i < kRowsWave / RC; ++i) {
            const int r = i * RC + ln / (D / 8);
            int t, h;
            small_divide(h0 + (r < live ? r : 0), G, t, h);
            dma16<false>(qb, t * (int)a.q_nb_t + h * (int)a.q_nb_h + (((ln % (D / 8)) ^ k_swz<D>(r)) << 4),
                         lds0 + Q_AT * STAGE + w * kRowsWave * ROW + i * 1024);
        }
        if constexpr (Q8) {
            load_q8(src, c.kb0, id0);
        } else {
            issue(src, 0, c.kb0, id0);
            issue(src, 1, c.kb0 + kBN, id1);
        }
    };

    int fix_id = 0;
    for (int p = g * share, seg = 0, p_next; p < p_end; p = p_next, ++seg) {
    const Cut c = find(p, seg == 0);
    p_next = c.next;
    if (c.empty) {
        if (p_next >= p_end || seg > 0) break;     // moved past its end, or its end to here
        if (p_next <= p) break;
        continue;
    }
    const Source src = source(c);
    if (c.n_tiles > 0) start(c, src);
    const int L = c.L, past = c.past, kb0 = c.kb0, n_tiles = c.n_tiles, rows = c.rows;
    const int wr0 = c.rt * kRowsWG + w * kRowsWave;
    const bool wave_live = wr0 < rows;
    float m = -INFINITY, lsum = 0.0f;
    f32x16 o[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
    if (n_tiles > 0) {                                        // uniform
        const PagedArgs& a = fresh_args();
        const int G = a.G;
        // keys [0, kend_w) are seen by some row of the wave, keys up to lim_w by every row
        const int kend_w = uni(wave_live ? max(0, min(L, past + div_g(a, min(wr0 + kRowsWave, rows) - 1) + 1)) : 0);
        const int lim_w = uni(min(L - 1, past + div_g(a, min(wr0, rows - 1))));
        int lim, hcol;                                        // the last key the lane's row sees
        const int wr = min(wr0, rows - 1), t0 = div_g(a, wr);
        const int l32 = lane_id() & 31;
        small_divide(wr - t0 * G + (wr0 + l32 < rows ? l32 : 0), G, lim, hcol);
        lim = min(L - 1, past + t0 + lim);
        if constexpr (Q8) put_q8(0);
        wait_vm<Q8 ? 0 : 2 * NLD>();                          // Q has landed
        if constexpr (Q8) {
            load_q8(src, kb0 + kBN, ids);
            fetch(src, kb0 + 2 * kBN, ids);
        }
        QF qf[DS];
        {
            const uint32_t qa = lds0 + Q_AT * STAGE + w * kRowsWave * ROW + k_lane_off<D>(lane_id());
#pragma unroll
            for (int ds = 0; ds < DS; ++ds) qf[ds] = q_frag<KT, OT>(lds_read(qa ^ (ds << 5)));
        }
        // K of tile 0 has landed (its V and tile 1 may still fly), and every wave has its Q
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(Q8 ? 63 : NI + NLD) : "memory");
        if constexpr (Q8) {
            put_q8(1);
            load_q8(src, kb0 + 2 * kBN, ids);
        } else {
            issue(src, 2, kb0 + 2 * kBN, ids);
        }
        fetch(src, kb0 + 3 * kBN, ids);
        auto stage = [&](int j) { return lds0 + (j % STAGES) * STAGE; };
        auto read_k = [&](uint32_t ka, int ds, int kt) { return lds_read((ka ^ (ds << 5)) + kt * 32 * ROW); };
        auto apply_mask = [&](f32x16 (&s)[2], int k0) {
            const int x = lim - k0 - 4 * (lane_id() >> 5);
#pragma unroll
            for (int kt = 0; kt < 2; ++kt)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    s[kt][r] = kt * 32 + 8 * (r / 4) + r % 4 > x ? -INFINITY : s[kt][r];
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
        // scores of tile j + 1, then P.V of tile j, with the softmax of tile j and the operand reads placed between them by
        // scheduling fences so that the VALU issues while the matrix cores run.
        const int n_live = max(0, min(n_tiles, (kend_w - kb0 + kBN - 1) / kBN));   // the wave's tiles
        auto needs_mask = [&](int j) { return kb0 + j * kBN + kBN - 1 > lim_w; };
        auto block = [&](const f32x16 (&cur)[2], f32x16 (&nxt)[2], uint32_t ka, uint32_t va) {
            constexpr int NQ = 2 * DS, NP = 4 * DT, NS = NQ + NP;
            constexpr int KAHEAD = 2, VAHEAD = 2;             // operand reads ahead of their slot
            const float nb = kLift<KT> - (m == -INFINITY ? 0.0f : m);   // no visible key yet: every s is -inf
            u32x4 kf[NQ], vf[NP];
            float pe[32];
            uint32_t pp[16];
            float ps = lsum;
            auto get_k = [&](int i) { kf[i] = read_k(ka, i >> 1, i & 1); };
            auto get_v = [&](int p) {
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
            for (int i = 0; i < KAHEAD; ++i) get_k(i);
#pragma unroll
            for (int sl = 0; sl < NS; ++sl) {
                if (sl < NQ) {
                    const int ds = sl >> 1, kt = sl & 1;
                    nxt[kt] = F::mma(as_vec<QF>(kf[sl]), qf[ds], ds == 0 ? f32x16{} : nxt[kt]);
                    if (sl + KAHEAD < NQ) get_k(sl + KAHEAD);
                } else {
                    const int p = sl - NQ, ch = p / DT;
                    const QF pf = as_vec<QF>(u32x4{pp[4 * ch], pp[4 * ch + 1], pp[4 * ch + 2], pp[4 * ch + 3]});
                    o[p % DT] = F::mma(as_vec<QF>(vf[p]), pf, o[p % DT]);
                }
                if (sl - NQ + VAHEAD >= 0 && sl - NQ + VAHEAD < NP) get_v(sl - NQ + VAHEAD);
                valu_slot(sl);
                __builtin_amdgcn_sched_barrier(0);
            }
            lsum = ps;
        };
        // A tile that some row of the workgroup must not see all of: each wave
        // looks at its share of V, and where a value is not finite every row adds
        // the ones that it sees and the tile goes on with zeros in their places
        // (the order of the barriers is the workgroup's; seen by no other tile).
        const int lim_wg = uni(min(L - 1, past + div_g(a, min(c.rt * kRowsWG, rows - 1))));
        auto fix_tile = [&](int j) {
            const int lane = lane_id();
            const uint32_t vs = stage(j) + TB;
            constexpr int NF = TB / 1024 / kWaves;
            bool nf = false;
#pragma unroll
            for (int i = 0; i < NF; ++i) nf = nf || chunk_not_finite<KT>(lds_read(vs + (i * kWaves + w) * 1024 + lane * 16));
            ++fix_id;
            if (__any(nf)) *(volatile __attribute__((address_space(3))) int*)&fix = fix_id;
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
            if (*(volatile __attribute__((address_space(3))) int*)&fix != fix_id) return;
            add_not_finite<D, KT, kBN>(vs, kb0 + j * kBN, lim, lane >> 5, o);
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
#pragma unroll
            for (int i = 0; i < NF; ++i) {
                auto* p = lds_vec(vs + (i * kWaves + w) * 1024 + lane * 16);
                const u32x4 x = *p;
                *p = u32x4{finite2<KT>(x.x), finite2<KT>(x.y), finite2<KT>(x.z), finite2<KT>(x.w)};
            }
            asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" : : : "memory");
        };
        f32x16 sa[2], sb[2];
        float mx = 0.0f;
        if (n_live > 0) {
            uint32_t ka = stage(0) + k_off;
            asm volatile("" : "+v"(ka));                      // its variants are made here, not held
#pragma unroll
            for (int ds = 0; ds < DS; ++ds)
#pragma unroll
                for (int kt = 0; kt < 2; ++kt) sa[kt] = F::mma(as_vec<QF>(read_k(ka, ds, kt)), qf[ds], ds == 0 ? f32x16{} : sa[kt]);
            if (needs_mask(0)) apply_mask(sa, kb0);
            mx = rowmax(sa);
        }
        auto step = [&](int j, const f32x16 (&cur)[2], f32x16 (&nxt)[2]) {
            // K of tile j + 1 and V of tile j have landed, and every wave is done
            // with tile j - 1, whose stage tile j + 3 now takes
            asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)\n\ts_barrier" : : "n"(Q8 ? 63 : NI + NLD) : "memory");
            if constexpr (Q8) {
                put_q8(j + 2);
                load_q8(src, kb0 + (j + 3) * kBN, ids);
            } else {
                issue(src, j + 3, kb0 + (j + 3) * kBN, ids);
            }
            fetch(src, kb0 + (j + 4) * kBN, ids);
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
        for (int j = 0; j < n_tiles; j += 2) {
            step(j, sa, sb);
            if (j + 1 < n_tiles) step(j + 1, sb, sa);
        }
        if (__any(bad)) *(volatile __attribute__((address_space(3))) int*)&bad_seg = seg;
        asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)\n\ts_barrier" : : : "memory");   // the padding tiles' loads
    }
    if (!wave_live) continue;
    // ---- this workgroup's sums of the wave's rows (lanes l and l ^ 32 summed
    // different keys); with the other pieces' where the row tile has several
    const int ln = lane_id();
    const PagedArgs& args = fresh_args();
    float lt = add_swap32(lsum);
    bool nan = c.n_tiles > 0 && *(volatile __attribute__((address_space(3))) int*)&bad_seg == seg;
    bool done = true;
    if (!c.whole) {
        const int g0 = cuts.first_of(c.place, c.len), pieces = cuts.final_of(c.place, c.len) - g0 + 1;
        // piece k's slot: workgroup g0's second, the others' first
        auto piece_rsrc = [&](int k) {
            const int slot = k == 0 ? 2 * g0 + 1 : 2 * min(g0 + k, wgs - 1);
            return make_rsrc((const char*)(uintptr_t)uniform64((uint64_t)(uintptr_t)ws + (uint64_t)(slot * kWaves + w) * WAVE), WAVE);
        };
        auto store = [&](int k) {
            const BufRsrc rs = piece_rsrc(k);
#pragma unroll
            for (int i = 0; i < DT * 4; ++i)
                __builtin_amdgcn_raw_buffer_store_b128(
                    u32x4{__float_as_uint(o[i / 4][4 * (i % 4)]), __float_as_uint(o[i / 4][4 * (i % 4) + 1]),
                          __float_as_uint(o[i / 4][4 * (i % 4) + 2]), __float_as_uint(o[i / 4][4 * (i % 4) + 3])},
                    rs, ln * 16 + i * 1024, 0, kSc1);
            __builtin_amdgcn_raw_buffer_store_b64(u32x2{nan ? kNanBits : __float_as_uint(m), __float_as_uint(lt)}, rs,
                                                  WAVE_O + ln * 8, 0, kSc1);
        };
        // whether this wave is the last of n at the ticket; its stores are done before
        auto last_of = [&](unsigned* tk, int n) {
            __builtin_amdgcn_s_waitcnt(0);
            unsigned old = 0;
            if (ln == 0) {
                old = __hip_atomic_fetch_add(tk, 1u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                if (old == (unsigned)(n - 1)) __hip_atomic_store(tk, 0u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
            }
            return __builtin_amdgcn_readfirstlane((int)old) == n - 1;
        };
        // pieces first, first + by, ... (n of them) added in this order
        auto add = [&](int first, int by, int n) {
            float M = -INFINITY, den = 0.0f;
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) o[dt] = f32x16{};
#pragma unroll 1
            for (int i = 0; i < n; ++i) {
                const BufRsrc rs = piece_rsrc(first + i * by);
                const u32x2 e = __builtin_amdgcn_raw_buffer_load_b64(rs, WAVE_O + ln * 8, 0, kSc1);
                u32x4 v[DT * 4];                   // loaded together: one round trip
#pragma unroll
                for (int k = 0; k < DT * 4; ++k) v[k] = __builtin_amdgcn_raw_buffer_load_b128(rs, ln * 16 + k * 1024, 0, kSc1);
                __builtin_amdgcn_sched_barrier(0);
                const bool hit = e.x == kNanBits;
                nan = nan || hit;
                const float mi = hit ? -INFINITY : __uint_as_float(e.x);
                const float mn = fmaxf(M, mi), base = mn == -INFINITY ? 0.0f : mn;
                const float f0 = __builtin_amdgcn_exp2f(M - base), f = __builtin_amdgcn_exp2f(mi - base);
                den = den * f0 + __uint_as_float(e.y) * f;
#pragma unroll
                for (int k = 0; k < DT * 4; ++k) {
#pragma unroll
                    for (int x = 0; x < 4; ++x) {
                        const int t = k / 4, r = 4 * (k % 4) + x;
                        o[t][r] = fmaf(__uint_as_float(v[k][x]), f, o[t][r] * f0);
                    }
                    __builtin_amdgcn_sched_barrier(0);
                }
                M = mn;
            }
            m = M;
            lt = den;
        };
        const int k = g - g0, grp = k / kGroup, groups = (pieces + kGroup - 1) / kGroup;
        store(k);
        unsigned* tk = tickets + kMaxWgs * kWaves + ((g0 * kWaves + w) * (kMaxWgs / kGroup) + grp);
        int first = grp * kGroup, by = 1, n = min(kGroup, pieces - first);
#pragma unroll 1
        for (int level = 0; level < 2; ++level) {
            if (n > 1) {
                done = last_of(tk, n);
                if (!done) break;
                add(first, by, n);
            }
            if (level > 0 || groups == 1) break;
            if (n > 1) store(first);               // its pieces have been added: the group's slot is the first one's
            tk = tickets + (g0 * kWaves + w);
            first = 0;
            by = kGroup;
            n = groups;
        }
    }
    if (done) {
        const int G = args.G, t0 = div_g(args, wr0);
        int t, h;
        small_divide(wr0 - t0 * G + (ln & 31), G, t, h);
        // lanes l and l + 32 have 4 dims each of 8: they trade halves of pairs
        // of such groups, so that each stores 16 bytes
        char* const op = args.out + (int64_t)(c.q0 + t0 + t) * args.o_nb_t + (int64_t)(c.kvh * G + h) * args.o_nb_h + 16 * (ln >> 5);
        // zeros where the row sees no key; all scores -inf: 0 * (1 / 0), the softmax's NaN
        const float inv = min(c.L - 1, c.past + t0 + t) >= 0 ? 1.0f / lt : 0.0f;
#pragma unroll
        for (int i = 0; i < DT * 2; ++i) {
            uint32_t y[2][2];
#pragma unroll
            for (int x = 0; x < 4; ++x) {
                const int q4 = 2 * (i % 2) + x / 2, r = 4 * q4 + 2 * (x % 2);
                y[x / 2][x % 2] = pack2<OT>(o[i / 2][r] * inv, o[i / 2][r + 1] * inv);
            }
            const auto s0 = __builtin_amdgcn_permlane32_swap(y[0][0], y[1][0], false, false);
            const auto s1 = __builtin_amdgcn_permlane32_swap(y[0][1], y[1][1], false, false);
            u32x4 z = {s0[0], s1[0], s0[1], s1[1]};
            if (nan) z = u32x4{0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu, 0x7fff7fffu};
            if (wr0 + (ln & 31) < c.rows) *(u32x4*)(op + i * 32) = z;
        }
    }
    }
}

template <int D, int PT, int OT>
__global__ void __launch_bounds__(kWaves * 64) paged_many_kernel(PagedArgs a, float* __restrict__ ws, unsigned* tickets) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    __shared__ __attribute__((aligned(1024))) char lds[ManyLds<D, PT>::BYTES];
    __shared__ int marks[2];
    const Seq mine = seq_of(a, min((int)threadIdx.x & 63, a.n_seq - 1));
    const ManyAxis axis = many_axis(a, mine);
    if (axis.head <= 0) return;
    const ManyPieces pc = many_pieces(a, axis, mine, gridDim.x, blockIdx.x);
    const int wgs = pc.head > 0 ? pc.head * a.Hkv : many_shares(a, axis, gridDim.x);
    if ((int)blockIdx.x < wgs) many_share<D, PT, OT>(a, ws, tickets, axis, pc, mine, blockIdx.x, wgs, lds, marks);
}

// Few rows beside many: share `item / Hkv` of kv head item % Hkv, the axis cut
// into at most `slots` equal shares, of a tile per wave and a piece's cost at
// least.  The workgroups are fewer than the pieces here, so that even work
// counts for more than what a cut costs (60 sequences of up to 8000 keys beside
// 700 tokens: 159 us with whole pieces by turns, 97 so).  False: no share.
template <int D, int PT, int OT>
__device__ __forceinline__ bool few_share(const PagedArgs& a, float* __restrict__ ws, unsigned* tickets, int cap, int item, int slots, int axis, const Seq& mine, char* lds) {
    const int n = max(1, min(slots, axis / (kWaves + kFewCost)));
    const Shares cuts{(axis + n - 1) / n, n, max(kFewCost + 1, min(kFewSnap, (axis + n - 1) / n / 2))};
    const int g = item / a.Hkv, kvh = item - g * a.Hkv;
    const int p_end = min(axis, (g + 1) * cuts.share);
    if (g >= n) return false;
    const int lane = threadIdx.x & 63;
    bool begin = true;
    int base = 0, block = -64, end = 0, len = 0;   // 64 sequences from `block` on: where each ends
    Seq q{};
    for (int p = g * cuts.share; p < p_end;) {
        uint64_t hit;
        while (!(hit = __ballot(p >= end - len && p < end))) {
            block += 64;
            if (block >= a.n_seq) return true;     // a batch that changed meanwhile
            if (block > 0) base = lane_of(end, 63);
            q = block > 0 ? seq_of(a, min(block + lane, a.n_seq - 1)) : mine;
            len = block + lane < a.n_seq ? few_weight(a, q) : 0;
            end = base + wave_scan(len);
        }
        const int l = __ffsll((unsigned long long)hit) - 1;
        const int size = lane_of(len, l), x = lane_of(end, l) - size;
        FewItem it;
        it.q.q0 = lane_of(q.q0, l);
        it.q.n = lane_of(q.n, l);
        it.q.L = lane_of(q.L, l);
        it.q.s = block + l;
        const int off = (begin ? cuts.cut(p, x, size) : p) - x;
        const int off_end = (p_end < x + size ? cuts.cut(p_end, x, size) : x + size) - x;
        begin = false;
        p = x + size;
        if (off_end <= off) continue;              // moved past its end, or its end to here
        it.first = off > 0 || off_end < size ? cuts.first_of(x, size) : g;
        it.parts = off > 0 || off_end < size ? cuts.final_of(x, size) - it.first + 1 : 1;
        it.part = g - it.first;
        it.t0 = max(0, off - kFewCost);            // a cut is more than kFewCost from the ends, or at one
        it.t1 = min(off_end - kFewCost, (it.q.L + kFewTile - 1) / kFewTile);   // no keys: none
        few_piece<D, PT, OT, kWaves, 32, true>(a, ws, tickets, cap, it, kvh, lds);
        __syncthreads();                           // the next piece's rows of Q go where this one's sums are
    }
    return true;
}

// Sequences of both kinds in one launch of a workgroup per CU: the first take
// shares of the many rows' work, the others of the few rows', as many as the
// times of both kinds say (on the device, from the batch).  So the bytes of the
// one come while the matrix cores work on the other, and no launch waits.
// Against the two kernels one after the other: 64 x 4096 keys and 512 tokens
// behind 4096 142 -> 109 us, 23 x 2000 and 512 tokens 50 -> 29, 1.5B prompts of
// 40 to 1100 tokens (no few rows) 35 -> 27; 8 x 1024 alone in a call that could
// have brought more 10 -> 13, 64 x 4096 alone 90 -> 85.
// Time of a few-row tile to that of a key tile of a row tile (0.16 and 0.22: D =
// 64, 64 x 2000 keys and 512 tokens 21.9 and 25.4 us; D = 128, 60 sequences of up
// to 8000 and 700 behind 2000 105 and 97), over 16-bit pages.  Q8_0 ones take the
// same: neither it nor the costs that are counted in tiles (kFewCost, kFewSnap,
// kRowTileCost) was fitted for them.
template <int D>
constexpr float kFewTime = D == 64 ? 0.16f : 0.22f;
template <int D, int PT, int OT>
__global__ void __launch_bounds__(kWaves * 64) paged_mixed_kernel(PagedArgs a, float* __restrict__ ws, float* __restrict__ few_ws, unsigned* tickets, int cap) {
    prefetch_kernargs<sizeof(PagedArgs)>();
    constexpr int FEW = FewLds<D, PT, kWaves, 32>::BYTES;
    __shared__ __attribute__((aligned(1024))) char lds[ManyLds<D, PT>::BYTES > FEW ? ManyLds<D, PT>::BYTES : FEW];
    __shared__ int marks[2];
    const Seq mine = seq_of(a, min((int)threadIdx.x & 63, a.n_seq - 1));
    const ManyAxis axis = many_axis(a, mine);
    const int few = few_axis(a, mine);
    int wgs = 0;
    if (axis.head > 0) {
        const float many = (float)(axis.head * a.Hkv) * (float)(1 << axis.shift) * (1.0f / 16), rest = kFewTime<D> * (float)few * (float)a.Hkv;
        const int n = (int)((float)gridDim.x * many * __builtin_amdgcn_rcpf(many + rest) * (1.0f / 8) + 0.5f) * 8;
        const int most = max(8, min(n, (int)gridDim.x - (few > 0 ? 8 : 0)));
        const ManyPieces pc = many_pieces(a, axis, mine, most, blockIdx.x);
        wgs = pc.head > 0 ? pc.head * a.Hkv : many_shares(a, axis, most);
        if ((int)blockIdx.x < wgs) {
            many_share<D, PT, OT>(a, ws, tickets, axis, pc, mine, blockIdx.x, wgs, lds, marks);
            return;
        }
    }
    if (few == 0) return;
    const int slots = max(1, ((int)gridDim.x - wgs) / a.Hkv);
    for (int i = blockIdx.x - wgs; few_share<D, PT, OT>(a, few_ws, tickets + kManyTickets, cap, i, slots, few, mine, lds);) i += gridDim.x - wgs;
}

size_t many_ws_bytes(const PagedArgs& a, const PagedPlan& p) {
    return (size_t)p.many_wgs * 2 * kWaves * (a.d * kRowsWave * sizeof(float) + 64 * 8);
}

template <int D, int PT, int OT>
hipError_t launch_paged(const PagedArgs& a, const PagedPlan& p, float* ws, unsigned* tickets, hipStream_t s) {
    if (p.many_wgs > 0 && p.few_pieces > 0) {
        hipLaunchKernelGGL((paged_mixed_kernel<D, PT, OT>), dim3(p.many_wgs), dim3(kWaves * 64), 0, s, a, ws, (float*)((char*)ws + many_ws_bytes(a, p)), tickets, p.few_cap);
    } else if (p.many_wgs > 0) {
        hipLaunchKernelGGL((paged_many_kernel<D, PT, OT>), dim3(p.many_wgs), dim3(kWaves * 64), 0, s, a, ws, tickets);
    } else {
        const dim3 g(p.few_pieces * a.Hkv), b(p.few_waves * 64);
        if constexpr (PT == VVA_TYPE_Q8_0) {
            if (p.few_waves == 8) {
                hipLaunchKernelGGL((paged_few_kernel<D, PT, OT, 8, 16>), g, b, 0, s, a, ws, tickets, p.few_slots, p.few_cap);
                return hipGetLastError();
            }
        }
        hipLaunchKernelGGL((paged_few_kernel<D, PT, OT, kFewWaves, 32>), g, b, 0, s, a, ws, tickets, p.few_slots, p.few_cap);
    }
    return hipGetLastError();
}

template <int D>
hipError_t launch_typed(const PagedArgs& a, const PagedPlan& p, float* ws, unsigned* tickets, hipStream_t s) {
    if (a.type == VVA_TYPE_Q8_0)
        return a.io_type == VVA_TYPE_F16 ? launch_paged<D, VVA_TYPE_Q8_0, VVA_TYPE_F16>(a, p, ws, tickets, s)
                                         : launch_paged<D, VVA_TYPE_Q8_0, VVA_TYPE_BF16>(a, p, ws, tickets, s);
    return a.type == VVA_TYPE_F16 ? launch_paged<D, VVA_TYPE_F16, VVA_TYPE_F16>(a, p, ws, tickets, s)
                                  : launch_paged<D, VVA_TYPE_BF16, VVA_TYPE_BF16>(a, p, ws, tickets, s);
}

static_assert(kManyTickets + 2 * kFewTickets <= kMaxPagedTickets, "the context holds the tickets");

}  // namespace

// What a call of these shapes may need: the lengths are on the device, so
// every count here is the most there can be, and workgroups beyond the work
// there is end at once.
PagedPlan paged_plan(const PagedArgs& a, int n_cu) {
    PagedPlan p{};
    const int64_t rows = (int64_t)a.max_new * a.G;
    const int64_t max_keys = (int64_t)a.max_pages << a.page_shift;
    // Every sequence brings max_new tokens where their number says so: one
    // kernel is launched, which takes any others as well (a batch padded to its
    // token rows).
    const bool even = (int64_t)a.n_seq * a.max_new == a.n_tok;
    if (rows > kFewRows) p.many_wgs = std::max(16, std::min(n_cu, kMaxWgs));   // 8 for each kind at least
    if (rows <= kFewRows || !even) {
        p.few_cap = (int)std::min<int64_t>(rows, kFewRows);
        // Half the workgroups that fit a CU, so that fewer partials are added and
        // no CU's share of the bytes is less (1 x 32768 keys 29.3 -> 22.3 us, 64 x 4096
        // 88.8 -> 83.8); all of them where the sequences are too many to be cut evenly
        // into that few (48 of 500 to 8000 keys: 94.2 -> 79.3)
        // Q8_0 pages and at most 16 rows: twice the waves in a workgroup
        p.few_waves = a.type == VVA_TYPE_Q8_0 && rows <= 16 ? 8 : kFewWaves;
        // of 17 to 32 rows of 64 dims over Q8_0 pages three fit, by their registers: two are
        // taken, for many sequences too (0.5B heads, 4 tokens, us with 4, 3 and 2: 130 sequences
        // of up to 4000 keys 36.9, 37.6, 32.8, 256 of up to 1000 28.7, 27.1, 22.0)
        const bool two = a.type == VVA_TYPE_Q8_0 && a.d == 64 && p.few_waves == kFewWaves;
        const int slots = std::min(n_cu, kMaxWgs) * (a.d == 64 && p.few_waves == kFewWaves ? 2 : 1);
        p.few_slots = std::max(1, (2 * a.n_seq * a.Hkv > slots && !two ? 2 : 1) * slots / a.Hkv);
        const int64_t seq_tiles = (max_keys + kFewTile - 1) / kFewTile;
        p.few_split = seq_tiles > (p.many_wgs > 0 ? kFewWaves : p.few_waves);
        p.few_pieces = (int)std::min<int64_t>(p.few_slots + (int64_t)a.n_seq, a.n_seq * ((seq_tiles + p.few_waves - 1) / p.few_waves));
    }
    return p;
}
size_t paged_ws_bytes(const PagedArgs& a, const PagedPlan& p) {
    // beside many rows: two places per share
    const size_t places = p.many_wgs > 0 ? (size_t)2 * std::max(p.many_wgs, a.Hkv) : (size_t)p.few_pieces * a.Hkv;
    return many_ws_bytes(a, p) + (p.few_split ? places * p.few_cap * (a.d + 2) * sizeof(float) : 0);
}

hipError_t launch_paged_attn(PagedArgs a, const PagedPlan& p, float* ws, unsigned* tickets, hipStream_t s) {
    a.few_rows = p.few_pieces > 0 ? kFewRows : 0;
    return a.d == 64 ? launch_typed<64>(a, p, ws, tickets, s) : launch_typed<128>(a, p, ws, tickets, s);
}

}  // namespace vva
