// paged_q8.hpp — Q8_0 pages in paged_attn.hip: their loads, their values as
// operands of v_mfma_f32_32x32x16_f16, and the few rows' walk over them.
// gfx950 only.  Included inside the anonymous namespace of paged_attn.hip.
//
// A run (a page of a head) is page_size rows of D codes, then D / 32 rows of
// page_size F16 scales.  Codes go into LDS as they are, 16-byte chunk c of row r
// at chunk c ^ f(r); beside a tile's codes lie its scales, [block][key].
#pragma once

typedef int i32x2 __attribute__((ext_vector_type(2)));

// XORed to the chunk index of a row of codes, so that what a phase of a read takes
// lies on different banks: K in chunks of 8 rows; V in 32 bytes of each of 8 rows (f
// even: a pair of chunks stays one); with 16-row products, K in half chunks of rows
// 8 i + 0 .. 3, and V as K is in the first case
template <int D> __device__ __forceinline__ int kq_swz(int row) { return D == 128 ? (row >> 1) & 7 : (row >> 2) & 3; }
template <int D> __device__ __forceinline__ int vq_swz(int row) { return D == 128 ? row & 6 : (row >> 1) & 2; }
template <int D> __device__ __forceinline__ int kq16_swz(int row) { return D == 128 ? (row >> 2 & 6) | (row >> 1 & 1) : row >> 3 & 3; }

// 64 lanes' 4 bytes, each from an address of its own, to LDS lds .. lds + 255; as
// dma16, non-temporal
__device__ __forceinline__ void dma4(uint64_t addr, uint32_t lds) {
    asm volatile("s_mov_b32 m0, %0\n\ts_nop 4\n\tglobal_load_lds_dword %1, off nt"
                 :
                 : "s"(__builtin_amdgcn_readfirstlane(lds)), "v"(addr)
                 : "memory", "m0");
}
// a T at base + off (a pointer made of integers alone would be a flat one)
template <typename T>
__device__ __forceinline__ T global_load(uint64_t base, uint32_t off) {
    return *(const __attribute__((address_space(1))) T*)((const __attribute__((address_space(1))) char*)base + off);
}
__device__ __forceinline__ h2 as_h2(uint32_t x) {
    h2 v;
    __builtin_memcpy(&v, &x, 4);
    return v;
}
__device__ __forceinline__ uint32_t as_bits(h2 v) {
    uint32_t x;
    __builtin_memcpy(&x, &v, 4);
    return x;
}
__device__ __forceinline__ h2 q8_scale(uint16_t bits) { return as_h2(bits | ((uint32_t)bits << 16)); }

// 4 codes as two pairs of F16: 1024 + (code + 128) has the code's byte as its
// last bits, so a byte permutation and an exact subtraction make a pair.
__device__ __forceinline__ void q8_codes(uint32_t codes, h2& a, h2& b) {
    const uint32_t x = codes ^ 0x80808080u;
    const h2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
    a = as_h2(__builtin_amdgcn_perm(0x64646464u, x, 0x04010400u)) - bias;
    b = as_h2(__builtin_amdgcn_perm(0x64646464u, x, 0x04030402u)) - bias;
}
// 8 codes (two words) times a pair's scales each, as an operand of 8 F16, and
// what its rounding left (exact but for the smallest values; the operand is
// infinite beyond 65504, and the rest of no use)
struct Q8Frag {
    u32x4 hi, lo;
};
template <bool LO>
__device__ __forceinline__ Q8Frag q8_frag(uint32_t c0, uint32_t c1, const h2 (&scale)[4]) {
    h2 c[4];
    q8_codes(c0, c[0], c[1]);
    q8_codes(c1, c[2], c[3]);
    Q8Frag f;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const h2 v = c[i] * scale[i];
        f.hi[i] = as_bits(v);
        if constexpr (LO) f.lo[i] = as_bits(__builtin_elementwise_fma(c[i], scale[i], -v));
    }
    return f;
}
// The rest beside an operand whose values may be infinite or NaN: none where they are
__device__ __forceinline__ u32x4 q8_rest(u32x4 hi, u32x4 lo) {
    u32x4 r;
#pragma unroll
    for (int i = 0; i < 4; ++i)
        r[i] = ((hi[i] & 0x7c00u) == 0x7c00u ? 0u : lo[i] & 0xffffu) | ((hi[i] & 0x7c000000u) == 0x7c000000u ? 0u : lo[i] & 0xffff0000u);
    return r;
}
// whether either of two scales may take a code's value beyond F16, or is not finite
__device__ __forceinline__ bool q8_big2(uint32_t x) { return (x & 0x7fffu) >= 0x6000u || ((x >> 16) & 0x7fffu) >= 0x6000u; }

// add(e, v) for each of 4 codes whose value v is infinite or NaN, where it is seen
template <typename F>
__device__ __forceinline__ void q8_add_not_finite4(uint32_t codes, h2 scale, bool seen, F add) {
    h2 x[2];
    q8_codes(codes, x[0], x[1]);
#pragma unroll
    for (int e = 0; e < 4; ++e) {
        const float v = (float)(x[e / 2] * scale)[e % 2];
        if (seen && (__float_as_uint(v) & 0x7f800000u) == 0x7f800000u) add(e, v);
    }
}
// O += the infinities and NaNs of a tile's V that this lane's row sees (keys k0
// .. of the tile up to lim).  Codes of N rows at v_lds, scales [block][N] at s_lds.
template <int D, int N>
__device__ __forceinline__ void q8_add_not_finite(uint32_t v_lds, uint32_t s_lds, int k0, int lim, int half, f32x16 (&o)[D / 32]) {
    for (int j = 0; j < N; ++j) {
        const bool seen = k0 + j <= lim;
#pragma unroll
        for (int dt = 0; dt < D / 32; ++dt) {
            const h2 s = q8_scale(*(const __attribute__((address_space(3))) uint16_t*)lds_at(s_lds + (dt * N + j) * 2));
#pragma unroll
            for (int q4 = 0; q4 < 4; ++q4) {
                const uint32_t c = *(const __attribute__((address_space(3))) uint32_t*)lds_at(
                    v_lds + j * D + (((2 * dt + (q4 >> 1)) ^ vq_swz<D>(j)) << 4) + 8 * (q4 & 1) + 4 * half);
                q8_add_not_finite4(c, s, seen, [&](int e, float v) { o[dt][4 * q4 + e] += v; });
            }
        }
    }
}

// A wave's tiles of 32 keys of a sequence and kv head, from the pages into LDS
// stages: the codes of K, of V, then the scales of K, of V.  ROWS16: for products of
// 16 rows.  HOLD: the lane's offsets stay in registers through the tiles, where there
// are any left (made anew for each tile: 48 sequences 46.2 -> 46.8 us).
template <int D, bool ROWS16, bool HOLD>
struct Q8Tiles {
    static constexpr int NB = D / 32;              // blocks of a row
    static constexpr int CB = kFewTile * D, SB = kFewTile * NB * 2;    // codes and scales of a tile
    static constexpr int STAGE = 2 * (CB + SB);
    static constexpr int NC = CB / 1024, RC = 1024 / D;                // loads of a tile's codes, rows of one
    static constexpr int NL = NC + 1;              // with its scales
    static constexpr int NV = 16 / RC;             // loads of 16 keys

    const PagedArgs& a;
    const ConstInts table;
    const int kvh, last_page, held;
    int ids[2];                                    // pages of the two 16-key halves of the next tile to load
    bool bad = false;

    static __device__ __forceinline__ int k_swz(int row) { return ROWS16 ? kq16_swz<D>(row) : kq_swz<D>(row); }
    static __device__ __forceinline__ int v_swz(int row) { return ROWS16 ? kq_swz<D>(row) : vq_swz<D>(row); }

    __device__ __forceinline__ Q8Tiles(const PagedArgs& args, const FewItem& it, int head, int lane)
        : a(args), table((ConstInts)(uintptr_t)(args.table + (int64_t)it.q.s * args.table_stride)), kvh(head),
          last_page((it.q.L - 1) >> args.page_shift), held(lane) {}
    __device__ __forceinline__ void fetch(int t) {
#pragma unroll
        for (int i = 0; i < 2; ++i) ids[i] = table[min((t * kFewTile + 16 * i) >> a.page_shift, last_page)];
    }
    template <bool V>
    __device__ __forceinline__ void issue(int t, uint32_t codes, uint32_t scales, const char* pool, int64_t nb_page, int64_t nb_head) {
        const int lane = HOLD ? held : lane_id();
        uint64_t run[2];
        int slot[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const bool ok = (uint32_t)ids[i] < (uint32_t)a.n_pages;
            bad = bad || !ok;
            run[i] = uniform64((uint64_t)(uintptr_t)pool + (int64_t)(ok ? ids[i] : 0) * nb_page + kvh * nb_head);
            slot[i] = (t * kFewTile + 16 * i) & ((1 << a.page_shift) - 1);
        }
#pragma unroll
        for (int c = 0; c < NC; ++c) {
            // of the load's rows, in their 16-key half; the swizzle of the upper half is the lower one's with bits turned
            const int row = c % NV * RC + lane / (D / 16), chunk = (lane % (D / 16)) ^ (V ? v_swz(row) : k_swz(row));
            const int turn = c / NV ? (V ? v_swz(16) : k_swz(16)) : 0;
            dma16<true>(run[c / NV] + (uint64_t)slot[c / NV] * D, (row * D + chunk * 16) ^ (turn << 4), codes + c * 1024);
        }
        // two keys of a block a lane
        const uint64_t s0 = run[0] + 2 * slot[0], s1 = run[1] + 2 * slot[1];
        const int soff = (D << a.page_shift) + (((lane >> 4) << a.page_shift) + 2 * (lane & 7)) * 2;
        if (D == 128 || lane < 32) dma4((lane & 8 ? s1 : s0) + soff, scales);
    }
    __device__ __forceinline__ void issue_k(int t, uint32_t st) { issue<false>(t, st, st + 2 * CB, a.k, a.k_nb_page, a.k_nb_head); }
    __device__ __forceinline__ void issue_v(int t, uint32_t st) { issue<true>(t, st + CB, st + 2 * CB + SB, a.v, a.v_nb_page, a.v_nb_head); }
    // The rows of Q, and the first tiles (t, t + WAVES) into the ring's stages, until Q has landed
    template <int WAVES, int ROWS, int STAGES>
    __device__ __forceinline__ void begin(const FewItem& it, int rows, int t, uint32_t qs, uint32_t ring) {
        if (t < it.t1) fetch(t);
        few_load_q<D, WAVES, ROWS>(a, it, kvh, rows, qs);
        if (t < it.t1) {
            issue_k(t, ring);
            issue_v(t, ring);
            if (STAGES == 2 && t + WAVES < it.t1) {
                fetch(t + WAVES);
                issue_k(t + WAVES, ring + STAGE);
                issue_v(t + WAVES, ring + STAGE);
                wait_vm<4 * NL>();
            } else {
                wait_vm<2 * NL>();
            }
        } else {
            wait_vm<0>();
        }
        asm volatile("s_barrier" : : : "memory");
    }
    // whether a tile's scales may take a value beyond F16 or are not finite (whole wave)
    __device__ __forceinline__ bool big(uint32_t scales) const {
        return (bool)__any(q8_big2(*(const __attribute__((address_space(3))) uint32_t*)lds_at(scales + ((HOLD ? held : lane_id()) & (SB / 4 - 1)) * 4)));
    }
};

// The tiles t0 + w, + WAVES, ... below t1 of a piece, as few_stream: of 32 keys,
// two under way while one is computed (a stage is 8.5 KB: one alone would leave
// less than half of what the 16-bit tiles have in flight).
// LO: the rounding of scale times code to F16 goes into the products as well,
// in a second one with the rest, so that K and V are what the pages hold but for
// 2^-22: results rounded to F16 show it (error of a 30k-key step 4.1e-4 of its
// size without, 2.7e-4 with, of which the rounding of the result is 2.1e-4; BF16
// ones do not).  Against tiles converted to F16 on their way into LDS, one under
// way: 48 sequences of 500 to 8000 keys (216 MB) 61.4 -> 48.1 us.  4 tokens a
// sequence, 7B heads: 48 of them 51.7 us (BF16), 60.2 (F16, whose second products
// show), one behind 30k keys 24.9.
template <int D, int OT, int WAVES>
__device__ __forceinline__ void few_stream_q8(const PagedArgs& a, const FewItem& it, int kvh, char* lds, FewSums<D, 32>& r) {
    using F = Frag<VVA_TYPE_F16>;
    constexpr int KT = VVA_TYPE_F16;
    constexpr bool LO = OT == VVA_TYPE_F16;
    using T = Q8Tiles<D, false, true>;
    constexpr int NB = T::NB, CB = T::CB, SB = T::SB, STAGE = T::STAGE, NL = T::NL;
    const int lane = threadIdx.x & 63, half = lane >> 5, l32 = lane & 31;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = it.q.L, rows = min(it.q.n, a.max_new) * a.G, past = L - it.q.n, t1 = it.t1;
    const uint32_t qs = (uint32_t)(uintptr_t)(lds_char*)lds, ring = qs + 32 * 2 * D + w * 2 * STAGE;
    T tiles(a, it, kvh, lane);
    int t = it.t0 + w;
    tiles.template begin<WAVES, 32, 2>(it, rows, t, qs, ring);
    // The keys of a tile in the order in which the transposing read of V gives
    // them: row x of the scores' operand is key x with bits 2 and 3 exchanged,
    // so a lane's accumulators are keys 16 kk + 8 half + 0 .. 7.  Of a block a lane
    // reads 16 dims of its key at once, so Q's dims are taken in that order too.
    const int key = (l32 & 19) | ((l32 & 4) << 1) | ((l32 & 8) >> 1);
    const int k_off = key * D + ((half ^ kq_swz<D>(key)) << 4);
    const int v_row = 8 * half + ((lane & 15) >> 1);
    const int v_off = v_row * D + ((((lane >> 4) & 1) ^ vq_swz<D>(v_row)) << 4) + 8 * (lane & 1);
    h8 qf[2 * NB];
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
        for (int e = 0; e < 2; ++e) qf[2 * b + e] = q_frag<KT, OT>(lds_read(qs + l32 * 2 * D + (((4 * b + 2 * half + e) ^ k_swz<D>(l32)) << 4)));
    const int lim = l32 < rows ? min(L - 1, past + div_g(a, l32)) : -1;   // the last key the lane's row sees
    const float sl2 = a.scale * kLog2e;
    for (uint32_t st = ring; t < t1; t += WAVES, st = st == ring ? ring + STAGE : ring) {
        const bool one = t + WAVES < t1, two = t + 2 * WAVES < t1;
        const uint32_t ks = st + 2 * CB, vs = ks + SB;
        if (two) tiles.fetch(t + 2 * WAVES);
        if (one) wait_vm<3 * NL>();                // K; V and the next tile may still fly
        else wait_vm<NL>();
        f32x16 s{};
        {
            u32x4 c[NB];
            uint16_t sc[NB];
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                c[b] = lds_read((st + k_off) ^ (b << 5));
                sc[b] = *(const __attribute__((address_space(3))) uint16_t*)lds_at(ks + b * kFewTile * 2 + key * 2);
            }
            auto scores = [&](auto care) {
#pragma unroll
                for (int b = 0; b < NB; ++b) {
                    const h2 x = q8_scale(sc[b]);
                    const h2 x4[4] = {x, x, x, x};
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        Q8Frag f = q8_frag<LO>(c[b][2 * e], c[b][2 * e + 1], x4);
                        if constexpr (decltype(care)::value) f.lo = q8_rest(f.hi, f.lo);
                        s = F::mma(as_vec<h8>(f.hi), qf[2 * b + e], s);
                        if constexpr (LO) s = F::mma(as_vec<h8>(f.lo), qf[2 * b + e], s);
                    }
                }
            };
            if constexpr (LO) {
                if (tiles.big(ks)) scores(std::true_type{});
                else scores(std::false_type{});
            } else {
                scores(std::false_type{});
            }
        }
        if (two) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // K is read
            tiles.issue_k(t + 2 * WAVES, st);
        }
        const int k0 = t * kFewTile;
        const bool masked = k0 + kFewTile - 1 > min(L - 1, past);      // some row must not see some key
        if (masked) {
#pragma unroll
            for (int x = 0; x < 16; ++x) s[x] = 16 * (x / 8) + x % 8 > lim - k0 - 8 * half ? -INFINITY : s[x];
        }
        uint32_t p[8];
        [[maybe_unused]] uint32_t none[8];
        few_probs<D, KT>(s, sl2, r, p, none);
        if (two) wait_vm<3 * NL>();                // V; what was asked for after it may still fly
        else if (one) wait_vm<2 * NL>();
        else wait_vm<0>();
        // the products straight through; a tile with a value that is not finite, or
        // near the end of F16, by a path of its own
        auto values = [&](auto care) {
#pragma unroll
            for (int kk = 0; kk < 2; ++kk) {
                const h8 pf = as_vec<h8>(u32x4{p[4 * kk], p[4 * kk + 1], p[4 * kk + 2], p[4 * kk + 3]});
#pragma unroll
                for (int dt = 0; dt < NB; ++dt) {
                    const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32(
                        (__attribute__((address_space(3))) i32x2*)lds_at(((st + CB + v_off) ^ (dt << 5)) + kk * 16 * D));
                    const u32x4 sc = lds_read(vs + dt * kFewTile * 2 + kk * 32 + half * 16);
                    const h2 x4[4] = {as_h2(sc.x), as_h2(sc.y), as_h2(sc.z), as_h2(sc.w)};
                    Q8Frag f = q8_frag<LO>((uint32_t)c.x, (uint32_t)c.y, x4);
                    if constexpr (decltype(care)::value) {
                        if constexpr (LO) f.lo = q8_rest(f.hi, f.lo);
                        if (masked) f.hi = u32x4{finite2<KT>(f.hi.x), finite2<KT>(f.hi.y), finite2<KT>(f.hi.z), finite2<KT>(f.hi.w)};
                    }
                    r.o[dt] = F::mma(as_vec<h8>(f.hi), pf, r.o[dt]);
                    if constexpr (LO) r.o[dt] = F::mma(as_vec<h8>(f.lo), pf, r.o[dt]);
                }
            }
        };
        if ((LO || masked) && tiles.big(vs)) {
            values(std::true_type{});
            if (masked) q8_add_not_finite<D, kFewTile>(st + CB, vs, k0, lim, half, r.o);
        } else {
            values(std::false_type{});
        }
        if (two) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // V is read
            tiles.issue_v(t + 2 * WAVES, st);
        }
    }
    r.bad = tiles.bad;
}

// The same for at most 16 rows (single tokens of up to 16 heads a group), with
// v_mfma_f32_16x16x32_f16: half the scores and sums a lane holds, so twice the
// waves fit and the conversions, which are the most of a tile's arithmetic, have
// other waves' waits to run in.  One tile of 128 dims a wave is under way then
// (two of 64), 4 waves per SIMD.  Against 32 rows and half the waves, us: 30k keys
// 17.4 -> 14.9; 12 sequences of up to 8000 keys 20.5 -> 16.4, 48 48.1 -> 46.3; 24 of
// the 1.5B model 20.0 -> 16.0.  In workgroups of one per CU, beside many rows, it was
// slower (48 sequences 51 -> 57): those keep 32 rows.  Of 128 dims it takes 128 of 128
// VGPRs and one spilled register, 8 bytes of scratch a lane: built with 162 and none
// spilled, on as many workgroups, 30k keys 15.1 -> 15.6 us, 40 keys 6.1 -> 6.4.  Layouts (lane l, l16 = l % 16, g = l / 16):
//   A (16 x 32): row l16, k = 8 g .. 8 g + 7     B (32 x 16): column l16, the same k
//   C (16 x 16): column l16, register r holds row 4 g + r
// Row x of score tile mt is key 8 (x / 4) + 4 mt + x % 4, so a lane's 8 scores are
// keys 8 g .. 8 g + 7, the ones that the transposing read gives of a dim of V.
template <int D, int OT, int WAVES, int STAGES>
__device__ __forceinline__ void few_stream16_q8(const PagedArgs& a, const FewItem& it, int kvh, char* lds, FewSums<D, 16>& r) {
    constexpr int KT = VVA_TYPE_F16;
    constexpr bool LO = OT == VVA_TYPE_F16;
    using T = Q8Tiles<D, true, !(LO && D == 128)>;
    constexpr int NB = T::NB, CB = T::CB, SB = T::SB, STAGE = T::STAGE, NL = T::NL;
    const int lane = threadIdx.x & 63, g = lane >> 4, l16 = lane & 15;
    const int w = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int L = it.q.L, rows = min(it.q.n, a.max_new) * a.G, past = L - it.q.n, t1 = it.t1;
    const uint32_t qs = (uint32_t)(uintptr_t)(lds_char*)lds, ring = qs + 16 * 2 * D + w * STAGES * STAGE;
    T tiles(a, it, kvh, lane);
    int t = it.t0 + w;
    tiles.template begin<WAVES, 16, STAGES>(it, rows, t, qs, ring);
    const int key = 8 * (l16 >> 2) + (l16 & 3);
    const int k_off = key * D + (((g >> 1) ^ kq16_swz<D>(key)) << 4) + 8 * (g & 1);
    const int v_row = 8 * g + (l16 >> 1);
    const int v_off = v_row * D + (kq_swz<D>(v_row) << 4) + 8 * (lane & 1);
    h8 qf[NB];
#pragma unroll
    for (int b = 0; b < NB; ++b) qf[b] = q_frag<KT, OT>(lds_read(qs + l16 * 2 * D + (((4 * b + g) ^ k_swz<D>(l16)) << 4)));
    const int lim = l16 < rows ? min(L - 1, past + div_g(a, l16)) : -1;   // the last key the lane's row sees
    const float sl2 = a.scale * kLog2e;
    for (uint32_t st = ring; t < t1; t += WAVES, st = STAGES == 1 || st != ring ? ring : ring + STAGE) {
        const bool one = t + WAVES < t1, next = t + STAGES * WAVES < t1;
        const uint32_t ks = st + 2 * CB, vs = ks + SB;
        if (next) tiles.fetch(t + STAGES * WAVES);
        if (STAGES == 2 && one) wait_vm<3 * NL>(); // K; V and the next tile may still fly
        else wait_vm<NL>();
        f32x4 s[2] = {};
        {
            u32x2 c[NB][2];
            uint16_t sc[NB][2];
#pragma unroll
            for (int b = 0; b < NB; ++b)
#pragma unroll
                for (int mt = 0; mt < 2; ++mt) {
                    c[b][mt] = *(const __attribute__((address_space(3))) u32x2*)lds_at(((st + k_off) ^ (b << 5)) + mt * 4 * D);
                    sc[b][mt] = *(const __attribute__((address_space(3))) uint16_t*)lds_at(ks + b * kFewTile * 2 + (key + 4 * mt) * 2);
                }
            auto scores = [&](auto care) {
#pragma unroll
                for (int b = 0; b < NB; ++b)
#pragma unroll
                    for (int mt = 0; mt < 2; ++mt) {
                        const h2 x = q8_scale(sc[b][mt]);
                        const h2 x4[4] = {x, x, x, x};
                        Q8Frag f = q8_frag<LO>(c[b][mt].x, c[b][mt].y, x4);
                        if constexpr (decltype(care)::value) f.lo = q8_rest(f.hi, f.lo);
                        s[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_vec<h8>(f.hi), qf[b], s[mt], 0, 0, 0);
                        if constexpr (LO) s[mt] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_vec<h8>(f.lo), qf[b], s[mt], 0, 0, 0);
                    }
            };
            if constexpr (LO) {
                if (tiles.big(ks)) scores(std::true_type{});
                else scores(std::false_type{});
            } else {
                scores(std::false_type{});
            }
        }
        if (next) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // K is read
            tiles.issue_k(t + STAGES * WAVES, st);
        }
        const int k0 = t * kFewTile;
        const bool masked = k0 + kFewTile - 1 > min(L - 1, past);      // some row must not see some key
        if (masked) {
#pragma unroll
            for (int x = 0; x < 8; ++x) s[x / 4][x % 4] = x > lim - k0 - 8 * g ? -INFINITY : s[x / 4][x % 4];
        }
        float mx = fmaxf(fmaxf(fmaxf(s[0][0], s[0][1]), fmaxf(s[0][2], s[0][3])), fmaxf(fmaxf(s[1][0], s[1][1]), fmaxf(s[1][2], s[1][3])));
        mx = max_swap32(max_swap16(mx)) * sl2;
        if (__any(mx > r.m + kLazy)) {
            if (mx > r.m + kLazy) {
                const float alpha = __builtin_amdgcn_exp2f(r.m - mx);  // 0 while m = -inf
                r.lsum *= alpha;
#pragma unroll
                for (int i = 0; i < D / 16; ++i) r.o[i] *= alpha;
                r.m = mx;
            }
        }
        const float nb = kLift<KT> - (r.m == -INFINITY ? 0.0f : r.m);
        u32x4 p;
#pragma unroll
        for (int x = 0; x < 4; ++x) {
            p[x] = pack2<KT>(__builtin_amdgcn_exp2f(fmaf(s[x / 2][2 * (x % 2)], sl2, nb)), __builtin_amdgcn_exp2f(fmaf(s[x / 2][2 * (x % 2) + 1], sl2, nb)));
            r.lsum = sum2<KT>(p[x], r.lsum);
        }
        const h8 pf = as_vec<h8>(p);
        if (STAGES == 2 && next) wait_vm<3 * NL>();                    // V; what was asked for after it may still fly
        else if (STAGES == 2 && one) wait_vm<2 * NL>();
        else if (STAGES == 1 && next) wait_vm<NL>();
        else wait_vm<0>();
        // the products straight through; a tile with a value that is not finite, or
        // near the end of F16, by a path of its own
        auto values = [&](auto care) {
#pragma unroll
            for (int b = 0; b < NB; ++b) {
                const u32x4 sc = lds_read(vs + b * kFewTile * 2 + g * 16);
                const h2 x4[4] = {as_h2(sc.x), as_h2(sc.y), as_h2(sc.z), as_h2(sc.w)};
#pragma unroll
                for (int i = 2 * b; i < 2 * b + 2; ++i) {
                    const i32x2 c = __builtin_amdgcn_ds_read_tr8_b64_v2i32((__attribute__((address_space(3))) i32x2*)lds_at((st + CB + v_off) ^ (i << 4)));
                    Q8Frag f = q8_frag<LO>((uint32_t)c.x, (uint32_t)c.y, x4);
                    if constexpr (decltype(care)::value) {
                        if constexpr (LO) f.lo = q8_rest(f.hi, f.lo);
                        if (masked) f.hi = u32x4{finite2<KT>(f.hi.x), finite2<KT>(f.hi.y), finite2<KT>(f.hi.z), finite2<KT>(f.hi.w)};
                    }
                    r.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_vec<h8>(f.hi), pf, r.o[i], 0, 0, 0);
                    if constexpr (LO) r.o[i] = __builtin_amdgcn_mfma_f32_16x16x32_f16(as_vec<h8>(f.lo), pf, r.o[i], 0, 0, 0);
                }
            }
        };
        if ((LO || masked) && tiles.big(vs)) {
            values(std::true_type{});
            if (masked) {                          // a lane's dims of tile i: 16 i + 4 g ..
                for (int j = 0; j < kFewTile; ++j) {
                    const bool seen = k0 + j <= lim;
#pragma unroll
                    for (int i = 0; i < D / 16; ++i) {
                        const h2 sc = q8_scale(*(const __attribute__((address_space(3))) uint16_t*)lds_at(vs + ((i / 2) * kFewTile + j) * 2));
                        const uint32_t c = *(const __attribute__((address_space(3))) uint32_t*)lds_at(st + CB + j * D + ((i ^ kq_swz<D>(j)) << 4) + 4 * g);
                        q8_add_not_finite4(c, sc, seen, [&](int e, float v) { r.o[i][e] += v; });
                    }
                }
            }
        } else {
            values(std::false_type{});
        }
        if (next) {
            asm volatile("s_waitcnt lgkmcnt(0)" : : : "memory");       // V is read
            tiles.issue_v(t + STAGES * WAVES, st);
        }
    }
    r.bad = tiles.bad;
}
