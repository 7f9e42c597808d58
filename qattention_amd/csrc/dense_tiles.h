// dense_tiles.h -- the key loop of 128-row query tiles over K/V blocks of 64
// keys, for the kernels whose keys are a causal prompt or a paged context.
//
// A workgroup of 4 waves; each wave owns 32 query rows as the N dimension of
// v_mfma_f32_32x32x16 products.  Per block a wave runs
//   S^T = K Q^T      2 key tiles x D/16 k-steps   (A: K rows from LDS, B: Q in registers)
//   O^T += V^T P^T   4 16-key steps x D/32 d-tiles (A: V^T from LDS, B: P^T in registers)
// Lane l holds query l % 32; lanes l and l + 32 split the query's keys (S^T)
// and head dims (O^T), so the softmax statistics need one xor-32 exchange.
// Element r of S tile t is key 32 t + 8 (r / 4) + 4 (l / 32) + r % 4 of the
// block; element 4 j + e of d-tile dt is dim 32 dt + 8 j + 4 (l / 32) + e.
//
// The pipeline is the prefix kernel's (prefix_attn.hip, where its steps are
// explained and measured): iteration j forms S_{j+1} while the weights of block
// j are computed, then adds P_j V_j while the last of them and the maximum of
// block j + 1 are; the LDS-DMA loads of K_{j+3} and V_{j+1} are spread between
// the products, and two workgroups of a CU stay side by side by running odd
// iterations at a higher priority.
//
// A source says where the keys are:
//   kEveryBlock         any block may be without a key that a row attends (else
//                       every row attends a key of block 0)
//   load_k / load_v     all loads of block j into a buffer, before the loop
//   dma(j)              the loads of iteration j one by one: k(n), v(n) of
//                       K_{j+3} and V_{j+1} into the buffers of a parity
//   mask(j, s)          -inf for the keys of block j that a row does not attend
//   clean<SCAN>(j, v, o...)
//                       V rows of block j that no row attends set to 0.  SCAN:
//                       also, what is not finite in rows that only some attend
//                       (their weight is 0 for the others, and 0 times an infinity
//                       or a NaN is NaN) taken out of the block and added to the
//                       rows that do (o: the wave's numerators, none for a wave
//                       without rows).  By all waves of the workgroup, with the
//                       barriers it needs.
#pragma once

#include <type_traits>

#include "kv_tiles.h"

namespace qattn {

// A mean of values of T lies in T's range; its rounded weights may carry it just
// past: fp16's largest, 65504, would become an infinity.
template <typename T>
__device__ __forceinline__ float in_range(float x) {
    if constexpr (T::kCode == F16::kCode) {
        const float y = __builtin_amdgcn_fmed3f(x, -65504.f, 65504.f);
        return __builtin_fabsf(x) < 131072.f ? y : x;  // (an infinity or NaN stays)
    }
    return x;
}

template <typename T, int D>
struct DenseTile {
    static constexpr int kThreads = 256;
    static constexpr int kBN = 64;          // keys per block
    static constexpr int kBM = 128;         // rows per workgroup
    static constexpr int KS = D / 16;       // k-steps of S^T over the head dim
    static constexpr int DT = D / 32;       // 32-row d-tiles of O^T
    static constexpr int DV = D / 8;        // 16-byte chunks per key row
    static constexpr int BLK = kBN * D;     // elements of one K or V block
    static constexpr int NI = D / 32;       // 1 KB LDS loads per thread per K (or V) block
    static constexpr int RPI = 512 / D;     // key rows per 1 KB load
    static constexpr int kSmem = 4 * BLK;   // elements of LDS: K 0, K 1, V 0, V 1
    static_assert(NI * 4 * 512 == BLK, "a block is 4 waves x NI loads of 1 KB");

    // All but the N newest DMA loads and every LDS read of this wave are done,
    // then the workgroup's barrier: what was loaded may be read, what was read
    // may be overwritten.
    template <int N>
    static __device__ __forceinline__ void publish() {
        __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));  // vmcnt(N) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    }

    // LDS writes and reads of this wave are done, then the workgroup's barrier
    // (loads in flight stay so).
    static __device__ __forceinline__ void sync_lds() {
        __builtin_amdgcn_s_waitcnt((63 & 15) | ((63 >> 4) << 14) | (7 << 4));  // lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    }

    // The wave's 32 rows (Q^T in qf) over blocks 0 .. nb - 1 of src, onto the
    // state m_run (maximum of raw scores), l_run (this lane's half of the sum)
    // and oacc.  live: the wave has rows (else it only stages its part of the
    // blocks).  Ends with the workgroup past its last use of the LDS only after
    // the caller's barrier.
    template <bool SCAN, class Src>
    static __device__ __forceinline__ void keys(const Src& src, uint16_t* smem, const Vec16 (&qf)[KS], bool live,
                                                int nb, float csc, float& m_run, float& l_run, f16v_t (&oacc)[DT]) {
        const int lane = threadIdx.x & 63;
        const int q32 = lane & 31, hl = lane >> 5;
        uint16_t *const Kb0 = smem, *const Kb1 = smem + BLK, *const Vb0 = smem + 2 * BLK;
        // Operand read addresses: K (A of S^T, step s, key tile t): row 32 t +
        // q32, chunk 2 s + hl: (kaddr0 ^ 16 s) + 32 D t (the swizzle flips only
        // chunk bits, which the row base leaves clear).  V^T (A of O^T, 16-key
        // step th, d-tile dt): two ds_read_b64_tr_b16, X for keys 16 th + 4 hl +
        // 0..3 and Y for + 8; within each 16-lane group lane j points at row
        // key0 + j / 4, dims 32 dt + 16 ((lane >> 4) & 1) + 4 (j % 4) .. + 3, and
        // receives keys key0 + 0..3 at dim 32 dt + q32.
        const int kaddr0 = q32 * D + 8 * (hl ^ kv_swz32(q32, DV));
        int vx0, vy0;
        {
            const int rx = 4 * hl + ((lane & 15) >> 2), ry = rx + 8;
            const int cx = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
            vx0 = rx * D + 8 * (cx ^ kv_swz32(rx, DV)) + 4 * (lane & 1);
            vy0 = ry * D + 8 * (cx ^ kv_swz32(ry, DV)) + 4 * (lane & 1);
        }
        // hide() keeps the compiler from holding one register per address and
        // buffer, which spills.
        uint32_t kad[KS], vxa[DT], vya[DT];
        const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)smem;
#pragma unroll
        for (int s = 0; s < KS; ++s) kad[s] = lds0 + 2 * (kaddr0 ^ (16 * s));
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
            vxa[dt] = lds0 + 2 * (vx0 ^ (32 * dt));
            vya[dt] = lds0 + 2 * (vy0 ^ (32 * dt));
        }
        auto hide = [&] {
#pragma unroll
            for (int s = 0; s < KS; ++s) asm volatile("" : "+v"(kad[s]));
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) asm volatile("" : "+v"(vxa[dt]), "+v"(vya[dt]));
        };
        constexpr int NS = 2 * KS;  // products of S^T per block: k-step i / 2, key tile i % 2
        constexpr int NP = 4 * DT;  // products of O^T per block: 16-key step i / DT, d-tile i % DT
        constexpr int PF = 3;       // operands read ahead of their product
        auto fetch_k = [&](auto buf, int i) {
            typedef uint32_t v4u __attribute__((ext_vector_type(4)));
            const v4u x = *(__attribute__((address_space(3))) const v4u*)(uintptr_t)(
                kad[i >> 1] + 2 * (decltype(buf)::value * BLK + 32 * D * (i & 1)));
            return Vec16{{x[0], x[1], x[2], x[3]}};
        };
        auto fetch_v_at = [&](uint32_t buf_off, int i) {
            typedef short v4s __attribute__((ext_vector_type(4)));
            typedef __attribute__((address_space(3))) v4s* lds_v4s;
            const uint32_t off = buf_off + 2 * 16 * D * (i / DT);
            const v4s x = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)(vxa[i % DT] + off));
            const v4s y = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)(vya[i % DT] + off));
            const uint2 x2 = __builtin_bit_cast(uint2, x), y2 = __builtin_bit_cast(uint2, y);
            return Vec16{{x2.x, x2.y, y2.x, y2.y}};
        };
        auto fetch_v = [&](auto buf, int i) { return fetch_v_at(2 * (2 + decltype(buf)::value) * BLK, i); };

        // Online softmax: raw-score maximum, p = exp2(s c - m c).  l sums the
        // unrounded weights, by block and then over the blocks; P is rounded to
        // the inputs' type for its product, half a step of each weight, so the
        // largest weight is exact where it is 1.  bf16 (8 bits) therefore moves
        // the reference m on every new maximum, as the prefix kernel does: a
        // reference up to 2^8 below the maximum takes 5% less time (16384 tokens, 32
        // / 8 heads: 1900 us, so 1992; 16 x 603-2011, heads of 64: 168 and 180), but
        // is 2.4 times as far off ahead of the output's rounding where few keys have
        // most of the weight (1024 tokens, heads of 64, inputs of scale 2: largest
        // error 3.6e-2, so 1.7e-2).  fp16 (11 bits) moves it only when a block passes
        // it by 2^kLazy, so that the accumulators are rescaled on a handful of blocks.
        constexpr float kLazy = T::kCode == BF16::kCode ? 0.f : 8.f;
        float mc = 0.f, ps0 = 0.f, ps1 = 0.f;
        auto set_mc = [&] {
            // (no key yet, or none but of -inf scores: weights of 0, not NaN)
            mc = m_run == -INFINITY ? 0.f : m_run * csc;
        };
        auto move_ref = [&](float mb) {
            mb = xor32_max(mb);
            const bool move = (mb - m_run) * csc > kLazy;  // (on the first block with a key)
            if (__builtin_expect(__any(move), 0)) {
                const float m_new = move ? mb : m_run;
                const float alpha = move ? fast_exp2((m_run - m_new) * csc) : 1.f;  // m_run = -inf: 0
#pragma unroll
                for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
                l_run *= alpha;
                m_run = m_new;
            }
            set_mc();
        };
        // One block's 32 weights per lane, element n = 8 th + e of 16-key step
        // th, in three stages: exponent (0), exponential (1), sum and packing
        // (2).  Stage q of element n runs at step n NT / 32 + q of an iteration's
        // NS + NP products, so no instruction waits for the one before it and
        // step th's weights are packed before its first product.  (The empty asm
        // statements hold each result in its half of the iteration: the compiler
        // moved all exponentials and packing of the first half past the mask's
        // branch into the second, 1995 us -> 1965 for a prompt of 16384 tokens.)
        constexpr int NT = NS + 3 * DT - 2;
        Vec16 pf[4];
        auto stage = [&](f16v_t (&s)[2], int n, int q) {
            float x = s[n >> 4][n & 15];
            if (q == 0) x = __builtin_fmaf(x, csc, -mc);
            if (q == 1) {
                x = fast_exp2(x);
                asm volatile("" : "+v"(x));
            }
            s[n >> 4][n & 15] = x;
            if (q == 2) {
                if (n & 1) {
                    ps1 = n == 1 ? x : ps1 + x;
                    pf[n >> 3].w[(n & 7) >> 1] = MfmaOps<T>::pack2(s[n >> 4][(n & 15) - 1], x);
                    asm volatile("" : "+v"(ps1), "+v"(pf[n >> 3].w[(n & 7) >> 1]));
                } else {
                    ps0 = n == 0 ? x : ps0 + x;
                    asm volatile("" : "+v"(ps0));
                }
            }
        };
        auto weights_at = [&](f16v_t (&s)[2], int i) {
#pragma unroll
            for (int q = 2; q >= 0; --q)
#pragma unroll
                for (int n = 0; n < 32; ++n)
                    if (n * NT / 32 + q == i) stage(s, n, q);
        };
        auto zero = [](f16v_t (&s)[2]) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) s[t][r] = 0.f;
        };
        auto block_max = [](f16v_t (&s)[2]) {
            float mb = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) mb = fmaxf(fmaxf(mb, s[e >> 3][2 * (e & 7)]), s[e >> 3][2 * (e & 7) + 1]);
            return mb;
        };
        // Each step of the loop is kept in its place: the compiler's own order
        // put the operand reads next to their products and all exponentials
        // into the PV half.
        auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
        using B0 = std::integral_constant<int, 0>;
        using B1 = std::integral_constant<int, 1>;

        src.load_k(0, Kb0);
        src.load_v(0, Vb0);
        if (nb > 1) {
            src.load_k(1, Kb1);
            publish<2 * NI>();  // Q and K_0 have landed
        } else {
            publish<NI>();
        }
        if (live) {
            constexpr int AB = NS - (PF < NS ? PF : NS), BB = NP - (PF < NP ? PF : NP);  // steps of the two barriers
            constexpr int FK = NS - AB, FV = NP - BB;                                    // operands ahead
            Vec16 ka[FK], va[FV];
            auto iter = [&](int j, auto par, f16v_t (&sc)[2], f16v_t (&sn)[2]) {
                constexpr int P = decltype(par)::value;
                using Pn = std::integral_constant<int, P ^ 1>;
                __builtin_amdgcn_s_setprio(P);
                hide();
                auto dma = src.dma(j);
                fence();
                zero(sn);
#pragma unroll
                for (int i = 0; i < NS; ++i) {
                    if (i == AB) {
                        publish<2 * NI>();
                        if constexpr (Src::kEveryBlock || SCAN) src.template clean<SCAN>(j, Vb0 + P * BLK, oacc);
                    }
                    sn[i & 1] = mma32<T>(ka[i % FK], qf[i >> 1], sn[i & 1]);
                    if (i + FK < NS) ka[i % FK] = fetch_k(Pn{}, i + FK);
                    if (i >= AB && i - AB < FV) va[i - AB] = fetch_v(par, i - AB);
#pragma unroll
                    for (int n = 0; n < NI; ++n)
                        if ((AB > 1 ? 1 + n * (AB - 1) / NI : 0) == i) dma.v(P ^ 1, n);
                    weights_at(sc, i);
                    fence();
                }
                src.mask(j + 1, sn);
                float mb = -INFINITY;
#pragma unroll
                for (int i = 0; i < NP; ++i) {
                    if (i == BB) publish<2 * NI>();
                    oacc[i % DT] = mma32<T>(va[i % FV], pf[i / DT], oacc[i % DT]);
                    if (i + FV < NP)
                        va[i % FV] = fetch_v(par, i + FV);
                    else if (i - BB < FK)
                        ka[i - BB] = fetch_k(par, i - BB);
#pragma unroll
                    for (int n = 0; n < NI; ++n)
                        if ((BB > 1 ? 1 + n * (BB - 1) / NI : 0) == i) dma.k(P ^ 1, n);
                    weights_at(sc, NS + i);
#pragma unroll
                    for (int e = 0; e < 16; ++e)
                        if (2 * DT + e * 2 * DT / 16 == i)
                            mb = fmaxf(fmaxf(mb, sn[e >> 3][2 * (e & 7)]), sn[e >> 3][2 * (e & 7) + 1]);
                    fence();
                }
                l_run += ps0 + ps1;
                move_ref(mb);
                fence();
            };
            f16v_t sA[2], sB[2];
            zero(sA);
#pragma unroll
            for (int i = 0; i < FK; ++i) ka[i] = fetch_k(B0{}, i);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                sA[i & 1] = mma32<T>(ka[i % FK], qf[i >> 1], sA[i & 1]);
                if (i + FK < NS) ka[i % FK] = fetch_k(B0{}, i + FK);
            }
            src.mask(0, sA);
            move_ref(block_max(sA));
            publish<0>();  // K_0 has been read; V_0 and K_1 have landed
            if (nb > 2) src.load_k(2, Kb0);
#pragma unroll
            for (int i = 0; i < FK; ++i) ka[i] = fetch_k(B1{}, i);
            int j = 0;
            for (; j + 2 < nb; j += 2) {
                iter(j, B0{}, sA, sB);
                iter(j + 1, B1{}, sB, sA);
            }
            if (j + 1 < nb) {
                iter(j, B0{}, sA, sB);
                sA[0] = sB[0];
                sA[1] = sB[1];
            }
            // ---- the last block, in one copy for both buffers (a copy for each
            // took D = 128 past 256 VGPRs) ----
            const uint32_t vbuf = 2 * (2 + ((nb - 1) & 1)) * BLK;
            publish<0>();
            src.template clean<SCAN>(nb - 1, Vb0 + ((nb - 1) & 1) * BLK, oacc);
#pragma unroll
            for (int i = 0; i < FV; ++i) va[i] = fetch_v_at(vbuf, i);
            // its weights, those of each 16-key step beside the products of the one before
#pragma unroll
            for (int i = -DT; i < NP; ++i) {
#pragma unroll
                for (int n = 0; n < 32; ++n) {
                    if (n * DT / 8 != i + DT) continue;
                    stage(sA, n, 0);
                    stage(sA, n, 1);
                    stage(sA, n, 2);
                }
                if (i < 0) continue;
                oacc[i % DT] = mma32<T>(va[i % FV], pf[i / DT], oacc[i % DT]);
                if (i + FV < NP) va[i % FV] = fetch_v_at(vbuf, i + FV);
            }
            __builtin_amdgcn_s_setprio(0);
            l_run += ps0 + ps1;
        } else {
            // a wave past the tile's rows stages its part of the blocks
            publish<0>();
            if (nb > 2) src.load_k(2, Kb0);
            for (int j = 0; j + 1 < nb; ++j) {
                auto dma = src.dma(j);
                const int buf = (j & 1) ^ 1;
#pragma unroll
                for (int n = 0; n < NI; ++n) dma.v(buf, n);
                publish<2 * NI>();
                if constexpr (Src::kEveryBlock || SCAN) src.template clean<SCAN>(j, Vb0 + (j & 1) * BLK);
#pragma unroll
                for (int n = 0; n < NI; ++n) dma.k(buf, n);
                publish<2 * NI>();
            }
            publish<0>();
            src.template clean<SCAN>(nb - 1, Vb0 + ((nb - 1) & 1) * BLK);
        }
    }

    // Stores the numerator as the fp32 row at acc.
    static __device__ __forceinline__ void store_state(const f16v_t (&oacc)[DT], float* acc) {
        acc += 4 * ((threadIdx.x >> 5) & 1);
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int j = 0; j < 4; ++j)
                *reinterpret_cast<float4*>(acc + 32 * dt + 8 * j) = make_float4(
                    oacc[dt][4 * j], oacc[dt][4 * j + 1], oacc[dt][4 * j + 2], oacc[dt][4 * j + 3]);
    }

    // Stores oacc * inv as the row at orow: a lane pair (l, l + 32) holds dims
    // 8 j + 0 .. 3 and 8 j + 4 .. 7 of its query; a half-wave exchange of
    // neighbouring groups gives each lane 16 contiguous bytes.
    static __device__ __forceinline__ void store_row(const f16v_t (&oacc)[DT], float inv, uint16_t* orow, bool valid) {
        const int hl = (threadIdx.x >> 5) & 1;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
            for (int j = 0; j < 4; j += 2) {
                uint32_t w[2][2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    float x[4];
#pragma unroll
                    for (int i = 0; i < 4; ++i) x[i] = in_range<T>(oacc[dt][4 * (j + e) + i] * inv);
                    w[e][0] = MfmaOps<T>::pack2(x[0], x[1]);
                    w[e][1] = MfmaOps<T>::pack2(x[2], x[3]);
                }
                auto a = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
                auto b = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
                // lanes 0-31: group j (own half, other half), lanes 32-63: group j + 1
                if (valid)
                    st16(orow + 32 * dt + 8 * (j + hl),
                         Vec16{{(uint32_t)a[0], (uint32_t)b[0], (uint32_t)a[1], (uint32_t)b[1]}});
            }
        }
    }
};

}  // namespace qattn
