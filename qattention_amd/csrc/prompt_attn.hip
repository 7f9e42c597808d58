// prompt_attn.hip -- causal attention of packed prompts, with LSE.
//
// For token i of a sequence and q head h (kv head h / group):
//   o = sum_{j <= i} softmax_j(scale q_i.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// in one pass over the keys with a running maximum m and sum l.
//
// Work unit: (sequence, kv head, tile of 128 rows); a row is a (token, q head)
// pair of the kv head's group, tokens outermost, so a tile spans 128 / group
// tokens and a K/V block staged in LDS serves every q head that reads it.
// Units with the most keys come first (last tiles of every sequence), sequences
// and heads innermost: with a multiple of 8 of those, every tile of one
// (sequence, kv head) runs on one XCD and shares its L2.
//
// The key loop is that of the prefix kernel (prefix_attn.hip): 4 waves own 32
// rows each as the N dimension of v_mfma_f32_32x32x16 products, S^T = K Q^T,
// O^T += V^T P^T over 64-key blocks, LDS-DMA double buffers, every step in its
// place.  Here it ends at the tile's last token, and the blocks that reach
// past a wave's first token are masked by row.
//
// Rows whose result is not finite are computed once more, row by row from
// the definition (redo_row): the product of a block's masked weights (0) and
// an infinity or NaN in the V row of a later token is NaN, and only the keys up
// to the row's own may show.
#include <algorithm>

#include "kv_tiles.h"
#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kPromptThreads = 256;
constexpr int kBN = 64;   // keys per block
constexpr int kBM = 128;  // rows per workgroup

struct PromptParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* o;
    float* lse;
    const int32_t* cu;
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h, so_t, so_h, sl_t, sl_h;
    int64_t total_tokens;
    int32_t B, Hq, Hkv, group, max_seqlen, qtiles, pairs;
    Divider gdiv, pairdiv, hkvdiv;  // group, pairs (B * Hkv), Hkv
    float scale_log2;
};

// One row from the definition, by one wave: keys 0 .. tok of the sequence
// whose first K/V row (of this kv head) is k / v; q, o: this row's.
template <typename T, int D>
__device__ void redo_row(const PromptParams& p, const uint16_t* q, const uint16_t* k, const uint16_t* v, int tok,
                         uint16_t* o, float* lse, int lane) {
    constexpr int E = D > 64 ? D / 64 : 1;  // dims of a lane (D = 32: lanes 0 .. 31)
    const bool live = lane * E < D;
    auto score = [&](int j) {
        float s = 0.f;
        for (int c = 0; c < D; c += 8) s += dot8<T>(ld16(q + c), ld16(k + (int64_t)j * p.sk_t + c));
        return s * p.scale_log2;
    };
    float m = -INFINITY;
    bool nan = false;
    for (int j = lane; j <= tok; j += 64) {
        const float s = score(j);
        nan |= s != s;
        m = fmaxf(m, s);
    }
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    if (__any(nan)) m = __builtin_nanf("");
    float l = 0.f, acc[E] = {};
    for (int j0 = 0; j0 <= tok; j0 += 64) {
        const float w = j0 + lane <= tok ? fast_exp2(score(j0 + lane) - m) : 0.f;
        l += w;
        for (int i = 0; i < 64 && j0 + i <= tok; ++i) {
            const float wi = __shfl(w, i);
            const uint16_t* vr = v + (int64_t)(j0 + i) * p.sv_t + (live ? lane * E : 0);
#pragma unroll
            for (int e = 0; e < E; ++e) {
                const uint32_t bits = vr[e];
                acc[e] = __builtin_fmaf(wi, MfmaOps<T>::lo(bits), acc[e]);
            }
        }
    }
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    if (live) {
#pragma unroll
        for (int e = 0; e < E; ++e) o[lane * E + e] = (uint16_t)MfmaOps<T>::pack2(acc[e] / l, 0.f);
    }
    if (lse && lane == 0) *lse = (m + fast_log2(l)) * kLn2;
}

template <typename T, int D>
__global__ __launch_bounds__(kPromptThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void prompt_attn_kernel(
    PromptParams p) {
    constexpr int KS = D / 16;      // k-steps of S^T over the head dim
    constexpr int DT = D / 32;      // 32-row d-tiles of O^T
    constexpr int DV = D / 8;       // 16-byte chunks per key row
    constexpr int BLK = kBN * D;    // elements of one K or V block
    constexpr int NI = D / 32;      // 1 KB LDS loads per thread per K (or V) block
    constexpr int RPI = 512 / D;    // key rows per 1 KB load
    static_assert(NI * 4 * 512 == BLK, "a block is 4 waves x NI loads of 1 KB");
    // Double buffers of the K and V blocks: K 0, K 1, V 0, V 1.
    __shared__ __attribute__((aligned(1024))) uint16_t smem[4 * BLK];
    uint16_t *const Kb0 = smem, *const Kb1 = smem + BLK, *const Vb0 = smem + 2 * BLK;

    const int r0 = divide(blockIdx.x, p.pairdiv);
    const int pair = blockIdx.x - r0 * p.pairs;
    const int qt = p.qtiles - 1 - r0;
    const int seq = divide(pair, p.hkvdiv);
    const int kvh = pair - seq * p.Hkv;
    const int32_t s0 = p.cu[seq], s1 = p.cu[seq + 1];
    if (s0 < 0 || s1 < s0 || (int64_t)s1 > p.total_tokens) return;
    int32_t n = s1 - s0;
    if (n > p.max_seqlen) n = p.max_seqlen;
    const int g = p.group;
    const int rows = n * g;
    if (qt * kBM >= rows) return;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int q32 = lane & 31, hl = lane >> 5;

    // this lane's query row (B operand column, output column)
    auto query_of = [&](int& tok, int& qh) {
        const int rr = qt * kBM + wave * 32 + q32;
        tok = divide(rr, p.gdiv);
        qh = kvh * g + (rr - tok * g);
        return rr < rows;
    };
    // Q^T operand of step s: dims 16 s + 8 hl .. + 7 of the lane's query
    Vec16 qf[KS];
    {
        int tok, qh;
        const bool valid = query_of(tok, qh);
        const uint16_t* qp = p.q + ((int64_t)s0 + tok) * p.sq_t + (int64_t)qh * p.sq_h + 8 * hl;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = Vec16{{0u, 0u, 0u, 0u}};
            if (valid) qf[s] = ld16(qp + 16 * s);
        }
    }

    constexpr int k_lo = 0;
    const int k_hi = divide(min(qt * kBM + kBM, rows) - 1, p.gdiv) + 1;  // past the tile's last token
    const int nb = (k_hi + kBN - 1) / kBN;
    const char* kbase = (const char*)(p.k + (int64_t)s0 * p.sk_t + (int64_t)kvh * p.sk_h);
    const char* vbase = (const char*)(p.v + (int64_t)s0 * p.sv_t + (int64_t)kvh * p.sv_h);
    const int64_t kst = 2 * p.sk_t, vst = 2 * p.sv_t;  // bytes between keys
    // first tokens of the wave and of the lane: keys past them are masked
    const int tok_w = divide(qt * kBM + wave * 32, p.gdiv);
    const int tok_l = divide(qt * kBM + wave * 32 + q32, p.gdiv);

    float m_run = -INFINITY, l_run = 0.f;  // l_run: this lane's half of the keys
    f16v_t oacc[DT];
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) oacc[dt][r] = 0.f;

    // ---- K/V blocks go straight from global memory to LDS (global_load_lds,
    // 16 bytes per lane, lane i of a load writes bytes [16 i, 16 i + 16) of its
    // 1 KB): load n of wave w covers key rows (w NI + n) RPI .. + RPI - 1, and
    // each lane fetches the chunk that the swizzle puts at its position.  The
    // byte offset of a lane's load n within a block is its row's offset plus
    // colb ^ 16 swz(n RPI) (the swizzle is linear over xor and row n's bits
    // are disjoint from the lane's), 32-bit (the host checks that 64 key rows
    // span less than 4 GB), added to the block's uniform base. ----
    const uint32_t colb = 16 * ((lane % DV) ^ kv_swz32(wave * NI * RPI + lane / DV, DV));
    const uint32_t krow = (uint32_t)(wave * NI * RPI + lane / DV) * (uint32_t)kst;
    const uint32_t vrow = (uint32_t)(wave * NI * RPI + lane / DV) * (uint32_t)vst;
    // First row of block i.  The last block of a range that is no multiple of
    // 64 keys starts early (its first keys, also in the block before, are
    // masked and their V rows cleared), and a block past the end repeats it:
    // every load of the key loop is of 64 whole rows, without a bound to clamp
    // to.
    auto block_row = [&](int i) { return min(k_lo + i * kBN, k_hi - kBN); };
    // a whole block at once, before the loop; block 0 may be the only one and
    // shorter than 64 rows: rows past the last repeat it
    auto issue = [&](const char* base, int64_t st, uint32_t row, int i, uint16_t* buf) {
        const int kb = i == 0 ? k_lo : block_row(i);
        const uint32_t last = (uint32_t)min(k_hi - 1 - kb, kBN - 1) * (uint32_t)st;
        const char* gb = base + (int64_t)kb * st;
#pragma unroll
        for (int n = 0; n < NI; ++n)
            lds_dma16((colb ^ (16 * kv_swz32(n * RPI, DV))) + min(row + (uint32_t)(n * RPI) * (uint32_t)st, last), gb,
                      buf + (wave * NI + n) * 512);
    };

    // Operand read addresses (elements).  K (A of S^T, step s, key tile t):
    // row 32 t + q32, chunk 2 s + hl: (kaddr0 ^ 16 s) + 32 D t (the swizzle
    // flips only chunk bits, which the row base leaves clear).  V^T (A of
    // O^T, 16-key step th = 2t + h, d-tile dt): two ds_read_b64_tr_b16, X for
    // keys 16 th + 4 hl + 0..3 and Y for + 8; within each 16-lane group lane
    // j points at row key0 + j / 4, dims 32 dt + 16 ((lane >> 4) & 1) +
    // 4 (j % 4) .. + 3, and receives keys key0 + 0..3 at dim 32 dt + q32.
    const int kaddr0 = q32 * D + 8 * (hl ^ kv_swz32(q32, DV));
    int vx0, vy0;
    {
        const int rx = 4 * hl + ((lane & 15) >> 2), ry = rx + 8;
        const int cx = 2 * ((lane >> 4) & 1) + ((lane & 3) >> 1);
        vx0 = rx * D + 8 * (cx ^ kv_swz32(rx, DV)) + 4 * (lane & 1);
        vy0 = ry * D + 8 * (cx ^ kv_swz32(ry, DV)) + 4 * (lane & 1);
    }
    // LDS byte addresses of this lane's operand reads in K 0 / V 0; buffer,
    // key tile and 16-key step are immediate offsets.  hide() keeps the
    // compiler from holding one register per address and buffer, which spills.
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

    // Online softmax (the lane's query; element r of S tile t is key 32 t +
    // 8 (r / 4) + 4 hl + r % 4 of the block): raw-score maximum, p = exp2(s c -
    // m c), the reference moved only past 2^kLazy for fp16 and on every new
    // maximum for bf16, whose 8 mantissa bits round all weights but 1 (as in the
    // prefix kernel).
    const float csc = p.scale_log2;
    constexpr float kLazy = T::kCode == QATTN_DTYPE_BF16 ? 0.f : 8.f;
    // m_run csc; the sum of one block's weights, in two parts (summed by block,
    // then over the blocks: one running sum of every weight doubled the LSE's
    // error, 2.0e-6 -> 5.5e-6 over 200000 keys)
    float mc = 0.f, ps0 = 0.f, ps1 = 0.f;
    auto move_ref = [&](float mb) {
        mb = xor32_max(mb);
        const bool move = (mb - m_run) * csc > kLazy;  // always true on the first block
        if (__builtin_expect(__any(move), 0)) {
            const float m_new = move ? mb : m_run;
            const float alpha = move ? fast_exp2((m_run - m_new) * csc) : 1.f;  // m_run = -inf: 0
#pragma unroll
            for (int dt = 0; dt < DT; ++dt) oacc[dt] *= alpha;
            l_run *= alpha;
            m_run = m_new;
        }
        mc = m_run * csc;
    };
    // -inf for the keys of a block (first row kb) below lo (they belong to the
    // block before) and past the lane's token
    auto mask_block = [&](int kb, int lo, f16v_t (&s)[2]) {
        if (__builtin_expect(kb < lo || kb + kBN - 1 > tok_w, 0)) {
            uint32_t k0 = (uint32_t)(kb - lo + 4 * hl);
            asm volatile("" : "+v"(k0));  // (32 key numbers held across the loop would spill)
            const uint32_t keys = (uint32_t)max(tok_l + 1 - lo, 0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (k0 + 32 * t + 8 * (r >> 2) + (r & 3) >= keys) s[t][r] = -INFINITY;  // (below lo: wrapped)
                }
        }
    };
    // One block's 32 weights per lane, element n = 8 th + e of 16-key step th,
    // in three stages: exponent (0), exponential (1), sum and packing (2).
    // Stage q of element n runs at step n NT / 32 + q of an iteration's
    // NS + NP products, so no instruction waits for the one before it and
    // step th's weights are packed before its first product.
    constexpr int NT = NS + 3 * DT - 2;
    Vec16 pf[4];
    auto stage = [&](f16v_t (&s)[2], int n, int q) {
        float x = s[n >> 4][n & 15];
        if (q == 0) x = __builtin_fmaf(x, csc, -mc);
        if (q == 1) x = fast_exp2(x);
        s[n >> 4][n & 15] = x;
        if (q == 2) {
            if (n & 1) {
                ps1 = n == 1 ? x : ps1 + x;
                pf[n >> 3].w[(n & 7) >> 1] = MfmaOps<T>::pack2(s[n >> 4][(n & 15) - 1], x);
            } else {
                ps0 = n == 0 ? x : ps0 + x;
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
    // Each step of the loop below is kept in its place: the compiler's own
    // order put the operand reads next to their products and all
    // exponentials into the PV half.
    auto fence = [] { __builtin_amdgcn_sched_barrier(0); };
    // All but the N newest DMA loads and every LDS read of this wave are done,
    // then the workgroup's barrier: what was loaded may be read, what was read
    // may be overwritten.
    auto publish = [](auto n) {
        constexpr int N = decltype(n)::value;
        __builtin_amdgcn_s_waitcnt((N & 15) | ((N >> 4) << 14) | (7 << 4));  // vmcnt(N) lgkmcnt(0)
        asm volatile("s_barrier" ::: "memory");
    };
    using W0 = std::integral_constant<int, 0>;
    using W1 = std::integral_constant<int, NI>;
    using W2 = std::integral_constant<int, 2 * NI>;
    using B0 = std::integral_constant<int, 0>;
    using B1 = std::integral_constant<int, 1>;
    // the DMA loads of an iteration, one at a time: K_{j+3} and V_{j+1}, both
    // into the buffers of parity B
    struct Dma {
        uint32_t col, kr, vr, ld;
        const char *gk, *gv;
        int64_t ks, vs;
        __device__ __forceinline__ void load(uint32_t off, const char*& base, int64_t step, uint32_t lds) {
            asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(off), "s"(base), "{m0}"(lds) : "memory");
            base += step;
        }
        __device__ __forceinline__ void k(int buf, int n) {
            load((col ^ (16 * kv_swz32(n * RPI, DV))) + kr, gk, ks, ld + 2 * buf * BLK + n * 1024);
        }
        __device__ __forceinline__ void v(int buf, int n) {
            load((col ^ (16 * kv_swz32(n * RPI, DV))) + vr, gv, vs, ld + 2 * (2 + buf) * BLK + n * 1024);
        }
    };
    auto dma_of = [&](int j) {
        Dma d{colb, krow, vrow, lds0 + wave * (NI * 1024), kbase + (int64_t)block_row(j + 3) * kst,
              vbase + (int64_t)block_row(j + 1) * vst, RPI * kst, RPI * vst};
        asm volatile("" : "+v"(d.col), "+v"(d.kr), "+v"(d.vr), "+s"(d.ld));  // (as hide())
        return d;
    };

    // ---- pipeline over the tile's blocks, as in the prefix kernel ----
    // The keys that the last block shares with the one before have weight 0
    // there, and 0 times an infinity is NaN: clear their V rows (every thread
    // of the workgroup, once the block has landed).
    auto drop_shared = [&](int buf) {
        const int shared = nb > 1 ? k_lo + (nb - 1) * kBN - block_row(nb - 1) : 0;
        if (shared > 0) {
            for (int i = tid; i < shared * DV; i += kPromptThreads)
                st16(Vb0 + buf * BLK + 8 * i, Vec16{{0u, 0u, 0u, 0u}});
            publish(W0{});
        }
    };
    issue(kbase, kst, krow, 0, Kb0);
    issue(vbase, vst, vrow, 0, Vb0);
    if (nb > 1) {
        issue(kbase, kst, krow, 1, Kb1);
        publish(W2{});  // Q and K_0 have landed
    } else {
        publish(W1{});
    }
    if (qt * kBM + wave * 32 < rows) {
        constexpr int AB = NS - (PF < NS ? PF : NS), BB = NP - (PF < NP ? PF : NP);  // steps of the two barriers
        Vec16 ka[NS - AB], va[NP - BB];
        constexpr int FK = NS - AB, FV = NP - BB;  // operands ahead
        auto iter = [&](int j, auto par, f16v_t (&sc)[2], f16v_t (&sn)[2]) {
            constexpr int P = decltype(par)::value;
            using Pn = std::integral_constant<int, P ^ 1>;
            __builtin_amdgcn_s_setprio(P);
            hide();
            Dma dma = dma_of(j);
            fence();
            zero(sn);
#pragma unroll
            for (int i = 0; i < NS; ++i) {
                if (i == AB) publish(W2{});
                sn[i & 1] = mma32<T>(ka[i % FK], qf[i >> 1], sn[i & 1]);
                if (i + FK < NS) ka[i % FK] = fetch_k(Pn{}, i + FK);
                if (i >= AB && i - AB < FV) va[i - AB] = fetch_v(par, i - AB);
#pragma unroll
                for (int n = 0; n < NI; ++n)
                    if ((AB > 1 ? 1 + n * (AB - 1) / NI : 0) == i) dma.v(P ^ 1, n);
                weights_at(sc, i);
                fence();
            }
            mask_block(block_row(j + 1), k_lo + (j + 1) * kBN, sn);
            float mb = -INFINITY;
#pragma unroll
            for (int i = 0; i < NP; ++i) {
                if (i == BB) publish(W2{});
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
        mask_block(k_lo, k_lo, sA);
        {
            float mb = -INFINITY;
#pragma unroll
            for (int e = 0; e < 16; ++e) mb = fmaxf(fmaxf(mb, sA[e >> 3][2 * (e & 7)]), sA[e >> 3][2 * (e & 7) + 1]);
            move_ref(mb);
        }
        publish(W0{});  // K_0 has been read; V_0 and K_1 have landed
        if (nb > 2) issue(kbase, kst, krow, 2, Kb0);
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
        publish(W0{});
        drop_shared((nb - 1) & 1);
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
        // a wave past the tile's rows only stages its part of the blocks (672
        // rows per kv head leave 3 of 24 waves without any: 408 -> 397 us)
        publish(W0{});
        if (nb > 2) issue(kbase, kst, krow, 2, Kb0);
        for (int j = 0; j + 1 < nb; ++j) {
            Dma dma = dma_of(j);
            const int buf = (j & 1) ^ 1;
#pragma unroll
            for (int n = 0; n < NI; ++n) dma.v(buf, n);
            publish(W2{});
#pragma unroll
            for (int n = 0; n < NI; ++n) dma.k(buf, n);
            publish(W2{});
        }
        publish(W0{});
        drop_shared((nb - 1) & 1);
    }

    // ---- normalise and store: a lane pair (l, l + 32) holds dims 8 j + 0 .. 3
    // and 8 j + 4 .. 7 of its query; a half-wave exchange of neighbouring
    // groups gives each lane 16 contiguous bytes ----
    const float l_tot = xor32_sum(l_run);  // both halves of the query's keys
    const float inv = 1.f / l_tot;
    int tok, qh;
    const bool valid = query_of(tok, qh);
    uint16_t* const orow = p.o + ((int64_t)s0 + tok) * p.so_t + (int64_t)qh * p.so_h;
    float* const lrow = p.lse ? p.lse + ((int64_t)s0 + tok) * p.sl_t + (int64_t)qh * p.sl_h : nullptr;
    const float lse = (m_run * p.scale_log2 + fast_log2(l_tot)) * kLn2;
    float odd = lse - lse;  // 0, or NaN if any result is not finite
#pragma unroll
    for (int dt = 0; dt < DT; ++dt) {
#pragma unroll
        for (int j = 0; j < 4; j += 2) {
            uint32_t w[2][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                float x[4];
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    x[i] = oacc[dt][4 * (j + e) + i] * inv;
                    odd += x[i] - x[i];
                }
                w[e][0] = MfmaOps<T>::pack2(x[0], x[1]);
                w[e][1] = MfmaOps<T>::pack2(x[2], x[3]);
            }
            auto a = __builtin_amdgcn_permlane32_swap(w[0][0], w[1][0], false, false);
            auto b = __builtin_amdgcn_permlane32_swap(w[0][1], w[1][1], false, false);
            // lanes 0-31: group j (own half, other half), lanes 32-63: group j + 1
            if (valid) st16(orow + 32 * dt + 8 * (j + hl), Vec16{{(uint32_t)a[0], (uint32_t)b[0], (uint32_t)a[1], (uint32_t)b[1]}});
        }
    }
    if (valid && lrow && hl == 0) *lrow = lse;
    uint64_t again = __ballot(valid && odd != 0.f);
    if (__builtin_expect(again != 0, 0)) {
        again |= again >> 32;
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // the rows' first stores come before the second
        for (uint32_t todo = (uint32_t)again; todo; todo &= todo - 1) {
            const int r = __builtin_ctz(todo);
            const int rr = qt * kBM + wave * 32 + r;
            const int t = divide(rr, p.gdiv);
            const int h = kvh * g + (rr - t * g);
            const int64_t row = (int64_t)s0 + t;
            redo_row<T, D>(p, p.q + row * p.sq_t + h * p.sq_h, (const uint16_t*)kbase, (const uint16_t*)vbase, t,
                           p.o + row * p.so_t + h * p.so_h, p.lse ? p.lse + row * p.sl_t + h * p.sl_h : nullptr, lane);
        }
    }
}

template <typename T, int D>
static int launch_prompt(const PromptParams& p, int64_t blocks, hipStream_t st) {
    hipLaunchKernelGGL((prompt_attn_kernel<T, D>), dim3((uint32_t)blocks), dim3(kPromptThreads), 0, st, p);
    return launch_status("prompt_attn_kernel");
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int qattn_prompt_fwd(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                     const void* v, const int64_t v_stride[3], void* o, const int64_t o_stride[3], float* lse,
                     const int64_t lse_stride[2], const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen,
                     int64_t total_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                     int32_t dtype, void* stream) {
    clear_error();
    const int rc = check_common(dtype, head_dim, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, 0);
    if (rc) return rc;
    if (!(scale > 0.f) || !(scale < INFINITY)) {
        set_error("scale must be positive and finite");
        return QATTN_ERR_ARG;
    }
    if (batch == 0 || max_seqlen == 0 || total_tokens == 0) return QATTN_OK;  // nothing to compute
    if (!q || !k || !v || !o || !q_stride || !k_stride || !v_stride || !o_stride || !cu_seqlens ||
        (lse && !lse_stride)) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    if (!row_aligned(q, q_stride, 2) || !row_aligned(o, o_stride, 2)) {
        set_error("q/o rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    if (!row_aligned(k, k_stride, 2) || !row_aligned(v, v_stride, 2)) {
        set_error("k/v rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    if (k_stride[0] < 0 || v_stride[0] < 0 || k_stride[0] >= (1 << 25) || v_stride[0] >= (1 << 25)) {
        set_error("k/v token strides must be in [0, 2^25) elements");  // 64 rows: 32-bit byte offsets
        return QATTN_ERR_LAYOUT;
    }
    PromptParams p{};
    p.q = (const uint16_t*)q, p.k = (const uint16_t*)k, p.v = (const uint16_t*)v, p.o = (uint16_t*)o;
    p.lse = lse;
    p.cu = cu_seqlens;
    p.sq_t = q_stride[0], p.sq_h = q_stride[1];
    p.sk_t = k_stride[0], p.sk_h = k_stride[1];
    p.sv_t = v_stride[0], p.sv_h = v_stride[1];
    p.so_t = o_stride[0], p.so_h = o_stride[1];
    if (lse) p.sl_t = lse_stride[0], p.sl_h = lse_stride[1];
    p.total_tokens = total_tokens;
    p.B = batch, p.Hq = num_q_heads, p.Hkv = num_kv_heads, p.group = num_q_heads / num_kv_heads;
    p.max_seqlen = (int32_t)std::min<int64_t>(max_seqlen, total_tokens);
    if ((int64_t)p.max_seqlen * p.group > INT32_MAX / 2 || (int64_t)batch * num_kv_heads > INT32_MAX) {
        set_error("sizes too large: max_seqlen=%d group=%d batch=%d num_kv_heads=%d", p.max_seqlen, p.group, batch,
                  num_kv_heads);
        return QATTN_ERR_ARG;
    }
    p.pairs = batch * num_kv_heads;
    p.qtiles = (p.max_seqlen * p.group + kBM - 1) / kBM;
    const int64_t blocks = (int64_t)p.qtiles * p.pairs;
    if (blocks > INT32_MAX) {
        set_error("grid too large (%lld blocks)", (long long)blocks);
        return QATTN_ERR_ARG;
    }
    p.gdiv = make_divider(p.group);
    p.pairdiv = make_divider(p.pairs);
    p.hkvdiv = make_divider(num_kv_heads);
    p.scale_log2 = scale * kLog2e;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == QATTN_DTYPE_F16)
        return head_dim == 32   ? launch_prompt<F16, 32>(p, blocks, st)
               : head_dim == 64 ? launch_prompt<F16, 64>(p, blocks, st)
                                : launch_prompt<F16, 128>(p, blocks, st);
    return head_dim == 32   ? launch_prompt<BF16, 32>(p, blocks, st)
           : head_dim == 64 ? launch_prompt<BF16, 64>(p, blocks, st)
                            : launch_prompt<BF16, 128>(p, blocks, st);
}

}  // extern "C"
