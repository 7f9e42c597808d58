// quant_attn.hip -- attention of query tokens over their sequence's context in a
// paged K/V cache that is held in 4 or 8 bits (quant_format.h), with LSE.
//
//   o = sum_j softmax_j(scale q.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// over keys 0 .. context - 1, where k_j and v_j are exactly the values that the
// cache's elements and scales stand for: they are widened to the queries' type on
// their way into the products (exact, quant_format.h), and everything behind that
// is as over a 16-bit cache (paged_attn.hip): rows (token, q head), the work dealt
// in runs and joined without atomics (paged_work.h), a running maximum and sum,
// weights rounded once to the queries' type for their product.
//
// Two kernels by the longest sequence's rows:
//   up to 32 (quant_attn_kernel): bound by reading the cache;
//   more (quant_wide_kernel): tiles of 128 rows share K/V blocks of 64 keys in
//   LDS (dense_tiles.h), bound by the matrix cores.
#include "paged_work.h"
#include "quant_format.h"

namespace qattn {

struct QuantParams : PagedParams {
    const uint8_t *ks, *vs;              // scales; K and V share all strides
    int64_t ss_head;                     // bytes
    // of a page and a slot, in 16-byte units of the elements and in rows of the scales
    // (a row's offset, kv head aside, is 32 bits wide)
    uint32_t row_page, row_slot, scale_page, scale_slot;
};

typedef uint32_t w2_t __attribute__((ext_vector_type(2)));
typedef uint32_t w4_t __attribute__((ext_vector_type(4)));

// N words at p (aligned to their size, up to 16 bytes).  ONCE: past the caches.
template <bool ONCE = false, int N>
__device__ __forceinline__ void ld_words(uint32_t (&w)[N], const char* p) {
    auto ld = [](auto* at) { return ONCE ? __builtin_nontemporal_load(at) : *at; };
    if constexpr (N == 1) {
        w[0] = ld(reinterpret_cast<const uint32_t*>(p));
    } else if constexpr (N == 2) {
        const w2_t x = ld(reinterpret_cast<const w2_t*>(p));
        w[0] = x[0], w[1] = x[1];
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const w4_t x = ld(reinterpret_cast<const w4_t*>(p + 4 * i));
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = x[j];
        }
    }
}

__device__ __forceinline__ uint32_t lds_at(const void* p) {
    return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)p;
}

// N scales at p, one byte each (aligned to N), the first in the low byte.
template <int N>
__device__ __forceinline__ uint32_t ld_scales(const char* p) {
    if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) return *reinterpret_cast<const uint16_t*>(p);
    else return *reinterpret_cast<const uint8_t*>(p);
}

// Word i of head h's operand from the loads x of a key tile: lanes g COLS .. of every
// 16 from load (g - h) % NH, whose lanes h COLS .. hold the head's words, turned by the
// groups in between.  (DPP: row_ror moves lane i to i + n; a bank is four lanes.)
template <int NH, int N>
__device__ __forceinline__ uint32_t turn_in(const uint32_t (&x)[NH][N], int i, int h) {
    static_assert(NH == 1 || NH == 2 || NH == 4, "groups of lanes");
    int w = (int)x[0][i];
    if constexpr (NH == 2) {
        w = h ? __builtin_amdgcn_update_dpp(w, (int)x[1][i], 0x128, 0xF, 0x3, false)
              : __builtin_amdgcn_update_dpp(w, (int)x[1][i], 0x128, 0xF, 0xC, false);
    } else if constexpr (NH == 4) {
        // load j into group (h + j) % 4
#define QATTN_TURN(J)                                                                                   \
    w = h == 0   ? __builtin_amdgcn_update_dpp(w, (int)x[J][i], 0x120 + 4 * J, 0xF, 1 << (J) % 4, false)     \
        : h == 1 ? __builtin_amdgcn_update_dpp(w, (int)x[J][i], 0x120 + 4 * J, 0xF, 1 << (1 + J) % 4, false) \
        : h == 2 ? __builtin_amdgcn_update_dpp(w, (int)x[J][i], 0x120 + 4 * J, 0xF, 1 << (2 + J) % 4, false) \
                 : __builtin_amdgcn_update_dpp(w, (int)x[J][i], 0x120 + 4 * J, 0xF, 1 << (3 + J) % 4, false)
        QATTN_TURN(1);
        QATTN_TURN(2);
        QATTN_TURN(3);
#undef QATTN_TURN
    }
    return (uint32_t)w;
}

// ---------------------------------------------------------------------------
// Few rows (16 QB per tile).  The waves' split, the products and the softmax are
// the 16-bit kernel's: per step a wave forms S^T = K Q^T and O^T += V^T P^T for 32
// keys of its own, and nothing is shared between the waves but a head's last join.
// What differs is the way in:
//   K  A lane's operand words are a quarter of a key row, contiguous: lane (l16, lq)
//      takes dims D/4 lq .. of key l16, k-step c the 8 from D/4 lq + 8 c on (Q^T is
//      read in that order, which is free), so a quarter has one scale.
//   V  A lane widens 16 (or 8) bytes of a row and stores them to the head's LDS block
//      as 16-byte chunks; chunk i of lane part ch lies at place i LPR + ch, so that
//      the lanes of a row write side by side.  O's columns come out in that order and
//      are put back where they are stored.
//   scales  A lane loads a word of one token's (K's and V's); lane exchanges hand the
//      words out.
// and the number of heads: a wave takes NH kv heads whose rows lie side by side in a
// token, 128 bytes where they reach, and each load takes whole tokens: a 64-byte row by
// itself is half a line, fetched again for the other half (64 x 5300-16000 tokens, 4
// bits, 8 heads of 128, 731 MB: 259 us with one head per wave, 154 with two, 143 of them
// the bare loads; with whole lines per load 150, the loads past the caches 142, columns
// chosen and not zeroed 131, where the bare loads take 121: 5.6 TB/s).
//   columns  Where a head's rows fit, each head has COLS = 16 / NH of the 16 columns of
//      one S^T, put together from the heads' products with all columns of Q^T, so that the
//      softmax is paid once for NH heads; P^T as it is serves every head's product with V
//      (a head's columns of the others' products are not read, and no column touches
//      another).  Otherwise two heads have a tile each.
//   rows  Load j of a key tile holds tokens COLS j .. + COLS - 1, lanes h COLS .. their
//      rows of head h.  Head h's operand has them in its lanes g COLS .. from load (g -
//      h) % NH, turned by (g - h) COLS lanes (DPP): its row r is token turned(r, -h),
//      where turned(r, x) moves r's group of COLS by x groups.  V's rows of head h are
//      stored in the same order, and its columns' masks read so.
// Loads run two steps ahead of their use in registers (three steps: the third spills,
// 167 us became 197; dealing whole lines out through LDS instead: 147-157).
// ---------------------------------------------------------------------------
constexpr int kNarrowWaves = 4;             // waves of a STREAM workgroup
constexpr int kItemWaves = 8;               // waves of a workgroup per item
constexpr int kAhead = 3;                   // V operands read ahead of their product

// Waves per SIMD that the registers are bounded for, by what two steps' loads and the
// accumulators take (a bound that they do not fit costs more than the wave it gains):
//   rows of 128 bytes         2, and 1 with two tiles (at 2: 64 x 7 tokens over 5300-16000
//                             327 us, at 1 322; 16 x 7 over 4000 42, 40)
//   heads of 128, two heads   2
//   heads of 64 in 8 bits     3, and 2 with two tiles (at 4, 3 spilling 6-14: 64 x 1 over
//                             16000, 3 heads, 136, so 107; 24 x 4 tokens over 4000 42, 36;
//                             64 x 6 tokens over 16000 407, 250; but 64 x 7 over 5300-16000
//                             248, 255)
//   others                    4, and 3 with two tiles
// (Heads of 128 in 4 bits spill 19-21 registers of a lane with a tile each for two heads,
// 1-6 with several heads in one; of 64 in 4 bits 1 with four heads.)
constexpr int quant_waves(int d, int bits, int qb, int nh) {
    if (d * bits == 1024) return qb > 1 ? 1 : 2;
    if (d == 128 || nh > 1) return 2;
    return (qb > 1 ? 3 : 4) - (d * bits == 512);
}

// NW waves for G sets of NH kv heads.  (NH > 1: QB = 1 is one tile of columns for all of
// them, QB = NH a tile each.)
template <typename T, int D, int BITS, int QB, int NW, int NH, int G, bool STREAM>
__global__ __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(quant_waves(D, BITS, QB, NH)))) void quant_attn_kernel(QuantParams p) {
    constexpr int NC = D / 32;              // k-steps of S^T over the head dim
    constexpr int ND = D / 16;              // d-tiles of O^T
    constexpr int DV = D / 8;               // 16-byte chunks per widened row
    constexpr int NS = D / kQuantBlock;     // scales per row
    constexpr int SW = (NH * NS + 3) / 4;   // words of a token's scales (K's or V's)
    constexpr int KW = D * BITS / 128;      // words of a quarter row
    constexpr int RB = D * BITS / 8;        // bytes of a row
    constexpr int VB = RB / 2 < 16 ? RB / 2 : 16;  // bytes of V per lane and load
    constexpr int LPR = RB / VB;            // lanes per V row
    constexpr int TPI = 64 / (NH * LPR);    // tokens per V load
    constexpr int NV = 32 / TPI;            // V loads per lane and step
    constexpr int SUB = VB / BITS;          // chunks of 8 elements per load
    constexpr int WBLK = 32 * D;            // elements of a head's V block
    constexpr bool OWN = NH > 1 && QB == NH;  // a tile of columns per head
    constexpr int ROWS = NH > 1 ? 16 : 16 * QB;  // of an item
    constexpr int COLS = 16 / NH;           // tokens of a K load; columns of a head, where heads share a tile
    constexpr int HC = OWN ? 16 : COLS;     // columns of a head
    constexpr int NO = OWN ? NH : QB * NH;  // tiles of O^T
    constexpr int WPH = NW / G;             // waves of a set of heads
    constexpr int KEYS = 32 * WPH;          // of a unit
    constexpr bool ONCE = NH * RB >= 128;   // a load's tokens are whole lines: past the caches
    static_assert(LPR * SUB == DV && NV * TPI == 32 && TPI % 8 == 0 && NC * BITS / 4 == KW, "a step is 32 rows");
    static_assert(NH == 1 || ((QB == 1 || OWN) && NH * RB <= 128), "one tile of columns, or one per head");
    // The waves' V blocks; after the key loop, the waves' numerators of one
    // row block (NW x 16 rows x D floats, the size of one head's).
    __shared__ __attribute__((aligned(4096))) uint16_t vlds[NW * NH * WBLK];  // (16 rows: bits of an address)
    __shared__ float ml[2][NW][16 * QB];

    Share sh{};
    if constexpr (STREAM) {
        if (!find_share<64 * NW>(p, sh)) return;
    } else {
        sh.end = 1;  // one part: the item
    }
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int l16 = lane & 15, lq = lane >> 4;

    // wave-private V block: chunk c of row r at c ^ kv_swz(r)
    // (byte addresses; the others are these with bits flipped.  hide() keeps the compiler
    // from holding a register for each, which spills.)
    const uint32_t vblk = lds_at(vlds + wave * NH * WBLK);
    const int vr = 4 * lq + (l16 >> 2);
    uint32_t vget = vblk + 2 * (vr * D + 8 * (((l16 & 3) >> 1) ^ kv_swz(vr, DV)) + 4 * (l16 & 1));
    // The lane's token in V's load 0 (+ n TPI) and head there: with four lanes per row
    // neighbouring quads take rows two apart, whose swizzles keep their stores in
    // different banks.
    const int vj = lane / LPR % TPI, vhead = lane / (LPR * TPI);
    const int vtok = LPR == 4 ? (vj & ~3) | (vj & 1) << 1 | (vj >> 1 & 1) : vj;
    auto turned = [](int r, int x) { return (r & ~15) | ((r / COLS + x) * COLS & 15) | r % COLS; };
    const int vrow = turned(vtok, vhead);
    uint32_t vput = vblk + 2 * (WBLK * vhead + vrow * D + 8 * (lane % LPR ^ kv_swz(vrow, DV)));
    auto hide = [&] { asm volatile("" : "+v"(vget), "+v"(vput)); };
    // the lane's scale in a word of them
    const int kshift = 8 * (lq * NS / 4);
    const int vshift = 8 * (vhead * NS % 4 + (lane % LPR) * (VB * 8 / BITS) / kQuantBlock);

    while (sh.u < sh.end) {
        Part part;
        SeqWork sw;
        if constexpr (STREAM) {
            sw = next_part(p, sh, part);
        } else {
            const int item = divide(blockIdx.x, p.groupdiv);
            part.group = blockIdx.x - item * p.groups;
            sh.seq = divide(item, p.tilediv);
            part.tile = item - sh.seq * p.tiles;
            sw = seq_work(p, sh.seq);
            if (part.tile >= sw.tiles) return;
            part.b0 = 0, part.b1 = sw.blocks, part.whole = true;
        }
        const int tile = part.tile, b0 = part.b0, b1 = part.b1, ctx = sw.ctx;
        const int kvh = (part.group * G + wave / WPH) * NH;  // the wave's first head

        // column r of the wave's tiles: a row of head kvh + r / HC (all of the tiles'
        // rows, where the wave has one head)
        auto query_of = [&](int r, int64_t& qrow, int& qh) {
            const int rr = NH == 1 ? tile * 16 * QB + r : r % HC;
            const int tok = divide(rr, p.gdiv);
            qh = (kvh + (NH == 1 ? 0 : r / HC)) * p.group + (rr - tok * p.group);
            qrow = (int64_t)sw.s0 + tok;
            return rr < sw.rows;
        };
        // Q^T operand of k-step c: dims D/4 lq + 8 c .. + 7 of the lane's column
        Vec16 qf[QB][NC];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            int64_t qrow;
            int qh;
            const bool valid = query_of(16 * b + l16, qrow, qh);
            const uint16_t* qp = p.q + qrow * p.sq_t + qh * p.sq_h + D / 4 * lq;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                qf[b][c] = Vec16{{0u, 0u, 0u, 0u}};
                if (valid) qf[b][c] = ld16(qp + 8 * c);
            }
        }
        float m_run[QB], l_run[QB];
        f4_t oacc[NO][ND];
#pragma unroll
        for (int b = 0; b < NO; ++b)
#pragma unroll
            for (int i = 0; i < ND; ++i) oacc[b][i] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
        for (int b = 0; b < QB; ++b) m_run[b] = -INFINITY, l_run[b] = 0.f;
        const char* const kb = (const char*)(p.kc + kvh * p.sk_head) + RB * (l16 / COLS) + 4 * KW * lq;
        const char* const vb = (const char*)(p.vc + kvh * p.sk_head) + RB * vhead + VB * (lane % LPR);
        // one word per token: lanes 0 .. 31 K's, 32 .. 63 V's; two: K's, then V's, lanes
        // 32 .. 63 the second
        const char* const sb = (const char*)(SW == 2 || lane < 32 ? p.ks : p.vs) + kvh * p.ss_head +
                               (SW == 2 ? lane / 32 * 4 : 0);
        const char* const sb2 = (const char*)p.vs + kvh * p.ss_head + lane / 32 * 4;
        const int32_t* const pt = p.table + (int64_t)sh.seq * p.pt_cols;

        // key lane % 32 of step b, and its page (within the table: what lies past the
        // context is not used)
        auto key_at = [&](int b) { return KEYS * b + 32 * (wave % WPH) + (lane & 31); };
        auto page_at = [&](int b) { return pt[divide(min(key_at(b), p.capacity - 1), p.pdiv)]; };
        // x of the lane at byte 4 * lane
        auto from = [](uint32_t x, int at) { return (uint32_t)__builtin_amdgcn_ds_bpermute(at, (int)x); };
        const int klane = 4 * (l16 % COLS), vlane = 4 * vtok;
        const int vslane = vlane + (SW == 2 ? 128 * (vhead * NS / 4) : 128);
        // A step's loads, requested two steps ahead.  Keys that do not exist, and those
        // of steps past the part, read the cache's first row and count for nothing.
        struct Raw {
            uint32_t k[2][NH][KW], v[NV][VB / 4], s[SW];
            uint32_t have;  // bit j: key j of the step exists
        };
        auto issue = [&](Raw& r, int b, int page) {
            const int pos = key_at(b);
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages && pos < ctx && b < b1;
            r.have = (uint32_t)__ballot(ok);
            const int slot = pos - divide(pos, p.pdiv) * p.page_size;
            // row offsets in 16-byte units, scales in rows of them (both below 2^32)
            const uint32_t off = ok ? (uint32_t)page * p.row_page + (uint32_t)slot * p.row_slot : 0u;
            const uint32_t so = ok ? (uint32_t)page * p.scale_page + (uint32_t)slot * p.scale_slot : 0u;
            uint32_t ko[2][NH], vo[NV];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < NH; ++j) ko[t][j] = from(off, klane + 64 * t + 4 * COLS * j);
#pragma unroll
            for (int n = 0; n < NV; ++n) vo[n] = from(off, vlane + 4 * TPI * n);
            r.s[0] = ld_scales<SW == 2 ? 4 : NH * NS>(sb + NS * (uint64_t)so);
            if constexpr (SW == 2) r.s[1] = ld_scales<4>(sb2 + NS * (uint64_t)so);
#pragma unroll
            for (int n = 0; n < NV; ++n) ld_words<ONCE>(r.v[n], vb + 16 * (uint64_t)vo[n]);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int j = 0; j < NH; ++j) ld_words<ONCE>(r.k[t][j], kb + 16 * (uint64_t)ko[t][j]);
            // (requests keep their order, so that a wait for one step's is no wait for the next one's)
            __builtin_amdgcn_sched_barrier(0);
        };
        int page = 0;  // of the step after the next
        auto step = [&](Raw& r, int b) {
            hide();
            const int after = page_at(b + 3);  // (ahead of the loads that it does not wait for)
            const uint32_t mask = r.have;
            // scales of the lane's V rows, and of the rows of K's operands
            float vscale[NV], kscale[2][NH];
#pragma unroll
            for (int n = 0; n < NV; ++n)
                vscale[n] = scale_of(from(r.s[SW - 1], vslane + 4 * TPI * n) >> vshift & 255u);
#pragma unroll
            for (int h = 0; h < NH; ++h)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    kscale[t][h] = scale_of(from(r.s[0], 4 * turned(l16, NH - h) + 64 * t + 128 * (h * NS / 4)) >>
                                                (8 * (h * NS % 4) + kshift) & 255u);
            // V to LDS; rows of keys that do not exist as zeros (weight 0
            // times what lies there could be NaN)
            if (mask != 0xffffffffu) {
                const uint32_t mine = mask >> vtok;
#pragma unroll
                for (int n = 0; n < NV; ++n) {
                    const bool there = mine >> (n * TPI) & 1;
                    vscale[n] = there ? vscale[n] : 1.f;
#pragma unroll
                    for (int i = 0; i < VB / 4; ++i) r.v[n][i] = there ? r.v[n][i] : 0u;
                }
            }
#pragma unroll
            for (int n = 0; n < NV; ++n)
#pragma unroll
                for (int i = 0; i < SUB; ++i) {
                    // (of 8 tokens per load, those of odd loads lie 8 rows further or before)
                    constexpr int ODD = TPI % 16;
                    const uint32_t at = (vput ^ (16 * (LPR * i) ^ (n % 2 ? 16 * kv_swz(ODD, DV) ^ 2 * D * ODD : 0))) +
                                        2 * D * (TPI * n / 16 * 16);
                    const Vec16 x = widen8<T, BITS>(r.v[n] + i * (BITS / 4), vscale[n]);
                    *(__attribute__((address_space(3))) w4_t*)(uintptr_t)at = w4_t{x.w[0], x.w[1], x.w[2], x.w[3]};
                }
            // scores: every head's K with its own tile of columns; where heads share one, with
            // all columns, each column from its own head (no zeros in the other columns: 0
            // times what is no number is none either)
            f4_t s[QB][2];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int h = 0; h < NH; ++h) {
                    uint32_t kw[KW];
#pragma unroll
                    for (int i = 0; i < KW; ++i) kw[i] = turn_in<NH>(r.k[t], i, h);
                    f4_t x[QB];
#pragma unroll
                    for (int q = 0; q < QB; ++q) x[q] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < NC; ++c) {
                        const Vec16 k = widen8<T, BITS>(kw + c * (BITS / 4), kscale[t][h]);
#pragma unroll
                        for (int q = 0; q < QB; ++q)
                            if (!OWN || q == h) x[q] = MfmaOps<T>::mma(k, qf[q][c], x[q]);
                    }
#pragma unroll
                    for (int q = 0; q < QB; ++q) {
                        if (OWN && q != h) continue;
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            s[q][t][i] = OWN || h == 0 || l16 / COLS == h ? x[q][i] : s[q][t][i];
                    }
                }
            issue(r, b + 2, page);
            page = after;
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            Vec16 pf[QB];
            float alpha[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                // lane: rows 16 t + 4 lq + i of column l16
                if (mask != 0xffffffffu) {
                    uint32_t mine = mask >> turned(4 * lq, NH - (OWN ? q : l16 / COLS));
                    asm volatile("" : "+v"(mine));  // (eight tests of one word, no eight lane masks)
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(mine >> (16 * t + i) & 1)) s[q][t][i] = -INFINITY;
                }
                float mb = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mb = fmaxf(mb, s[q][t][i]);
                const float m_new = fmaxf(m_run[q], col4_max(mb));
                // (a row of -inf scores alone keeps weights of zero)
                const float mc = m_new == -INFINITY ? 0.f : m_new * p.scale_log2;
                alpha[q] = fast_exp2(__builtin_fmaf(m_run[q], p.scale_log2, -mc));
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[q][t][i] = fast_exp2(__builtin_fmaf(s[q][t][i], p.scale_log2, -mc));
                        sum += s[q][t][i];
                    }
                l_run[q] = l_run[q] * alpha[q] + sum;
                m_run[q] = m_new;
                // P is rounded to the queries' type for the product (its sum is
                // not): half a step of each weight, as one rounding of the output
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    pf[q].w[2 * t] = MfmaOps<T>::pack2(s[q][t][0], s[q][t][1]);
                    pf[q].w[2 * t + 1] = MfmaOps<T>::pack2(s[q][t][2], s[q][t][3]);
                }
            }
            bool moved = false;
#pragma unroll
            for (int q = 0; q < QB; ++q) moved |= alpha[q] != 1.f;
            if (__any(moved)) {
#pragma unroll
                for (int o = 0; o < NO; ++o)
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) oacc[o][dt] *= alpha[QB == 1 ? 0 : o];
            }
            auto v_operand = [&](int i) {  // d-tile i % ND of head i / ND
                typedef short v4s __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) v4s* lds_v4s;
                const uint32_t a = (vget ^ (32 * (i % ND))) + 2 * WBLK * (i / ND);
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)a);
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(uintptr_t)(a + 32 * D));
                const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                return Vec16{{l2.x, l2.y, h2.x, h2.y}};
            };
            constexpr int NT = NH * ND, AHEAD = NT < kAhead ? NT : kAhead;
            Vec16 va[AHEAD];
#pragma unroll
            for (int i = 0; i < AHEAD; ++i) va[i] = v_operand(i);
#pragma unroll
            for (int i = 0; i < NT; ++i) {
                const Vec16 v = va[i % AHEAD];
#pragma unroll
                for (int q = 0; q < QB; ++q) {
                    if (OWN && q != i / ND) continue;
                    const int o = OWN ? q : q + i / ND;
                    oacc[o][i % ND] = MfmaOps<T>::mma(v, pf[q], oacc[o][i % ND]);
                }
                if (i + AHEAD < NT) va[i % AHEAD] = v_operand(i + AHEAD);
                __builtin_amdgcn_sched_barrier(0);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();  // the block's reads come before the next step's writes
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        };
        if (ctx > 0) {  // (no context: nothing to read, maybe no cache)
            Raw r0, r1;
            const int first = page_at(b0), second = page_at(b0 + 1);
            page = page_at(b0 + 2);
            __builtin_amdgcn_sched_barrier(0);
            issue(r0, b0, first);
            issue(r1, b0 + 1, second);
            for (int b = b0;;) {
                step(r0, b);
                if (++b >= b1) break;
                step(r1, b);
                if (++b >= b1) break;
            }
        }
        auto dims_of = [](int ch) { return ch % LPR * SUB + ch / LPR; };
        auto state_of = [&](int r) {
            return (wave / WPH * NH + (NH == 1 ? 0 : r / HC)) * ROWS + (NH == 1 ? r : r % HC);
        };
        if constexpr (NH > 1 && !OWN) {
            // each column of the head that it belongs to
            f4_t own[1][ND];
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                own[0][dt] = oacc[0][dt];
#pragma unroll
                for (int h = 1; h < NH; ++h)
#pragma unroll
                    for (int i = 0; i < 4; ++i) own[0][dt][i] = l16 / COLS == h ? oacc[h][dt][i] : own[0][dt][i];
            }
            join_waves<T, D, 1, NW, G>(p, sh, part, query_of, m_run, l_run, own, vlds, ml, dims_of, NH * G * ROWS, state_of);
        } else {
            join_waves<T, D, QB, NW, G>(p, sh, part, query_of, m_run, l_run, oacc, vlds, ml, dims_of, NH * G * ROWS, state_of);
        }
        __syncthreads();  // the LDS is free for the next item
        sh.u += STREAM ? b1 - b0 : 1;
    }
}

// ---------------------------------------------------------------------------
// Many rows (128 per tile): the key loop of dense_tiles.h over blocks that are
// widened on their way into its LDS buffers.  A thread has a quarter of a key row
// of each block: its elements and scale are loaded into registers where that loop
// would start the block's LDS loads one iteration earlier, widened and stored in
// D/32 pieces of 16 bytes, each where the loop would start one load.  Chunk n of
// quarter qd lies at place 4 n + qd of its row (a quarter-row's writes side by
// side, no bank twice), which orders the dims of S's products (Q is read alike) and
// of O's columns (put back where they are stored).
// 2 x 1009 tokens over 6007, 8 bits, 8 heads of 128 for 32: 212 us, 0.93 PFLOP/s of 1.23 that
// a library product of 8192^3 reaches (229 over 16 bits); 4 x 60 over 10240, 4 bits: 66, 8 of
// them the join and some 15 the first loads and the states of the 512 workgroups' cut
// items.  With heads of 128, 14 to 20 registers of a lane spill.
// ---------------------------------------------------------------------------
constexpr int kWideKeys = 64;
// Blocks whose keys are looked up at once: the LDS that the buffers leave two workgroups.  (A
// table's end empties the loop, and the next one waits for its pages and first blocks: 0.8
// us.  94 blocks per workgroup, 2 x 1009 tokens over 6007: 212.5 us, by tables of 12 215.8.)
constexpr int kTable = 24;

struct QuantTable {
    uint32_t row[kTable][kWideKeys];    // offsets in 16-byte units
    uint32_t scale[kTable][kWideKeys];  // in rows of scales
    uint64_t have[kTable];              // bit r: key r exists
};

template <typename T, int D, int BITS>
struct QuantKeys {
    using Tile = DenseTile<T, D>;
    static constexpr bool kEveryBlock = true;
    static constexpr int NI = Tile::NI, DV = Tile::DV, BLK = Tile::BLK;
    static constexpr int KW = D * BITS / 128, W = BITS / 4, NS = D / kQuantBlock;
    const QuantTable* tab;
    const char *kbase, *vbase, *ksbase, *vsbase;
    int nb;        // blocks in the table
    uint32_t bad;  // blocks with a key that does not exist
    uint32_t lds0, put;
    int row;
    // loaded and not yet widened: K and V of the block that dma(j) stores next, and
    // (before the loop) K of block 1
    mutable uint32_t rk[KW], rv[KW], r1[KW], ck, cv, c1;

    // Fills the table with blocks b0 .. b0 + n - 1 of the sequence.
    __device__ __forceinline__ QuantKeys(const QuantParams& p, QuantTable& t, const int32_t* pages, int ctx, int kvh,
                                         int b0, int n, const uint16_t* smem)
        : tab(&t), nb(n) {
        const int lane = threadIdx.x & 63;
        const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        const int qd = threadIdx.x & 3;
        row = threadIdx.x >> 2;
        kbase = (const char*)(p.kc + (int64_t)kvh * p.sk_head) + 4 * KW * qd;
        vbase = (const char*)(p.vc + (int64_t)kvh * p.sk_head) + 4 * KW * qd;
        ksbase = (const char*)p.ks + kvh * p.ss_head + qd * NS / 4;
        vsbase = (const char*)p.vs + kvh * p.ss_head + qd * NS / 4;
        lds0 = lds_at(smem);
        put = 2 * D * row + 16 * (qd ^ kv_swz32(row, DV));
        __syncthreads();  // the table's and the buffers' last readers are done
        for (int i = wave; i < n; i += 4) {
            const int pos = (b0 + i) * kWideKeys + lane;
            int page = -1;
            const int col = divide(pos, p.pdiv);
            if (pos < ctx) page = pages[col];
            const int slot = pos - col * p.page_size;
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages;
            // (keys that do not exist read the cache's first row)
            t.row[i][lane] = ok ? (uint32_t)page * p.row_page + (uint32_t)slot * p.row_slot : 0u;
            t.scale[i][lane] = ok ? (uint32_t)page * p.scale_page + (uint32_t)slot * p.scale_slot : 0u;
            const uint64_t have = __ballot(ok);
            if (lane == 0) t.have[i] = have;
        }
        __syncthreads();
        bad = (uint32_t)__ballot(lane < n && t.have[lane < n ? lane : 0] != ~0ull);
        fetch(0, kbase, ksbase, rk, ck);
        fetch(0, vbase, vsbase, rv, cv);
        fetch(1, kbase, ksbase, r1, c1);
    }
    __device__ __forceinline__ void fetch(int j, const char* base, const char* sbase, uint32_t (&r)[KW],
                                          uint32_t& c) const {
        const int b = min(j, nb - 1);  // (past the last block: stored, never read)
        ld_words(r, base + 16 * (uint64_t)tab->row[b][row]);
        c = *reinterpret_cast<const uint8_t*>(sbase + NS * (uint64_t)tab->scale[b][row]);
    }
    // A key of block j that does not exist is zeros.  (Once per block: a test at each
    // piece cut the loop into 8 basic blocks more.)
    __device__ __forceinline__ void drop(int j, uint32_t (&r)[KW], uint32_t& c) const {
        const int b = min(j, nb - 1);
        if (__builtin_expect(bad >> b & 1, 0)) {
            if (!(tab->have[b] >> row & 1)) {
                c = 127;
#pragma unroll
                for (int i = 0; i < KW; ++i) r[i] = 0;
            }
        }
    }
    // Piece n of the quarter to the buffer at dst.
    __device__ __forceinline__ void store(int n, const uint32_t (&r)[KW], uint32_t c, uint32_t dst) const {
        const Vec16 x = widen8<T, BITS>(r + n * W, scale_of(c));
        *(__attribute__((address_space(3))) w4_t*)(uintptr_t)(dst + (put ^ (64 * n))) =
            w4_t{x.w[0], x.w[1], x.w[2], x.w[3]};
    }
    struct Dma {
        const QuantKeys& src;
        int j;
        __device__ __forceinline__ void k(int buf, int n) {
            if (n == 0) src.drop(j + 3, src.rk, src.ck);
            src.store(n, src.rk, src.ck, src.lds0 + 2 * buf * BLK);
            if (n == NI - 1) src.fetch(j + 4, src.kbase, src.ksbase, src.rk, src.ck);
        }
        __device__ __forceinline__ void v(int buf, int n) {
            if (n == 0) src.drop(j + 1, src.rv, src.cv);
            src.store(n, src.rv, src.cv, src.lds0 + 2 * (2 + buf) * BLK);
            if (n == NI - 1) src.fetch(j + 2, src.vbase, src.vsbase, src.rv, src.cv);
        }
    };
    __device__ __forceinline__ Dma dma(int j) const { return Dma{*this, j}; }
    // Blocks 0 to 2, before the loop.
    __device__ __forceinline__ void load_k(int j, uint16_t* buf) const {
        if (j == 1) drop(1, r1, c1);
        else drop(j, rk, ck);
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            if (j == 1) store(n, r1, c1, lds_at(buf));
            else store(n, rk, ck, lds_at(buf));
        }
        if (j == 0) fetch(2, kbase, ksbase, rk, ck);
        if (j == 2) fetch(3, kbase, ksbase, rk, ck);
    }
    __device__ __forceinline__ void load_v(int j, uint16_t* buf) const {
        drop(j, rv, cv);
#pragma unroll
        for (int n = 0; n < NI; ++n) store(n, rv, cv, lds_at(buf));
        fetch(j + 1, vbase, vsbase, rv, cv);
    }
    __device__ __forceinline__ void mask(int j, f16v_t (&s)[2]) const {
        if (__builtin_expect(bad >> j & 1, 0)) {
            const uint64_t have = tab->have[j] >> (4 * ((threadIdx.x >> 5) & 1));
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r)
                    if (!((uint32_t)(have >> (32 * t)) >> (8 * (r >> 2) + (r & 3)) & 1)) s[t][r] = -INFINITY;
        }
    }
    template <bool SCAN, class... O>
    __device__ __forceinline__ void clean(int, uint16_t*, O&...) const {}  // (zeros already)
};

template <typename T, int D, int BITS>
__global__ __launch_bounds__(kPagedThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void quant_wide_kernel(
    QuantParams p) {
    using Tile = DenseTile<T, D>;
    constexpr int KS = Tile::KS, DT = Tile::DT, ROWS = Tile::kBM;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[Tile::kSmem];
    __shared__ __attribute__((aligned(16))) QuantTable table;

    Share sh;
    if (!find_share(p, sh)) return;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    const int q32 = lane & 31, hl = lane >> 5;

    while (sh.u < sh.end) {
        Part part;
        const SeqWork sw = next_part(p, sh, part);
        auto query_of = [&](int64_t& qrow, int& qh) {
            const int rr = part.tile * ROWS + wave * 32 + q32;
            const int tok = divide(rr, p.gdiv);
            qh = part.group * p.group + (rr - tok * p.group);
            qrow = (int64_t)sw.s0 + tok;
            return rr < sw.rows;
        };
        // k-step s takes the chunks at places 2 s + hl of a row
        Vec16 qf[KS];
        {
            int64_t qrow;
            int qh;
            const bool valid = query_of(qrow, qh);
            const uint16_t* qp = p.q + qrow * p.sq_t + qh * p.sq_h + D / 4 * hl;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[s] = Vec16{{0u, 0u, 0u, 0u}};
                if (valid) qf[s] = ld16(qp + D / 4 * (2 * s % 4) + 8 * (2 * s / 4));
            }
        }
        float m_run = -INFINITY, l_run = 0.f;
        f16v_t oacc[DT];
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[dt][r] = 0.f;
        const bool live = part.tile * ROWS + wave * 32 < sw.rows;
        for (int b = part.b0; b < part.b1 && sw.ctx > 0; b += kTable) {
            const QuantKeys<T, D, BITS> src(p, table, p.table + (int64_t)sh.seq * p.pt_cols, sw.ctx, part.group, b,
                                            min(kTable, part.b1 - b), smem);
            Tile::template keys<false>(src, smem, qf, live, src.nb, p.scale_log2, m_run, l_run, oacc);
        }
        const float l = xor32_sum(l_run);
        int64_t qrow;
        int qh;
        const bool valid = query_of(qrow, qh);
        if (part.whole) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
            Tile::template store_row<true>(oacc, inv, p.o + qrow * p.so_t + qh * p.so_h, valid);
            if (valid && p.lse && hl == 0)
                p.lse[qrow * p.sl_t + qh * p.sl_h] = (m_run * p.scale_log2 + fast_log2(l)) * kLn2;
        } else if (valid) {
            const int64_t r = part_slot(sh) * ROWS + wave * 32 + q32;
            if (hl == 0) {
                p.part_m[r] = m_run * p.scale_log2;
                p.part_l[r] = l;
            }
            Tile::template store_state<true>(oacc, p.part_acc + r * D);
        }
        sh.u += part.b1 - part.b0;
    }
}

// ---------------------------------------------------------------------------
// Joins the parts of the wide kernel's cut items: SUB workgroups per run, for the item
// that the run starts inside (the first such run joins it), D / 8 lanes per row, kParts
// states in flight.  Where nothing is cut a workgroup ends on its first load: a wave
// per row of the call instead looked for nothing for 21 us of a chunk's 237 (2 x 1009
// tokens over 6007).  A run's states are read on the XCD that wrote them.
// ---------------------------------------------------------------------------
constexpr int kParts = 4;

template <int D>
constexpr int kJoinRows = 4 * 64 / (D / 8);  // of a workgroup

template <typename T, int D>
__global__ __launch_bounds__(kPagedThreads) void quant_join_kernel(PagedParams p) {
    constexpr int LPR = D / 8, SUB = DenseTile<T, D>::kBM / kJoinRows<D>;
    const int per = p.nwg >> 3, in = blockIdx.x >> 3;
    const int w = (blockIdx.x & 7) * per + in / SUB;
    const RunStart c = p.cuts[w];
    if (c.b0 == 0) return;
    const Runs runs(c.total, p.nwg, p.least);
    const int32_t a = c.first;
    if (w > 0 && runs.first(w - 1) > a) return;
    const int rr = in % SUB * kJoinRows<D> + threadIdx.x / LPR, ch = threadIdx.x % LPR;
    const int in_seq = (c.tile << p.row_shift) + rr;
    if (in_seq >= c.rows) return;
    const int w0 = runs.of(a), w1 = runs.of(a + c.blocks - 1) + 1;
    float m = -INFINITY, l = 0.f, acc[8] = {};
    for (int v = w0; v < w1; v += kParts) {
        float mi[kParts], li[kParts];
        float4 x[kParts], y[kParts];
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            // (past the last part: the last one again, with a weight of 0)
            const int ww = min(v + u, w1 - 1);
            const int64_t row = ((2 * (int64_t)ww + (runs.first(ww) >= a ? 0 : 1)) << p.row_shift) + rr;
            mi[u] = v + u < w1 ? p.part_m[row] : -INFINITY;
            li[u] = v + u < w1 ? p.part_l[row] : 0.f;
            const float4* from = reinterpret_cast<const float4*>(p.part_acc + row * D + 8 * ch);
            x[u] = from[0], y[u] = from[1];
        }
        float mn = m;
#pragma unroll
        for (int u = 0; u < kParts; ++u) mn = fmaxf(mn, mi[u]);
        const float mc = mn == -INFINITY ? 0.f : mn, old = fast_exp2(m - mc);
        l *= old;
#pragma unroll
        for (int i = 0; i < 8; ++i) acc[i] *= old;
#pragma unroll
        for (int u = 0; u < kParts; ++u) {
            if (v + u >= w1) break;
            const float f = fast_exp2(mi[u] - mc);
            l += f * li[u];
            acc[0] += f * x[u].x, acc[1] += f * x[u].y, acc[2] += f * x[u].z, acc[3] += f * x[u].w;
            acc[4] += f * y[u].x, acc[5] += f * y[u].y, acc[6] += f * y[u].z, acc[7] += f * y[u].w;
        }
        m = mn;
    }
    const int tok = divide(in_seq, p.gdiv);
    const int qh = c.group * p.group + (in_seq - tok * p.group);
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
    for (int i = 0; i < 8; ++i) acc[i] = in_range<T>(acc[i] * inv);
    const int64_t qrow = (int64_t)c.s0 + tok;
    st16(p.o + qrow * p.so_t + qh * p.so_h + 8 * ch, pack8<T>(acc));
    if (p.lse && ch == 0) p.lse[qrow * p.sl_t + qh * p.sl_h] = ((m == -INFINITY ? 0.f : m) + fast_log2(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Largest power of two up to `most` that divides n.
static int pow2_part(int n, int most) {
    int g = 1;
    while (2 * g <= most && n % (2 * g) == 0) g *= 2;
    return g;
}

// together: the heads of a token lie side by side, elements and scales.
//
// The choices, each with both sides measured (us a call, graphs of calls on caches that
// no call before left in the chip's; 32 q heads for 8 kv heads of 128 where nothing else
// is said):
//   A workgroup per item (8 waves, nothing joined by a second launch) or runs: up to 4
//   steps per wave, but up to 2 where rows are 128 bytes and the items no more than 64.  Two
//   more steps take 3 us in rows of up to 64 bytes, about what the second launch and the
//   states of runs take, but 6 in rows of 128, as a workgroup draws some 22 bytes a ns however
//   few there are; with more items runs hold several steps too.  4 bits: 2 x 731
//   9.3, runs 11.4; 1 x 1000 10.4, 11.1; 16 x 1000 14.1, 15.8; 32 x 1000 18.4, 19.5; but
//   4 x 1000 with 32 kv heads 16.9, 15.8, 32 x 1000 with heads of 32 14.3, 12.7 (11.7 and 16.4
//   in 8 bits where the contexts differ).  8 bits, heads of 64: 2 x 1000 9.0, 10.4; 32 x 1000
//   16.2, 16.4.  8 bits, heads of 128: 1 x 480 10.2, 10.5; 2 x 1000 17.2, 11.1; 8 x 800
//   17.0, 14.0; 10 x 800 17.1, 18.1; 10 x 1000 18.6, 18.2; 32 x 1000 22.3, 26.5.
//   Heads of a wave (nh): as many as fill a 128-byte line (see above).
//   Sets of heads of a workgroup (g), each to one wave, or all four waves on one set's
//   keys (g = 1): the first saves the waves' join, the second has more and shorter parts.
//   One head per wave takes sets from 8 steps per wave on, 8 bits: 48 x 4000-12001: 146,
//   g = 1 176; 32 x 4000: 67, 74; 16 x 4000: 43, 42.  Several heads per wave from 16 on,
//   4 bits: 64 x 5300-16000: 154, g = 1 171; 8 x 8000 with 32 kv heads: 77, 84; below,
//   1 x 131072: 54.5, 43.4; 32 x 4000: 44.8, 42.0; 1 x 131072 with 4 heads of 64: 29.1, 24.2.
//   9 .. 16 rows: two heads with a tile of columns each where several sets get 8 steps per
//   wave (48 with heads of 128, whose registers spill), else one head, 4 tokens, 4 bits: 64
//   x 16000 with heads of 64 148, one head 183; 40 x 8000 of 64 63, 67, of 32 44, 54; 24 x
//   8000 of 64 in 8 bits 59, 64; of 128 64 x 5300-16000 167, 182, but 24 x 16000 114, 112.
//   Workgroups per CU with several heads per wave and g = 1: one (1 x 30000: 23.5, two
//   25.1; 32 x 2000: 28.5, 30.2; 4 x 20000 with heads of 64: 25.6, 28.8): a wave's start
//   and the join of twice the parts cost more than the second workgroup hides.
static PagedShape quant_shape(int bits, bool together, int64_t max_rows, int64_t pairs, int hkv, int64_t capacity,
                              int head_dim) {
    const int steps = head_dim * bits < 1024 || pairs > 64 ? 4 : 2;
    if (max_rows <= 16 && capacity <= steps * 32 * kItemWaves && pairs <= 256) return {1, 4, 8, 1, 1, true, 1};
    if (max_rows <= 32) {
        const int qb = max_rows <= 16 ? 1 : 2, row_bytes = head_dim * bits / 8;
        int nh = 1;
        while (together && nh < 4 && 2 * nh * row_bytes <= 128 && max_rows * 2 * nh <= 16 && hkv % (2 * nh) == 0)
            nh *= 2;
        bool own = together && nh == 1 && qb == 1 && 2 * row_bytes <= 128 && hkv % 2 == 0;
        int per_cu, g;
        for (;; own = false) {
            const int n = own ? 2 : nh;
            per_cu = quant_waves(head_dim, bits, qb, n);
            g = max_rows <= 16 ? pow2_part(hkv / n, kNarrowWaves) : 1;
            const int least = own ? (head_dim == 128 ? 48 : 8) : n > 1 ? 16 : 8;
            if (pairs / (n * g) * ((capacity + 31) / 32) < least * 256 * per_cu) g = 1;
            if (!own || g > 1) break;
        }
        if (own) nh = 2;
        if (nh > 1 && g == 1) per_cu = 1;
        return {own ? 2 : qb, qb == 1 ? 4 : 5, 7 - __builtin_ctz((unsigned)g), nh * g, per_cu, false, nh};
    }
    return {0, 7, 6, 1, 2, false, 1};
}

// Whether the wide kernel's cut items are joined by quant_join_kernel: not where an item
// is cut into more than 16 parts, which four waves per row read faster (one context of
// 60000, 10 tokens: 52.8 us against 66.2; 60 tokens 101 and 103; 4 x 60 over 10240 72.4
// and 71.7; 64 x 16 over 300 34.3 and 25.7).
static bool by_runs(const PagedParams& p, const PagedShape& sh) {
    return sh.qb == 0 && (int64_t)p.B * p.Hkv * p.tiles * 16 >= p.nwg;
}

// The main kernel of a call by its name (qattn_debug_quant_kernel): 100 QB + 10 NH + G.
static int form_of(const PagedShape& sh) {
    return sh.qb == 0 ? 0 : 100 * sh.qb + 10 * sh.wave_heads + sh.heads / sh.wave_heads;
}
static const char* name_of(const PagedShape& sh) {
    if (sh.items) return "quant_attn_kernel, a workgroup per item";
    switch (form_of(sh)) {
        case 0: return "quant_wide_kernel";
        case 211: return "quant_attn_kernel, 2 tiles, 1 head";
        case 222: return "quant_attn_kernel, 2 tiles, 2 heads, 2 sets";
        case 224: return "quant_attn_kernel, 2 tiles, 2 heads, 4 sets";
        case 111: return "quant_attn_kernel, 1 head";
        case 112: return "quant_attn_kernel, 1 head, 2 sets";
        case 114: return "quant_attn_kernel, 1 head, 4 sets";
        case 121: return "quant_attn_kernel, 2 heads";
        case 122: return "quant_attn_kernel, 2 heads, 2 sets";
        case 124: return "quant_attn_kernel, 2 heads, 4 sets";
        case 141: return "quant_attn_kernel, 4 heads";
        case 142: return "quant_attn_kernel, 4 heads, 2 sets";
        default: return "quant_attn_kernel, 4 heads, 4 sets";
    }
}

template <typename T, int D, int BITS>
static int launch_quant(const QuantParams& p, const PagedShape& sh, hipStream_t st) {
    const dim3 grid(p.nwg), block(kPagedThreads);
    if (sh.items) {
        hipLaunchKernelGGL((quant_attn_kernel<T, D, BITS, 1, kItemWaves, 1, 1, false>),
                           dim3((uint32_t)(p.B * p.tiles * p.Hkv)), dim3(64 * kItemWaves), 0, st, p);
        return launch_status(name_of(sh));
    }
    constexpr int NH2 = D * BITS / 8 <= 64 ? 2 : 1, NH4 = D * BITS / 8 <= 32 ? 4 : NH2;
#define QATTN_NARROW(QB, NH, G) \
    hipLaunchKernelGGL((quant_attn_kernel<T, D, BITS, QB, kNarrowWaves, NH, G, true>), grid, block, 0, st, p)
    switch (form_of(sh)) {
        case 0: hipLaunchKernelGGL((quant_wide_kernel<T, D, BITS>), grid, block, 0, st, p); break;
        case 211: QATTN_NARROW(2, 1, 1); break;
        case 222: QATTN_NARROW(NH2, NH2, 2); break;
        case 224: QATTN_NARROW(NH2, NH2, 4); break;
        case 111: QATTN_NARROW(1, 1, 1); break;
        case 112: QATTN_NARROW(1, 1, 2); break;
        case 114: QATTN_NARROW(1, 1, 4); break;
        case 121: QATTN_NARROW(1, NH2, 1); break;
        case 122: QATTN_NARROW(1, NH2, 2); break;
        case 124: QATTN_NARROW(1, NH2, 4); break;
        case 141: QATTN_NARROW(1, NH4, 1); break;
        case 142: QATTN_NARROW(1, NH4, 2); break;
        default: QATTN_NARROW(1, NH4, 4);
    }
#undef QATTN_NARROW
    int rc = launch_status(name_of(sh));
    if (rc) return rc;
    if (by_runs(p, sh)) {
        hipLaunchKernelGGL((quant_join_kernel<T, D>), dim3(p.nwg * (DenseTile<T, D>::kBM / kJoinRows<D>)), block, 0,
                           st, p);
        rc = launch_status("quant_join_kernel");
    } else {
        rc = launch_merge<T, D>(p, st);
    }
    return rc ? rc : launch_status(name_of(sh));  // (what a call is told apart by)
}

template <typename T, int BITS>
static int launch_quant(const QuantParams& p, const PagedShape& sh, int head_dim, hipStream_t st) {
    return head_dim == 32   ? launch_quant<T, 32, BITS>(p, sh, st)
           : head_dim == 64 ? launch_quant<T, 64, BITS>(p, sh, st)
                            : launch_quant<T, 128, BITS>(p, sh, st);
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int64_t qattn_prefix_quant_workspace_bytes(int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int32_t pt_cols, int32_t page_size, int32_t bits) {
    // (for heads side by side or not: the call knows the strides)
    int64_t most = 0;
    for (bool together : {false, true})
        most = std::max(most, paged_workspace([=](auto... a) { return quant_shape(bits, together, a...); }, batch,
                                              max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim, pt_cols,
                                              page_size));
    return most;
}

const char* qattn_debug_quant_kernel(int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim, int32_t pt_cols, int32_t page_size,
                                     int32_t bits, int32_t together) {
    PagedPlan plan;
    if (!paged_plan(plan, [=](auto... a) { return quant_shape(bits, together != 0, a...); }, batch, max_seqlen,
                    total_tokens, num_q_heads, num_kv_heads, head_dim, pt_cols, page_size))
        return "";
    return name_of(plan.shape);
}

int qattn_prefix_quant_fwd(const void* q, const int64_t q_stride[3], const void* k_cache, const void* v_cache,
                           const int64_t cache_stride[4], const void* k_scale, const void* v_scale,
                           const int64_t scale_stride[4], const int32_t* page_table, int32_t pt_cols,
                           int32_t num_pages, int32_t page_size, const int32_t* context_lens, void* o,
                           const int64_t o_stride[3], float* lse, const int64_t lse_stride[2],
                           const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale, int32_t dtype,
                           int32_t bits, void* workspace, int64_t workspace_size, void* stream) {
    clear_error();
    int rc = check_quant(k_cache, v_cache, cache_stride, k_scale, v_scale, scale_stride, pt_cols, num_pages, page_size,
                         num_kv_heads, head_dim, dtype, bits);
    if (rc) return rc;
    QuantParams p{};
    PagedPlan plan;
    const int64_t half[4] = {cache_stride[0] / 2, cache_stride[1] / 2, cache_stride[2] / 2, 1};
    // What a wave of NH heads loads of a token's scales at once, words of NH unit bytes or of
    // four, must be aligned; NH is a power of two that divides the heads.  (4 bits, heads of
    // 32, 4 kv heads, whose tokens have 4 scales: 64 x 8000 x 4 tokens 37.5 us, one head per
    // wave 40.1; 8 x 4000 11.0 and 11.9.)
    const int64_t unit = head_dim / kQuantBlock;
    const int64_t sides = std::min<int64_t>(4, (num_kv_heads & -num_kv_heads) * unit);
    const int64_t* ss = scale_stride;
    const bool together = cache_stride[2] == head_dim * bits / 8 && ss[2] == unit && (ss[0] | ss[1]) % sides == 0 &&
                          ((uintptr_t)k_scale | (uintptr_t)v_scale) % sides == 0;
    rc = paged_setup(p, plan, [=](auto... a) { return quant_shape(bits, together, a...); }, q, q_stride, k_cache, half,
                     v_cache, half, page_table, pt_cols, num_pages, page_size, context_lens, o, o_stride, lse,
                     lse_stride, cu_seqlens, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim,
                     scale, dtype, workspace, workspace_size);
    if (rc || plan.nothing) return rc;
    // a row's scales are found by a 32-bit offset in rows of them
    if (pt_cols > 0 && num_pages > 0 &&
        (ss[0] < 0 || ss[1] < 0 || ss[0] > (int64_t(1) << 40) || ss[1] > (int64_t(1) << 32) ||
         (double)(num_pages - 1) * (ss[0] / unit) + (double)(page_size - 1) * (ss[1] / unit) >= 4294967296.0)) {
        set_error("scale strides must be non-negative and a cache's scales span less than 2^32 rows");
        return QATTN_ERR_LAYOUT;
    }
    if (by_runs(p, plan.shape))
        p.cuts = (RunStart*)((char*)workspace + paged_space(batch, plan.nwg, plan.shape, head_dim).cuts);
    p.ks = (const uint8_t*)k_scale, p.vs = (const uint8_t*)v_scale;
    p.ss_head = ss[2];
    // (one page, one slot: the stride is not used)
    p.row_page = num_pages > 1 ? (uint32_t)(half[0] / 8) : 0u;
    p.row_slot = page_size > 1 ? (uint32_t)(half[1] / 8) : 0u;
    p.scale_page = num_pages > 1 ? (uint32_t)(ss[0] / unit) : 0u;
    p.scale_slot = page_size > 1 ? (uint32_t)(ss[1] / unit) : 0u;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == QATTN_DTYPE_F16)
        return bits == 4 ? launch_quant<F16, 4>(p, plan.shape, head_dim, st)
                         : launch_quant<F16, 8>(p, plan.shape, head_dim, st);
    return bits == 4 ? launch_quant<BF16, 4>(p, plan.shape, head_dim, st)
                     : launch_quant<BF16, 8>(p, plan.shape, head_dim, st);
}

}  // extern "C"
