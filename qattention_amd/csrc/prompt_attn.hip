// prompt_attn.hip -- causal attention of packed prompts, with LSE.
//
// For token i of a sequence and q head h (kv head h / group):
//   o = sum_{j <= i} softmax_j(scale q_i.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// in one pass over the keys with a running maximum m and sum l.
//
// Work unit: (sequence, kv head, tile of 128 rows); a row is a (token, q head)
// pair of the kv head's group, tokens outermost, so a tile spans 128 / group
// tokens and a K/V block staged in LDS serves every q head that reads it.
// All tiles of a (sequence, kv head) run on one XCD, the longest first and
// next to those of as many others as fit its L2, so the ~64 workgroups that run
// there at a time read their K/V from it; with fewer pairs than XCDs, or a number
// that 8 does not divide, a pair's tiles are dealt to several.
//
// The key loop (dense_tiles.h) ends at the tile's last token; the blocks that
// reach past a wave's first token are masked by row.
//
// What later tokens hold never shows, although the weights of masked keys are 0
// and 0 times an infinity or a NaN is NaN: a tile whose results are not all
// finite is computed once more, and then infinities and NaN in V are taken out of
// the blocks that hold masked keys and added to the rows that attend them by
// themselves.  (Looking through those blocks always: 16 prompts of 603 .. 2011
// tokens, 32 / 8 heads of 64, bf16: 192 us, so 183.  8192 tokens, 32 / 8 heads of
// 128: 519 us, with NaN in one V row 889.)
#include <algorithm>

#include "dense_tiles.h"
#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kPromptThreads = 256;
constexpr int kBM = 128;  // rows per workgroup
// Waves per SIMD: 64-wide heads have half the products per exponential, and a
// third wave covers what two leave (16 x 1300 tokens, 32 / 8 heads, bf16: 159 us
// with two, 150 with three).
constexpr int prompt_waves(int d) { return d == 64 ? 3 : 2; }

struct PromptParams {
    const uint16_t* q;
    const uint16_t* k;
    const uint16_t* v;
    uint16_t* o;
    float* lse;
    const int32_t* cu;
    int64_t sq_t, sq_h, sk_t, sk_h, sv_t, sv_h, so_t, so_h, sl_t, sl_h;
    int64_t total_tokens;
    int32_t B, Hq, Hkv, group, max_seqlen;
    int32_t qtiles, spread, list;    // tiles of the longest prompt, log2 of lists per pair, tiles of a list
    int32_t xcd_lists, group_lists;  // lists per XCD, lists of a group
    Divider gdiv, groupdiv, hkvdiv;  // group, tiles of a group of lists, Hkv
    // Tiles that sequences of these lengths can have (a multiple of 8), if the
    // launch numbers the tiles that there are; 0: every prompt has qtiles
    int32_t tiles;
    // Cut tiles: blocks of a part at most (0: no tile is cut), parts of the
    // longest tile; states [tile][part][row] of those that are cut
    int32_t part, parts;
    Divider partdiv, hqdiv, msdiv;  // parts, Hq, max_seqlen
    float* part_m;                  // in log2 units
    float* part_l;
    float* part_acc;                // [...][D]
    float scale_log2;
};

// Parts of a tile of nb blocks; part c starts at block first(c).  Equal but for
// one block, so with p.part >= 8 a part of a cut tile has four blocks or more:
// the keys ahead of a tile's last part end 193 keys before the tile's last
// token, and every row (of 128 tokens at most) sees the first block of each part.
struct TileParts {
    int32_t n, q, rem;
    __device__ __forceinline__ TileParts(const PromptParams& p, int nb) {
        n = (int)((uint32_t)(nb + p.part - 1) / (uint32_t)p.part);
        q = (int)((uint32_t)nb / (uint32_t)n);
        rem = nb - q * n;
    }
    __device__ __forceinline__ int first(int c) const { return c * q + min(c, rem); }
};

// The sequence's tokens, 0 where its offsets are not ascending rows of Q.
__device__ __forceinline__ int prompt_tokens(const PromptParams& p, int seq, int& s0) {
    s0 = p.cu[seq];
    const int32_t s1 = p.cu[seq + 1];
    if (s0 < 0 || s1 < s0 || (int64_t)s1 > p.total_tokens) return 0;
    return min(s1 - s0, p.max_seqlen);
}

// Tile i of a launch that numbers the tiles that there are: kv heads innermost
// (8 of them lie on 8 XCDs), then a sequence's tiles, the longest first, then
// sequences.  Every wave looks for it in the offsets by itself.
__device__ __forceinline__ bool numbered_tile(const PromptParams& p, int i, int& seq, int& kvh, int& qt) {
    const int lane = threadIdx.x & 63;
    int t = divide(i, p.hkvdiv);
    kvh = i - t * p.Hkv;
    for (int c = 0; c < p.B; c += 64) {
        int s0, tiles = 0;
        if (c + lane < p.B) tiles = (prompt_tokens(p, c + lane, s0) * p.group + kBM - 1) / kBM;
        int inc = tiles;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int up = __shfl_up(inc, d);
            if (lane >= d) inc += up;
        }
        const uint64_t past = __ballot(t < inc);
        if (past) {
            const int at = __builtin_ctzll(past);
            seq = c + at;
            qt = __builtin_amdgcn_readlane(inc, at) - 1 - t;
            return true;
        }
        t -= __builtin_amdgcn_readlane(inc, 63);
    }
    return false;
}

// The keys of a prompt tile, or of one part of it: rows k_lo .. k_hi - 1 of the
// sequence, contiguous at a token stride (of a tile's last part k_hi - 1 is the
// tile's last token).
template <typename T, int D>
struct PromptKeys {
    using Tile = DenseTile<T, D>;
    static constexpr bool kEveryBlock = false;
    static constexpr int kBN = Tile::kBN, NI = Tile::NI, RPI = Tile::RPI, DV = Tile::DV, BLK = Tile::BLK;
    const char *kbase, *vbase;
    int64_t kst, vst;  // bytes between keys
    int k_lo, k_hi, nb;  // the part's keys and blocks
    int tok_t, tok_w, tok_l;  // first tokens of the tile and of the wave, the lane's token: keys past it are masked
    uint32_t colb, krow, vrow, lds0;
    int wave;
    int* found;  // LDS: 1 + the last block where something not finite was found

    __device__ __forceinline__ PromptKeys(const PromptParams& p, int64_t s0, int kvh, int row0, int lo, int hi,
                                          const uint16_t* smem, int* lds_found)
        : found(lds_found) {
        const int lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        kbase = (const char*)(p.k + s0 * p.sk_t + (int64_t)kvh * p.sk_h);
        vbase = (const char*)(p.v + s0 * p.sv_t + (int64_t)kvh * p.sv_h);
        kst = 2 * p.sk_t, vst = 2 * p.sv_t;
        k_lo = lo, k_hi = hi;
        nb = (hi - lo + kBN - 1) / kBN;
        tok_t = divide(row0, p.gdiv);
        tok_w = divide(row0 + wave * 32, p.gdiv);
        tok_l = divide(row0 + wave * 32 + (lane & 31), p.gdiv);
        // Load n of wave w covers key rows (w NI + n) RPI .. + RPI - 1 of a
        // block; each lane fetches the chunk that the swizzle puts at its
        // position (the swizzle is linear over xor and row n's bits are disjoint
        // from the lane's).  Offsets in a block are 32-bit: the host checks that
        // 64 rows span less than 4 GB.
        colb = 16 * ((lane % DV) ^ kv_swz32(wave * NI * RPI + lane / DV, DV));
        krow = (uint32_t)(wave * NI * RPI + lane / DV) * (uint32_t)kst;
        vrow = (uint32_t)(wave * NI * RPI + lane / DV) * (uint32_t)vst;
        lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)smem + wave * (NI * 1024);
    }
    // First row of block j.  The last block of a range that is no multiple of 64
    // keys starts early (its first keys, also in the block before, are masked
    // and their V rows cleared), and a block past the end repeats it: every load
    // of the key loop is of 64 whole rows, without a bound to clamp to.
    __device__ __forceinline__ int first(int j) const { return min(k_lo + j * kBN, k_hi - kBN); }
    // block 0 may be the only one and shorter than 64 rows: rows past the last repeat it
    __device__ __forceinline__ void load(const char* base, int64_t st, uint32_t row, int j, uint16_t* buf) const {
        const int kb = j == 0 ? k_lo : first(j);
        const uint32_t last = (uint32_t)min(k_hi - 1 - kb, kBN - 1) * (uint32_t)st;
        const char* gb = base + (int64_t)kb * st;
#pragma unroll
        for (int n = 0; n < NI; ++n)
            lds_dma16((colb ^ (16 * kv_swz32(n * RPI, DV))) + min(row + (uint32_t)(n * RPI) * (uint32_t)st, last), gb,
                      buf + (wave * NI + n) * 512);
    }
    __device__ __forceinline__ void load_k(int j, uint16_t* buf) const { load(kbase, kst, krow, j, buf); }
    __device__ __forceinline__ void load_v(int j, uint16_t* buf) const { load(vbase, vst, vrow, j, buf); }

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
    __device__ __forceinline__ Dma dma(int j) const {
        Dma d{colb, krow, vrow, lds0, kbase + (int64_t)first(j + 3) * kst, vbase + (int64_t)first(j + 1) * vst,
              RPI * kst, RPI * vst};
        // (kept from being held in registers per load)
        asm volatile("" : "+v"(d.col), "+v"(d.kr), "+v"(d.vr), "+s"(d.ld));
        return d;
    }
    // keys below lo (they belong to the block before) and past the lane's token
    __device__ __forceinline__ void mask(int j, f16v_t (&s)[2]) const {
        const int lo = k_lo + j * kBN, kb = j == 0 ? k_lo : first(j);
        if (__builtin_expect(kb < lo || kb + kBN - 1 > tok_w, 0)) {
            uint32_t k0 = (uint32_t)(kb - lo + 4 * ((threadIdx.x >> 5) & 1));
            asm volatile("" : "+v"(k0));  // (32 key numbers held across the loop would spill)
            const uint32_t keys = (uint32_t)max(tok_l + 1 - lo, 0);
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int r = 0; r < 16; ++r) {
                    if (k0 + 32 * t + 8 * (r >> 2) + (r & 3) >= keys) s[t][r] = -INFINITY;  // (below lo: wrapped)
                }
        }
    }
    // The rows that the last block shares with the one before set to 0.  SCAN: in a
    // block with keys past the tile's first token, what is not finite goes to the
    // numerators of the rows that attend it (weight 1: an infinity or a NaN is
    // one whatever its weight) and is replaced by 0 in the block.
    template <bool SCAN, class... O>  // (the numerators, or nothing)
    __device__ __forceinline__ void clean(int j, uint16_t* v, O&... o) const {
        const int kb = j == 0 ? k_lo : first(j);
        if (SCAN && kb + kBN - 1 <= tok_t && j + 1 < nb) return;
        const int shared = k_lo + j * kBN - kb;  // (0 but in the last block)
        if (shared > 0) {
            for (int i = threadIdx.x; i < shared * DV; i += Tile::kThreads) st16(v + 8 * i, Vec16{{0u, 0u, 0u, 0u}});
            Tile::sync_lds();
        }
        if constexpr (!SCAN) return;
        constexpr uint32_t kExp = T::kCode == F16::kCode ? 0x7c007c00u : 0x7f807f80u;
        // a word whose low or high half has all exponent bits
        auto odd_word = [&](uint32_t w) {
            const uint32_t x = ~w & kExp;
            return !(x & 0xffffu) || !(x >> 16);
        };
        bool odd = false;
        for (int i = threadIdx.x; i < kBN * DV; i += Tile::kThreads) {
            const Vec16 x = ld16(v + 8 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) odd |= odd_word(x.w[e]);
        }
        if (__any(odd) && (threadIdx.x & 63) == 0) *found = j + 1;
        Tile::sync_lds();
        if (__builtin_expect(__builtin_amdgcn_readfirstlane(*found) != j + 1, 1)) return;
        if constexpr (sizeof...(o) > 0) {
            const int lane = threadIdx.x & 63, hl = lane >> 5;
            // dim 32 dt + 8 i + 4 hl + e of row r: chunk 4 dt + i, at its swizzled place
#pragma unroll 1
            for (int r = 0; r < kBN; ++r) {
                const bool mine = kb + r <= tok_l;
#pragma unroll
                for (int dt = 0; dt < Tile::DT; ++dt)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        const uint2 x = *reinterpret_cast<const uint2*>(
                            v + r * D + 8 * ((4 * dt + i) ^ kv_swz32(r, DV)) + 4 * hl);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t w = e < 2 ? x.x : x.y;
                            const float y = e & 1 ? MfmaOps<T>::hi(w) : MfmaOps<T>::lo(w);
                            ((o[dt][4 * i + e] += mine && !(__builtin_fabsf(y) < INFINITY) ? y : 0.f), ...);
                        }
                    }
            }
        }
        Tile::sync_lds();  // every wave has read the block
        for (int i = threadIdx.x; i < kBN * DV; i += Tile::kThreads) {
            Vec16 x = ld16(v + 8 * i);
#pragma unroll
            for (int e = 0; e < 4; ++e) {
                const uint32_t y = ~x.w[e] & kExp;
                if (!(y & 0xffffu)) x.w[e] &= 0xffff0000u;
                if (!(y >> 16)) x.w[e] &= 0xffffu;
            }
            st16(v + 8 * i, x);
        }
        Tile::sync_lds();
    }
};

template <typename T, int D, bool CUT>
__global__ __launch_bounds__(kPromptThreads) __attribute__((amdgpu_waves_per_eu(prompt_waves(D), prompt_waves(D)))) void prompt_attn_kernel(
    PromptParams p) {
    using Tile = DenseTile<T, D>;
    constexpr int KS = Tile::KS, DT = Tile::DT;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[Tile::kSmem];
    __shared__ int flags[2];  // PromptKeys::found; a wave's results are not finite

    const int i0 = blockIdx.x >> 3;
    const int i = CUT ? divide(i0, p.partdiv) : i0;  // (a tile's parts next to each other)
    const int cut = i0 - i * p.parts;
    int seq, kvh, qt, slot;
    if (p.tiles) {
        slot = 8 * i + (blockIdx.x & 7);
        if (!numbered_tile(p, slot, seq, kvh, qt)) return;
    } else {
        // XCD x (blockIdx % 8) takes lists x, x + 8, ...: list v is every
        // (1 << spread)-th tile of pair v >> spread, the longest first.  Lists are
        // taken in groups, the longest tiles of a group's lists first.
        const int grp = divide(i, p.groupdiv);
        const int in = i - grp * p.group_lists * p.list;
        const int here = min(p.group_lists, p.xcd_lists - grp * p.group_lists);  // lists of this group
        const int k = (int)((uint32_t)in / (uint32_t)here);
        // An XCD deals its workgroups to its shader engines in turn, however busy
        // they are: with a list in the same place of every round, one engine would
        // have the longest prompts' tiles to itself (16 prompts of 603 .. 2011 tokens,
        // 32 / 8 heads of 64, bf16: 215 us; turned by one place per round: 183).
        int at = in - k * here;
        if (!(here & 1)) at = (int)((uint32_t)(at + k) % (uint32_t)here);
        const int v = (blockIdx.x & 7) + 8 * (grp * p.group_lists + at);
        const int pair = v >> p.spread;
        const int rank = (k << p.spread) + (v & ((1 << p.spread) - 1));
        qt = p.qtiles - 1 - rank;
        if (qt < 0) return;
        seq = divide(pair, p.hkvdiv);
        kvh = pair - seq * p.Hkv;
        slot = pair * p.qtiles + qt;
    }
    int32_t s0;
    const int n = prompt_tokens(p, seq, s0);
    const int g = p.group;
    const int rows = n * g;
    if (qt * kBM >= rows) return;

    const int k_hi = divide(min(qt * kBM + kBM, rows) - 1, p.gdiv) + 1;  // past the tile's last token
    int k_first = 0, k_last = k_hi;
    if constexpr (CUT) {
        const TileParts tp(p, (k_hi + Tile::kBN - 1) / Tile::kBN);
        if (cut >= tp.n) return;
        k_first = tp.first(cut) * Tile::kBN;
        k_last = min(k_hi, tp.first(cut + 1) * Tile::kBN);
    }
    const bool whole = !CUT || (k_first == 0 && k_last == k_hi);

    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
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
    auto load_q = [&] {
        int tok, qh;
        const bool valid = query_of(tok, qh);
        const uint16_t* qp = p.q + ((int64_t)s0 + tok) * p.sq_t + (int64_t)qh * p.sq_h + 8 * hl;
#pragma unroll
        for (int s = 0; s < KS; ++s) {
            qf[s] = Vec16{{0u, 0u, 0u, 0u}};
            if (valid) qf[s] = ld16(qp + 16 * s);
        }
    };
    float m_run, l_run;  // l_run: this lane's half of the keys
    f16v_t oacc[DT];
    auto clear = [&] {
        m_run = -INFINITY, l_run = 0.f;
#pragma unroll
        for (int dt = 0; dt < DT; ++dt)
#pragma unroll
            for (int r = 0; r < 16; ++r) oacc[dt][r] = 0.f;
    };
    load_q();
    clear();
    if (threadIdx.x < 2) flags[threadIdx.x] = 0;  // (ahead of the key loop's first barrier)
    const PromptKeys<T, D> src(p, s0, kvh, qt * kBM, k_first, k_last, smem, flags);
    const bool live = qt * kBM + wave * 32 < rows;
    Tile::template keys<false>(src, smem, qf, live, src.nb, p.scale_log2, m_run, l_run, oacc);

    // Results that are not finite: once more, with a look at V.
    float odd = l_run * 0.f;  // 0, or NaN if anything is not finite
#pragma unroll
    for (int dt = 0; dt < DT; ++dt)
#pragma unroll
        for (int r = 0; r < 16; ++r) odd = __builtin_fmaf(oacc[dt][r], 0.f, odd);
    {
        int tok, qh;
        if (__any(query_of(tok, qh) && odd != 0.f) && lane == 0) flags[1] = 1;
    }
    Tile::sync_lds();
    if (__builtin_expect(__builtin_amdgcn_readfirstlane(flags[1]), 0)) {
        load_q();
        clear();
        Tile::template keys<true>(src, smem, qf, live, src.nb, p.scale_log2, m_run, l_run, oacc);
    }

    const float l_tot = xor32_sum(l_run);  // both halves of the query's keys
    int tok, qh;
    const bool valid = query_of(tok, qh);
    if (CUT && !whole) {
        if (valid) {
            const int64_t r = ((int64_t)slot * p.parts + cut) * kBM + wave * 32 + q32;
            if (hl == 0) {
                p.part_m[r] = m_run * p.scale_log2;
                p.part_l[r] = l_tot;
            }
            Tile::store_state(oacc, p.part_acc + r * D);
        }
        return;
    }
    uint16_t* const orow = p.o + ((int64_t)s0 + tok) * p.so_t + (int64_t)qh * p.so_h;
    float* const lrow = p.lse ? p.lse + ((int64_t)s0 + tok) * p.sl_t + (int64_t)qh * p.sl_h : nullptr;
    Tile::store_row(oacc, 1.f / l_tot, orow, valid);
    if (valid && lrow && hl == 0) *lrow = (m_run * p.scale_log2 + fast_log2(l_tot)) * kLn2;
}

// Joins the parts of cut tiles: a wave per row (token, q head), lanes across the
// head dim.
template <typename T, int D>
__global__ __launch_bounds__(kPromptThreads) void prompt_merge_kernel(PromptParams p, int32_t n_rows) {
    constexpr int E = D / 64 ? D / 64 : 1;  // floats of a lane (D = 32: lanes 0 .. 31)
    constexpr int kBN = DenseTile<T, D>::kBN;
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = blockIdx.x * 4 + wave;
    if (row >= n_rows) return;
    int seq, kvh, qt, slot, rr;  // rr: the row in its (sequence, kv head)
    if (p.tiles) {
        slot = row / kBM;
        if (!numbered_tile(p, slot, seq, kvh, qt)) return;
        rr = qt * kBM + row % kBM;
    } else {
        const int r0 = divide(row, p.hqdiv);
        const int qh = row - r0 * p.Hq;
        seq = divide(r0, p.msdiv);
        kvh = divide(qh, p.gdiv);
        rr = (r0 - seq * p.max_seqlen) * p.group + (qh - kvh * p.group);
        qt = rr / kBM;
        slot = (seq * p.Hkv + kvh) * p.qtiles + qt;
    }
    int32_t s0;
    const int rows = prompt_tokens(p, seq, s0) * p.group;
    if (rr >= rows) return;
    const int tok = divide(rr, p.gdiv), qh = kvh * p.group + (rr - tok * p.group);
    const int k_hi = divide(min(qt * kBM + kBM, rows) - 1, p.gdiv) + 1;
    const int parts = TileParts(p, (k_hi + kBN - 1) / kBN).n;
    if (parts == 1) return;  // finished by its workgroup
    const int64_t first = (int64_t)slot * p.parts * kBM + (rr - qt * kBM);
    const bool in = lane * E < D;
    float m = -INFINITY, l = 0.f, acc[E] = {};
    constexpr int U = 4;
    for (int c = 0; c < parts; c += U) {
        float mi[U], li[U], x[U][E];
#pragma unroll
        for (int u = 0; u < U; ++u) {
            const int64_t r = first + (int64_t)min(c + u, parts - 1) * kBM;
            mi[u] = p.part_m[r];
            li[u] = p.part_l[r];
#pragma unroll
            for (int e = 0; e < E; ++e) x[u][e] = p.part_acc[r * D + (in ? lane * E : 0) + e];
        }
#pragma unroll
        for (int u = 0; u < U; ++u) {
            if (c + u >= parts) break;
            const float mn = fmaxf(m, mi[u]);
            const float mc = mn == -INFINITY ? 0.f : mn;
            const float old = fast_exp2(m - mc), f = fast_exp2(mi[u] - mc);
            l = l * old + f * li[u];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] = acc[e] * old + f * x[u][e];
            m = mn;
        }
    }
    const int64_t t = (int64_t)s0 + tok;
    uint16_t* const o = p.o + t * p.so_t + qh * p.so_h;
    float* const lse = p.lse ? p.lse + t * p.sl_t + qh * p.sl_h : nullptr;
    const float inv = 1.f / l;
#pragma unroll
    for (int e = 0; e < E; ++e) acc[e] = in_range<T>(acc[e] * inv);
    if (in) {
        if constexpr (E == 2)
            *reinterpret_cast<uint32_t*>(o + 2 * lane) = MfmaOps<T>::pack2(acc[0], acc[1]);
        else
            o[lane] = (uint16_t)MfmaOps<T>::pack2(acc[0], 0.f);
    }
    if (lse && lane == 0) *lse = (m + fast_log2(l)) * kLn2;
}

template <typename T, int D>
static int launch_prompt(const PromptParams& p, int64_t blocks, hipStream_t st) {
    if (!p.part) {
        hipLaunchKernelGGL((prompt_attn_kernel<T, D, false>), dim3((uint32_t)blocks), dim3(kPromptThreads), 0, st, p);
        return launch_status("prompt_attn_kernel");
    }
    hipLaunchKernelGGL((prompt_attn_kernel<T, D, true>), dim3((uint32_t)(blocks * p.parts)), dim3(kPromptThreads), 0, st,
                       p);
    const int rc = launch_status("prompt_attn_kernel, cut tiles");
    if (rc) return rc;
    const int64_t rows = p.tiles ? (int64_t)p.tiles * kBM : (int64_t)p.B * p.max_seqlen * p.Hq;
    hipLaunchKernelGGL((prompt_merge_kernel<T, D>), dim3((uint32_t)((rows + 3) / 4)), dim3(kPromptThreads), 0, st, p,
                       (int32_t)rows);
    return launch_status("prompt_merge_kernel");
}

// Tiles of a call, and how they are cut.
struct PromptPlan {
    int32_t max_seqlen, group, qtiles, part, parts;
    int32_t tiles;  // of launches that number them, else 0
    int64_t pairs, slots, m, l, bytes;  // slots: tiles that the launch has a place for;
                                        // workspace: states' maxima at 0, sums at m, numerators at l
    bool fits;
};
static PromptPlan prompt_plan(int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t hq, int32_t hkv,
                              int32_t head_dim) {
    PromptPlan q{};
    q.max_seqlen = (int32_t)std::min<int64_t>(max_seqlen, total_tokens);
    q.group = hq / hkv;
    q.pairs = (int64_t)batch * hkv;
    q.fits = (int64_t)q.max_seqlen * q.group <= INT32_MAX / 2 && q.pairs <= INT32_MAX;
    if (!q.fits || q.max_seqlen <= 0 || q.pairs <= 0) return q;
    q.qtiles = (q.max_seqlen * q.group + kBM - 1) / kBM;
    q.parts = 1;
    q.slots = q.pairs * q.qtiles;
    int64_t full = batch;  // sequences, if all were of the longest one's length
    // Numbering the tiles that there are costs a look through the offsets ahead
    // of everything else; a workgroup without a tile costs 1/3 us of a slot (one
    // prompt of 2048 tokens, 32 / 8 heads, bf16, with 63 of one token: 50 us
    // numbered, 68 with a place for 64 prompts of 2048; with 255: 58 and 145).
    const int64_t numbered = ((total_tokens * q.group + kBM - 1) / kBM + batch) * hkv;
    if (q.slots > 4 * numbered && numbered < INT32_MAX / kBM - 8) {
        q.tiles = (int32_t)((numbered + 7) / 8 * 8);
        q.slots = q.tiles;
        full = std::min<int64_t>(batch, (total_tokens + q.max_seqlen - 1) / q.max_seqlen);
    }
    // Tiles are cut where the longest one alone holds the call up: a CU with one
    // workgroup takes 4/5 of the time per block that it takes with two, and the
    // second kernel and the states cost what about 16 blocks take.  With as many
    // tiles as slots the short ones next to the long ones even the CUs out by
    // themselves (504 tiles of 2000 tokens, 32 / 8 heads, bf16: 46 us whole, 74 cut
    // in two); 63 tiles of 2000 tokens, 4 heads over one: 36.0 us whole, 23.2 in
    // parts; 4000 tokens of those: 66 and 45.
    const int64_t longest = (q.max_seqlen + 63) / 64;
    const int64_t blocks = full * hkv * q.qtiles * (longest + 1) / 2;
    const int64_t share = std::max<int64_t>(8, (blocks + 255) / 256);  // of a CU
    if (longest > share * 5 / 4 + 16) {
        q.part = (int32_t)share;
        q.parts = (int32_t)((longest + share - 1) / share);
        const int64_t rows = q.slots * q.parts * kBM;
        q.m = rows * 4;
        q.l = 2 * rows * 4;
        q.bytes = q.l + rows * head_dim * 4;
        // (a place for every short prompt's tile, too: thousands of them are not
        // worth gigabytes that no one writes)
        if (q.bytes > int64_t(1) << 29) q.part = 0, q.parts = 1, q.bytes = 0;
    }
    return q;
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int64_t qattn_prompt_workspace_bytes(int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t num_q_heads,
                                     int32_t num_kv_heads, int32_t head_dim) {
    if (batch <= 0 || max_seqlen <= 0 || total_tokens <= 0 || num_q_heads <= 0 || num_kv_heads <= 0 || head_dim <= 0 ||
        num_q_heads % num_kv_heads)
        return 0;
    return prompt_plan(batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim).bytes;
}

int qattn_prompt_fwd(const void* q, const int64_t q_stride[3], const void* k, const int64_t k_stride[3],
                     const void* v, const int64_t v_stride[3], void* o, const int64_t o_stride[3], float* lse,
                     const int64_t lse_stride[2], const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen,
                     int64_t total_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                     int32_t dtype, void* workspace, int64_t workspace_size, void* stream) {
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
    const PromptPlan plan = prompt_plan(batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim);
    if (!plan.fits || plan.slots > INT32_MAX ||
        (plan.part && !plan.tiles && (int64_t)batch * plan.max_seqlen * num_q_heads > INT32_MAX)) {
        set_error("sizes too large: max_seqlen=%d group=%d batch=%d num_kv_heads=%d", plan.max_seqlen, plan.group, batch,
                  num_kv_heads);
        return QATTN_ERR_ARG;
    }
    if (plan.bytes && (!workspace || workspace_size < plan.bytes || (uintptr_t)workspace & 255u)) {
        set_error("a 256-byte aligned workspace of %lld bytes needed, %lld given", (long long)plan.bytes,
                  (long long)workspace_size);
        return QATTN_ERR_WORKSPACE;
    }
    p.max_seqlen = plan.max_seqlen;
    p.qtiles = plan.qtiles;
    p.tiles = plan.tiles;
    p.part = plan.part;
    p.parts = plan.parts;
    if (plan.part) {
        p.part_m = (float*)workspace;
        p.part_l = (float*)((char*)workspace + plan.m);
        p.part_acc = (float*)((char*)workspace + plan.l);
        p.partdiv = make_divider(plan.parts);
        p.hqdiv = make_divider(num_q_heads);
        p.msdiv = make_divider(plan.max_seqlen);
    }
    const int64_t pairs = plan.pairs;
    while (pairs << p.spread & 7) ++p.spread;  // lists: a multiple of the 8 XCDs
    p.list = (p.qtiles + (1 << p.spread) - 1) >> p.spread;
    const int64_t blocks = p.tiles ? p.tiles : (pairs << p.spread) * p.list;
    // As many lists side by side as have their K/V in one XCD's L2 (4 MB): the
    // longest tiles of them all start first, and the last ones end together.
    const int64_t kv_bytes = 4 * (int64_t)p.max_seqlen * head_dim;
    p.xcd_lists = (int32_t)((pairs << p.spread) / 8);
    p.group_lists = (int32_t)std::min<int64_t>(p.xcd_lists, std::max<int64_t>(1, (4 << 20) / kv_bytes));
    if (blocks * p.parts > INT32_MAX) {
        set_error("grid too large (%lld blocks)", (long long)blocks);
        return QATTN_ERR_ARG;
    }
    p.gdiv = make_divider(p.group);
    p.groupdiv = make_divider((int32_t)std::min<int64_t>((int64_t)p.group_lists * p.list, INT32_MAX));
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
