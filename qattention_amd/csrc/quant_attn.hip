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
    int64_t ss_page, ss_slot, ss_head;   // bytes
};

// N words at p (aligned to their size, up to 16 bytes).
template <int N>
__device__ __forceinline__ void ld_words(uint32_t (&w)[N], const char* p) {
    if constexpr (N == 1) {
        w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else if constexpr (N == 2) {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        w[0] = x.x, w[1] = x.y;
    } else {
#pragma unroll
        for (int i = 0; i < N; i += 4) {
            const Vec16 x = ld16(p + 4 * i);
#pragma unroll
            for (int j = 0; j < 4; ++j) w[i + j] = x.w[j];
        }
    }
}

// One head's N scales at p, one byte each.
template <int N>
__device__ __forceinline__ uint32_t ld_scales(const char* p) {
    if constexpr (N == 4) return *reinterpret_cast<const uint32_t*>(p);
    else if constexpr (N == 2) return *reinterpret_cast<const uint16_t*>(p);
    else return *reinterpret_cast<const uint8_t*>(p);
}

// ---------------------------------------------------------------------------
// Few rows (16 QB per tile).  The waves' split, the products and the softmax are
// the 16-bit kernel's: per step a wave forms S^T = K Q^T and O^T += V^T P^T for 32
// keys of its own.  What differs is the way in:
//   K  A lane's operand words are a quarter of a key row, contiguous: lane (l16, lq)
//      takes dims D/4 lq .. of key l16, k-step c the 8 from D/4 lq + 8 c on (Q^T is
//      read in that order, which is free), so a quarter has one scale.
//   V  A lane widens 16 (or 8) bytes of a row and stores them to the wave's LDS block
//      as 16-byte chunks; chunk i of lane part ch lies at place i LPR + ch, so that
//      the lanes of a row write side by side.  O's columns come out in that order and
//      are put back where they are stored.
//   scales  One load per step: lane j that of K's key j (j < 32) or V's key j - 32;
//      lane exchanges hand them out.
// ---------------------------------------------------------------------------
constexpr int kNarrowWaves = 4;             // waves of a STREAM workgroup
constexpr int kItemWaves = 8;               // waves of a workgroup per item

constexpr int quant_waves(int d, int qb) { return d == 128 ? (qb > 1 ? 2 : 3) : 4; }

template <typename T, int D, int BITS, int QB, int NW, int HW, bool STREAM>
__global__ __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(quant_waves(D, QB)))) void quant_attn_kernel(QuantParams p) {
    constexpr int NC = D / 32;              // k-steps of S^T over the head dim
    constexpr int ND = D / 16;              // d-tiles of O^T
    constexpr int DV = D / 8;               // 16-byte chunks per widened row
    constexpr int NS = D / kQuantBlock;     // scales per row
    constexpr int KW = D * BITS / 128;      // words of a quarter row
    constexpr int RB = D * BITS / 8;        // bytes of a row
    constexpr int VB = RB / 2 < 16 ? RB / 2 : 16;  // bytes of V per lane and load
    constexpr int LPR = RB / VB;            // lanes per V row
    constexpr int RPI = 64 / LPR;           // V rows per load
    constexpr int NV = 32 / RPI;            // V loads per lane and step
    constexpr int SUB = VB / BITS;          // chunks of 8 elements per load
    constexpr int WBLK = 32 * D;            // elements of a wave's V block
    constexpr int ROWS = 16 * QB;
    constexpr int WPH = NW / HW;            // waves of a kv head
    constexpr int KEYS = 32 * WPH;          // of a unit
    static_assert(LPR * SUB == DV && NV * RPI == 32 && NC * BITS / 4 == KW, "a step is 32 rows");
    // The waves' V blocks; after the key loop, the waves' numerators of one
    // row block (NW x 16 rows x D floats, the same size).
    __shared__ __attribute__((aligned(1024))) uint16_t vlds[NW * WBLK];
    __shared__ float ml[2][NW][ROWS];

    Share sh{};
    if constexpr (STREAM) {
        if (!find_share(p, sh)) return;
    } else {
        sh.end = 1;  // one part: the item
    }
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int l16 = lane & 15, lq = lane >> 4;

    // wave-private V block: chunk c of row r at c ^ kv_swz(r)
    uint16_t* const vblk = vlds + wave * WBLK;
    const int vr = 4 * lq + (l16 >> 2);
    const int vaddr0 = vr * D + 8 * (((l16 & 3) >> 1) ^ kv_swz(vr, DV)) + 4 * (l16 & 1);
    const int kshift = 8 * (lq * NS / 4);                               // the lane's scale in a word of them
    const int vshift = 8 * ((lane % LPR) * (VB * 8 / BITS) / kQuantBlock);

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
        const int kvh = part.group * HW + wave / WPH;

        auto query_of = [&](int r, int64_t& qrow, int& qh) {
            const int rr = tile * 16 * QB + r;
            const int tok = divide(rr, p.gdiv);
            qh = kvh * p.group + (rr - tok * p.group);
            qrow = (int64_t)sw.s0 + tok;
            return rr < sw.rows;
        };
        // Q^T operand of k-step c: dims D/4 lq + 8 c .. + 7 of row 16 b + l16
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
        f4_t oacc[QB][ND];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            m_run[b] = -INFINITY;
            l_run[b] = 0.f;
#pragma unroll
            for (int i = 0; i < ND; ++i) oacc[b][i] = f4_t{0.f, 0.f, 0.f, 0.f};
        }
        const char* const kb = (const char*)(p.kc + kvh * p.sk_head) + 4 * KW * lq;
        const char* const vb = (const char*)(p.vc + kvh * p.sk_head) + VB * (lane % LPR);
        const char* const sb = (const char*)(lane < 32 ? p.ks : p.vs) + kvh * p.ss_head;
        const int32_t* const pt = p.table + (int64_t)sh.seq * p.pt_cols;

        // key lane % 32 of step b: its page (asked for without waiting for the
        // context's length), or -1 past the table
        auto key_at = [&](int b) { return KEYS * b + 32 * (wave % WPH) + (lane & 31); };
        auto page_of = [&](int b) {
            const int pos = key_at(b);
            return pos < p.capacity ? pt[divide(pos, p.pdiv)] : -1;
        };
        // the step's loads.  Keys that do not exist read the cache's first row and
        // count for nothing below.
        uint32_t kx[2][KW], vx[NV][VB / 4], sx = 0;
        uint32_t have = 0;  // bit j: key j of the step exists
        auto issue = [&](int b, int page) {
            const int pos = key_at(b);
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages && pos < ctx;
            have = (uint32_t)__ballot(ok);
            const int slot = pos - divide(pos, p.pdiv) * p.page_size;
            // row offsets in 16-byte units, scales in rows of them (below 2^32:
            // checked on the host)
            const uint32_t off = ok ? (uint32_t)((page * p.sk_page + slot * p.sk_slot) >> 3) : 0u;
            const uint32_t so = ok ? (uint32_t)((uint64_t)(page * p.ss_page + slot * p.ss_slot) / NS) : 0u;
            sx = ld_scales<NS>(sb + NS * (uint64_t)so);
#pragma unroll
            for (int t = 0; t < 2; ++t)
                ld_words(kx[t], kb + 16 * (uint64_t)(uint32_t)__shfl((int)off, 16 * t + l16));
#pragma unroll
            for (int n = 0; n < NV; ++n)
                ld_words(vx[n], vb + 16 * (uint64_t)(uint32_t)__shfl((int)off, n * RPI + lane / LPR));
        };
        int page = page_of(b0);
        int next = page_of(b0 + 1);
        if (ctx > 0) issue(b0, page);  // (no context: nothing to read, maybe no cache)
        for (int b = b0; b < b1; ++b) {
            const uint32_t mask = have, scales = sx;
            auto scale_at = [&](int from, int shift) {
                return scale_of((uint32_t)__shfl((int)scales, from) >> shift & 255u);
            };
            // V to LDS; rows of keys that do not exist as zeros (weight 0
            // times what lies there could be NaN)
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int r = n * RPI + lane / LPR;
                float s = scale_at(32 + r, vshift);
                if (mask != 0xffffffffu && !(mask >> r & 1)) {
                    s = 1.f;
#pragma unroll
                    for (int i = 0; i < VB / 4; ++i) vx[n][i] = 0;
                }
#pragma unroll
                for (int i = 0; i < SUB; ++i)
                    st16(vblk + r * D + 8 * ((i * LPR + lane % LPR) ^ kv_swz(r, DV)),
                         widen8<T, BITS>(vx[n] + i * (BITS / 4), s));
            }
            uint32_t kf[2][KW];
            float kscale[2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                kscale[t] = scale_at(16 * t + l16, kshift);
#pragma unroll
                for (int i = 0; i < KW; ++i) kf[t][i] = kx[t][i];
            }
            if (b + 1 < b1) {
                page = next;
                next = page_of(b + 2);
                issue(b + 1, page);
            }
            if (mask == 0) continue;  // none of the wave's keys exists
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            f4_t s[QB][2];
#pragma unroll
            for (int t = 0; t < 2; ++t) {
#pragma unroll
                for (int q = 0; q < QB; ++q) s[q][t] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int c = 0; c < NC; ++c) {
                    const Vec16 k = widen8<T, BITS>(kf[t] + c * (BITS / 4), kscale[t]);
#pragma unroll
                    for (int q = 0; q < QB; ++q) s[q][t] = MfmaOps<T>::mma(k, qf[q][c], s[q][t]);
                }
            }
            Vec16 pf[QB];
            float alpha[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                // lane: keys 16 t + 4 lq + i of row l16
                if (mask != 0xffffffffu) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(mask >> (16 * t + 4 * lq + i) & 1)) s[q][t][i] = -INFINITY;
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
                for (int q = 0; q < QB; ++q)
#pragma unroll
                    for (int dt = 0; dt < ND; ++dt) oacc[q][dt] *= alpha[q];
            }
#pragma unroll
            for (int dt = 0; dt < ND; ++dt) {
                typedef short v4s __attribute__((ext_vector_type(4)));
                typedef __attribute__((address_space(3))) v4s* lds_v4s;
                uint16_t* a = vblk + (vaddr0 ^ (16 * dt));
                const v4s lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)a);
                const v4s hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_v4s)(a + 16 * D));
                const uint2 l2 = __builtin_bit_cast(uint2, lo), h2 = __builtin_bit_cast(uint2, hi);
                const Vec16 va{{l2.x, l2.y, h2.x, h2.y}};
#pragma unroll
                for (int q = 0; q < QB; ++q) oacc[q][dt] = MfmaOps<T>::mma(va, pf[q], oacc[q][dt]);
            }
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();  // the block's reads come before the next step's writes
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        }
        join_waves<T, D, QB, NW, HW>(p, sh, part, query_of, m_run, l_run, oacc, vlds, ml,
                                     [](int ch) { return ch % LPR * SUB + ch / LPR; });
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
// ---------------------------------------------------------------------------
constexpr int kWideKeys = 64;
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
        lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)smem;
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
            t.row[i][lane] = ok ? (uint32_t)((page * p.sk_page + slot * p.sk_slot) >> 3) : 0u;
            t.scale[i][lane] = ok ? (uint32_t)((uint64_t)(page * p.ss_page + slot * p.ss_slot) / NS) : 0u;
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
    // Piece n of block j's quarter to the buffer at dst.  A key that does not exist
    // is zeros.
    __device__ __forceinline__ void store(int j, int n, const uint32_t (&r)[KW], uint32_t c, uint32_t dst) const {
        uint32_t w[W];
        float s = scale_of(c);
#pragma unroll
        for (int i = 0; i < W; ++i) w[i] = r[n * W + i];
        const int b = min(j, nb - 1);
        if (__builtin_expect(bad >> b & 1, 0)) {
            if (!(tab->have[b] >> row & 1)) {
                s = 1.f;
#pragma unroll
                for (int i = 0; i < W; ++i) w[i] = 0;
            }
        }
        typedef uint32_t v4u __attribute__((ext_vector_type(4)));
        const Vec16 x = widen8<T, BITS>(w, s);
        *(__attribute__((address_space(3))) v4u*)(uintptr_t)(dst + (put ^ (64 * n))) = v4u{x.w[0], x.w[1], x.w[2], x.w[3]};
    }
    struct Dma {
        const QuantKeys& src;
        int j;
        __device__ __forceinline__ void k(int buf, int n) {
            src.store(j + 3, n, src.rk, src.ck, src.lds0 + 2 * buf * BLK);
            if (n == NI - 1) src.fetch(j + 4, src.kbase, src.ksbase, src.rk, src.ck);
        }
        __device__ __forceinline__ void v(int buf, int n) {
            src.store(j + 1, n, src.rv, src.cv, src.lds0 + 2 * (2 + buf) * BLK);
            if (n == NI - 1) src.fetch(j + 2, src.vbase, src.vsbase, src.rv, src.cv);
        }
    };
    __device__ __forceinline__ Dma dma(int j) const { return Dma{*this, j}; }
    static __device__ __forceinline__ uint32_t lds_of(const uint16_t* buf) {
        return (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)buf;
    }
    // Blocks 0 to 2, before the loop.
    __device__ __forceinline__ void load_k(int j, uint16_t* buf) const {
#pragma unroll
        for (int n = 0; n < NI; ++n) {
            if (j == 1) store(1, n, r1, c1, lds_of(buf));
            else store(j, n, rk, ck, lds_of(buf));
        }
        if (j == 0) fetch(2, kbase, ksbase, rk, ck);
        if (j == 2) fetch(3, kbase, ksbase, rk, ck);
    }
    __device__ __forceinline__ void load_v(int j, uint16_t* buf) const {
#pragma unroll
        for (int n = 0; n < NI; ++n) store(j, n, rv, cv, lds_of(buf));
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
// Host side
// ---------------------------------------------------------------------------
static PagedShape quant_shape(int64_t max_rows, int64_t pairs, int hkv, int64_t capacity, int head_dim) {
    const int steps = pairs >= 128 ? 4 : 2;
    if (max_rows <= 16 && capacity <= steps * 32 * kItemWaves && pairs <= 256) return {1, 4, 8, 1, 1, true};
    if (max_rows <= 32) {
        const int qb = max_rows <= 16 ? 1 : 2;
        const int per_cu = quant_waves(head_dim, qb);
        int heads = hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;
        const int64_t work = pairs * ((capacity + 127) / 128);
        if (max_rows > 8 || pairs / heads * 16 < 256 * per_cu || work < 16 * 256 * per_cu) heads = 1;
        return {qb, qb == 1 ? 4 : 5, heads == 4 ? 5 : heads == 2 ? 6 : 7, heads, per_cu, false};
    }
    return {0, 7, 6, 1, 2, false};
}

template <typename T, int D, int BITS>
static int launch_quant(const QuantParams& p, const PagedShape& sh, hipStream_t st) {
    const dim3 grid(p.nwg), block(kPagedThreads);
    if (sh.items) {
        hipLaunchKernelGGL((quant_attn_kernel<T, D, BITS, 1, kItemWaves, 1, false>),
                           dim3((uint32_t)(p.B * p.tiles * p.Hkv)), dim3(64 * kItemWaves), 0, st, p);
        return launch_status("quant_attn_kernel, a workgroup per item");
    }
#define QATTN_NARROW(QB, HW) \
    hipLaunchKernelGGL((quant_attn_kernel<T, D, BITS, QB, kNarrowWaves, HW, true>), grid, block, 0, st, p)
    switch (8 * sh.qb + sh.heads) {
        case 8 + 1: QATTN_NARROW(1, 1); break;
        case 8 + 2: QATTN_NARROW(1, 2); break;
        case 8 + 4: QATTN_NARROW(1, 4); break;
        case 16 + 1: QATTN_NARROW(2, 1); break;
        default: hipLaunchKernelGGL((quant_wide_kernel<T, D, BITS>), grid, block, 0, st, p);
    }
#undef QATTN_NARROW
    const int rc = launch_status(sh.qb ? "quant_attn_kernel" : "quant_wide_kernel");
    return rc ? rc : launch_merge<T, D>(p, st);
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
                                           int32_t pt_cols, int32_t page_size) {
    return paged_workspace(quant_shape, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim, pt_cols,
                           page_size);
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
    rc = paged_setup(p, plan, quant_shape, q, q_stride, k_cache, half, v_cache, half, page_table, pt_cols, num_pages,
                     page_size, context_lens, o, o_stride, lse, lse_stride, cu_seqlens, batch, max_seqlen,
                     total_tokens, num_q_heads, num_kv_heads, head_dim, scale, dtype, workspace, workspace_size);
    if (rc || plan.nothing) return rc;
    const int64_t unit = head_dim / kQuantBlock;
    const int64_t* ss = scale_stride;
    // a row's scales are found by a 32-bit offset in rows of them
    if (pt_cols > 0 && num_pages > 0 &&
        (ss[0] < 0 || ss[1] < 0 || ss[0] > (int64_t(1) << 40) || ss[1] > (int64_t(1) << 32) ||
         (double)(num_pages - 1) * (ss[0] / unit) + (double)(page_size - 1) * (ss[1] / unit) >= 4294967296.0)) {
        set_error("scale strides must be non-negative and a cache's scales span less than 2^32 rows");
        return QATTN_ERR_LAYOUT;
    }
    p.ks = (const uint8_t*)k_scale, p.vs = (const uint8_t*)v_scale;
    p.ss_page = ss[0], p.ss_slot = ss[1], p.ss_head = ss[2];
    hipStream_t st = (hipStream_t)stream;
    if (dtype == QATTN_DTYPE_F16)
        return bits == 4 ? launch_quant<F16, 4>(p, plan.shape, head_dim, st)
                         : launch_quant<F16, 8>(p, plan.shape, head_dim, st);
    return bits == 4 ? launch_quant<BF16, 4>(p, plan.shape, head_dim, st)
                     : launch_quant<BF16, 8>(p, plan.shape, head_dim, st);
}

}  // extern "C"
