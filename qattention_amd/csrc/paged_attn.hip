// paged_attn.hip -- attention of query tokens over their sequence's context in
// a paged K/V cache, with LSE.
//
// Row r of sequence s and kv head g is query token r / group, q head
// g * group + r % group; every row attends keys 0 .. context - 1:
//   o = sum_j softmax_j(scale q.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// in one pass with a running maximum m and sum l.
//
// The work is dealt to workgroups, and cut items are joined, as paged_work.h says.
//
// Two kernels by the longest sequence's rows:
//   up to 32 (paged_attn_kernel): per step a wave forms, for 32 keys of its own,
//     S^T = K Q^T      2 key tiles x D/32 products of v_mfma_f32_16x16x32
//     O^T += V^T P^T   D/16 products
//   with K rows loaded from the cache straight into the A operand's layout and
//   V rows through a wave-private LDS block that the transposing reads
//   (ds_read_b64_tr_b16) take as V^T; S^T has one row (query) per lane column,
//   and its registers are the P^T operand.  The loads of the next step are
//   requested before the products of this one; page numbers one step earlier.
//   more (paged_wide_kernel): tiles of 128 rows share K/V blocks of 64 keys in
//   LDS (dense_tiles.h).
#include "paged_work.h"

namespace qattn {

// Waves per SIMD of the narrow kernel: two, but one with 128-wide heads from 32
// rows on, whose accumulators, K operand and loads in flight take the registers
// of both.
constexpr int narrow_waves(int d, int qb) { return d == 128 && qb > 1 ? 1 : 2; }

// ---------------------------------------------------------------------------
// Few rows (16 QB per tile): bound by reading the cache.  A workgroup's NW waves
// are NW / HW for each of HW kv heads, 32 keys per wave and step; nothing is
// shared between the waves but a head's last join.  Four heads per workgroup
// read 1 KB of each cached token at a time where one head reads 256 bytes: 6.2
// TB/s against 5.6 for the bare loads of 64 x 10240 keys.
// STREAM: runs of units, as above.  Otherwise a workgroup per item, for short
// contexts, where the launch is all latency: no scan ahead of the first load and
// no second kernel (2 x 300 keys, 32 / 8 heads, in a graph: 8.1 us against 11.2 in
// runs, 2 x 500: 9.4 against 11.3).  A workgroup draws about 53 GB/s from far away
// however many loads it has in flight (two steps of them were 3-10% slower than
// one), so a few longer contexts want many CUs: 2 x 700 keys take 12.0 us so and
// 11.3 in runs, 2 x 2000 23.9 and 11.
// ---------------------------------------------------------------------------
constexpr int kNarrowWaves = 4;             // waves of a STREAM workgroup
constexpr int kItemWaves = 8;               // waves of a workgroup per item

template <typename T, int D, int QB, int NW, int HW, bool STREAM>
__global__ __launch_bounds__(64 * NW)
    __attribute__((amdgpu_waves_per_eu(narrow_waves(D, QB)))) void paged_attn_kernel(PagedParams p) {
    constexpr int NC = D / 32;     // k-steps of S^T over the head dim
    constexpr int ND = D / 16;     // d-tiles of O^T
    constexpr int DV = D / 8;      // 16-byte chunks per row
    constexpr int RPI = 512 / D;   // V rows per load instruction of a wave
    constexpr int NV = 32 / RPI;   // V loads per lane and step
    constexpr int WBLK = 32 * D;   // elements of a wave's V block
    constexpr int ROWS = 16 * QB;
    constexpr int WPH = NW / HW;   // waves of a kv head
    constexpr int KEYS = 32 * WPH;  // of a unit
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
        const int seq = sh.seq, tile = part.tile, b0 = part.b0, b1 = part.b1, ctx = sw.ctx;
        const int kvh = part.group * HW + wave / WPH;

        auto query_of = [&](int r, int64_t& qrow, int& qh) {
            const int rr = tile * 16 * QB + r;
            const int tok = divide(rr, p.gdiv);
            qh = kvh * p.group + (rr - tok * p.group);
            qrow = (int64_t)sw.s0 + tok;
            return rr < sw.rows;
        };
        // Q^T operand: dims 32 c + 8 lq .. + 7 of row 16 b + l16
        Vec16 qf[QB][NC];
#pragma unroll
        for (int b = 0; b < QB; ++b) {
            int64_t qrow;
            int qh;
            const bool valid = query_of(16 * b + l16, qrow, qh);
            const uint16_t* qp = p.q + qrow * p.sq_t + qh * p.sq_h + 8 * lq;
#pragma unroll
            for (int c = 0; c < NC; ++c) {
                qf[b][c] = Vec16{{0u, 0u, 0u, 0u}};
                if (valid) qf[b][c] = ld16(qp + 32 * c);
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
        const char* const kb = (const char*)(p.kc + kvh * p.sk_head);
        const char* const vb = (const char*)(p.vc + kvh * p.sv_head);
        const int32_t* const pt = p.table + (int64_t)seq * p.pt_cols;

        // key lane % 32 of step b: its page (asked for without waiting for the
        // context's length), or -1 past the table
        auto key_at = [&](int b) { return KEYS * b + 32 * (wave % WPH) + (lane & 31); };
        auto page_of = [&](int b) {
            const int pos = key_at(b);
            return pos < p.capacity ? pt[divide(pos, p.pdiv)] : -1;
        };
        // the step's loads: K rows in the A operand's layout, V rows by row
        // (load n: row n RPI + lane / DV, chunk lane % DV).  Keys that do not
        // exist read the cache's first row and count for nothing below.
        Vec16 kx[2][NC], vx[NV];
        uint32_t have = 0;  // bit j: key j of the step exists
        auto issue = [&](int b, int page) {
            const int pos = key_at(b);
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages && pos < ctx;
            have = (uint32_t)__ballot(ok);
            const int slot = pos - divide(pos, p.pdiv) * p.page_size;
            // row offsets in 16-byte units (below 2^32: checked on the host)
            const uint32_t ko = ok ? (uint32_t)((page * p.sk_page + slot * p.sk_slot) >> 3) : 0u;
            const uint32_t vo = ok ? (uint32_t)((page * p.sv_page + slot * p.sv_slot) >> 3) : 0u;
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const char* row = kb + 16 * (uint64_t)(uint32_t)__shfl((int)ko, 16 * t + l16) + 16 * lq;
#pragma unroll
                for (int c = 0; c < NC; ++c) kx[t][c] = ld16(row + 64 * c);
            }
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const char* row = vb + 16 * (uint64_t)(uint32_t)__shfl((int)vo, n * RPI + lane / DV);
                vx[n] = ld16(row + 16 * (lane % DV));
            }
        };
        int page = page_of(b0);
        int next = page_of(b0 + 1);
        if (ctx > 0) issue(b0, page);  // (no context: nothing to read, maybe no cache)
        for (int b = b0; b < b1; ++b) {
            // V to LDS; rows of keys that do not exist as zeros (weight 0
            // times what lies there could be NaN)
            const uint32_t mask = have;
#pragma unroll
            for (int n = 0; n < NV; ++n) {
                const int r = n * RPI + lane / DV;
                Vec16 x = vx[n];
                if (mask != 0xffffffffu && !(mask >> r & 1)) x = Vec16{{0u, 0u, 0u, 0u}};
                st16(vblk + r * D + 8 * ((lane % DV) ^ kv_swz(r, DV)), x);
            }
            Vec16 kf[2][NC];
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int c = 0; c < NC; ++c) kf[t][c] = kx[t][c];
            if (b + 1 < b1) {
                page = next;
                next = page_of(b + 2);
                issue(b + 1, page);
            }
            if (mask == 0) continue;  // none of the wave's keys exists
            __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
            __builtin_amdgcn_wave_barrier();
            __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
            Vec16 pf[QB];
            float alpha[QB];
#pragma unroll
            for (int q = 0; q < QB; ++q) {
                f4_t s[2];
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    s[t] = f4_t{0.f, 0.f, 0.f, 0.f};
#pragma unroll
                    for (int c = 0; c < NC; ++c) s[t] = MfmaOps<T>::mma(kf[t][c], qf[q][c], s[t]);
                }
                // lane: keys 16 t + 4 lq + i of row l16
                if (mask != 0xffffffffu) {
#pragma unroll
                    for (int t = 0; t < 2; ++t)
#pragma unroll
                        for (int i = 0; i < 4; ++i)
                            if (!(mask >> (16 * t + 4 * lq + i) & 1)) s[t][i] = -INFINITY;
                }
                float mb = -INFINITY;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) mb = fmaxf(mb, s[t][i]);
                const float m_new = fmaxf(m_run[q], col4_max(mb));
                // (a row of -inf scores alone keeps weights of zero)
                const float mc = m_new == -INFINITY ? 0.f : m_new * p.scale_log2;
                alpha[q] = fast_exp2(__builtin_fmaf(m_run[q], p.scale_log2, -mc));
                float sum = 0.f;
#pragma unroll
                for (int t = 0; t < 2; ++t)
#pragma unroll
                    for (int i = 0; i < 4; ++i) {
                        s[t][i] = fast_exp2(__builtin_fmaf(s[t][i], p.scale_log2, -mc));
                        sum += s[t][i];
                    }
                l_run[q] = l_run[q] * alpha[q] + sum;
                m_run[q] = m_new;
                // P is rounded to the inputs' type for the product (its sum is
                // not): half a step of each weight, as one rounding of the output
#pragma unroll
                for (int t = 0; t < 2; ++t) {
                    pf[q].w[2 * t] = MfmaOps<T>::pack2(s[t][0], s[t][1]);
                    pf[q].w[2 * t + 1] = MfmaOps<T>::pack2(s[t][2], s[t][3]);
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

        join_waves<T, D, QB, NW, HW>(
            p, sh, part, query_of, m_run, l_run, oacc, vlds, ml, [](int ch) { return ch; }, HW * ROWS,
            [&](int r) { return wave / WPH * ROWS + r; });
        __syncthreads();  // the LDS is free for the next item
        sh.u += STREAM ? b1 - b0 : 1;
    }
}

// ---------------------------------------------------------------------------
// Many rows (128 per tile): the key loop of dense_tiles.h, the rows of a K/V
// block found through a table of row offsets in LDS that the workgroup fills
// for kTable blocks at a time.
// ---------------------------------------------------------------------------
constexpr int kWideKeys = 64;
constexpr int kTable = 24;

struct PageTable {
    // per block, row r at (r / 16, r % RPI, r % 16 / RPI): the NI rows that a
    // lane loads lie next to each other
    uint32_t k[kTable][kWideKeys], v[kTable][kWideKeys];  // in 16-byte units
    uint64_t have[kTable];                                // bit r: key r exists
};

template <typename T, int D>
struct PagedKeys {
    using Tile = DenseTile<T, D>;
    static constexpr bool kEveryBlock = true;
    static constexpr int NI = Tile::NI, RPI = Tile::RPI, DV = Tile::DV, BLK = Tile::BLK;
    const PageTable* tab;
    const char *kbase, *vbase;
    int nb;             // blocks in the table
    uint32_t bad;       // blocks with a key that does not exist
    uint32_t colb, lds0, at;
    int wave;

    // Fills the table with blocks b0 .. b0 + n - 1 of the sequence.
    __device__ __forceinline__ PagedKeys(const PagedParams& p, PageTable& t, const int32_t* pages, int ctx, int kvh,
                                         int b0, int n, const uint16_t* smem)
        : tab(&t), nb(n) {
        const int lane = threadIdx.x & 63;
        wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
        kbase = (const char*)(p.kc + (int64_t)kvh * p.sk_head);
        vbase = (const char*)(p.vc + (int64_t)kvh * p.sv_head);
        colb = 16 * ((lane % DV) ^ kv_swz32(wave * NI * RPI + lane / DV, DV));
        at = (wave * RPI + lane / DV) * NI;
        lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) const void*)smem + wave * (NI * 1024);
        const int place = ((lane / 16) * RPI + lane % RPI) * NI + lane % 16 / RPI;
        __syncthreads();  // the table's and the buffers' last readers are done
        for (int i = wave; i < n; i += 4) {
            const int pos = (b0 + i) * kWideKeys + lane;
            int page = -1;
            const int col = divide(pos, p.pdiv);
            if (pos < ctx) page = pages[col];
            const int slot = pos - col * p.page_size;
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages;
            // (keys that do not exist read the cache's first row)
            t.k[i][place] = ok ? (uint32_t)((page * p.sk_page + slot * p.sk_slot) >> 3) : 0u;
            t.v[i][place] = ok ? (uint32_t)((page * p.sv_page + slot * p.sv_slot) >> 3) : 0u;
            const uint64_t have = __ballot(ok);
            if (lane == 0) t.have[i] = have;
        }
        __syncthreads();
        bad = (uint32_t)__ballot(lane < n && t.have[lane < n ? lane : 0] != ~0ull);
    }
    struct Offsets {
        uint32_t x[NI];
    };
    __device__ __forceinline__ Offsets rows(const uint32_t (&tab_)[kTable][kWideKeys], int j) const {
        const uint32_t* r = &tab_[min(j, nb - 1)][at];
        Offsets o;
        if constexpr (NI == 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(r);
            o.x[0] = x.x, o.x[1] = x.y, o.x[2] = x.z, o.x[3] = x.w;
        } else if constexpr (NI == 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(r);
            o.x[0] = x.x, o.x[1] = x.y;
        } else {
            o.x[0] = *r;
        }
        return o;
    }
    static __device__ __forceinline__ void load(const char* base, uint32_t off, uint32_t col, uint32_t lds) {
        const uint64_t a = (uint64_t)(uintptr_t)base + ((uint64_t)off << 4) + col;
        asm volatile("global_load_lds_dwordx4 %0, off" ::"v"(a), "{m0}"(lds) : "memory");
    }
    struct Dma {
        Offsets ko, vo;
        uint32_t col, ld;
        const char *gk, *gv;
        __device__ __forceinline__ void k(int buf, int n) {
            load(gk, ko.x[n], col ^ (16 * kv_swz32(n * RPI, DV)), ld + 2 * buf * BLK + n * 1024);
        }
        __device__ __forceinline__ void v(int buf, int n) {
            load(gv, vo.x[n], col ^ (16 * kv_swz32(n * RPI, DV)), ld + 2 * (2 + buf) * BLK + n * 1024);
        }
    };
    __device__ __forceinline__ Dma dma(int j) const {
        Dma d{rows(tab->k, j + 3), rows(tab->v, j + 1), colb, lds0, kbase, vbase};
        asm volatile("" : "+v"(d.col), "+s"(d.ld));
        return d;
    }
    __device__ __forceinline__ void load_k(int j, uint16_t* buf) const {
        const Offsets o = rows(tab->k, j);
#pragma unroll
        for (int n = 0; n < NI; ++n)
            load(kbase, o.x[n], colb ^ (16 * kv_swz32(n * RPI, DV)),
                 (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)(buf + (wave * NI + n) * 512));
    }
    __device__ __forceinline__ void load_v(int j, uint16_t* buf) const {
        const Offsets o = rows(tab->v, j);
#pragma unroll
        for (int n = 0; n < NI; ++n)
            load(vbase, o.x[n], colb ^ (16 * kv_swz32(n * RPI, DV)),
                 (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)(buf + (wave * NI + n) * 512));
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
    __device__ __forceinline__ void clean(int j, uint16_t* v, O&...) const {
        if (__builtin_expect(bad >> j & 1, 0)) {
            const uint64_t have = tab->have[j];
            for (int i = threadIdx.x; i < kWideKeys * DV; i += Tile::kThreads)
                if (!(have >> (i / DV) & 1)) st16(v + 8 * i, Vec16{{0u, 0u, 0u, 0u}});
            Tile::template publish<0>();
        }
    }
};

template <typename T, int D>
__global__ __launch_bounds__(kPagedThreads) __attribute__((amdgpu_waves_per_eu(2, 2))) void paged_wide_kernel(
    PagedParams p) {
    using Tile = DenseTile<T, D>;
    constexpr int KS = Tile::KS, DT = Tile::DT, ROWS = Tile::kBM;
    __shared__ __attribute__((aligned(1024))) uint16_t smem[Tile::kSmem];
    __shared__ __attribute__((aligned(16))) PageTable table;

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
        Vec16 qf[KS];
        {
            int64_t qrow;
            int qh;
            const bool valid = query_of(qrow, qh);
            const uint16_t* qp = p.q + qrow * p.sq_t + qh * p.sq_h + 8 * hl;
#pragma unroll
            for (int s = 0; s < KS; ++s) {
                qf[s] = Vec16{{0u, 0u, 0u, 0u}};
                if (valid) qf[s] = ld16(qp + 16 * s);
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
            const PagedKeys<T, D> src(p, table, p.table + (int64_t)sh.seq * p.pt_cols, sw.ctx, part.group, b,
                                      min(kTable, part.b1 - b), smem);
            Tile::template keys<false>(src, smem, qf, live, src.nb, p.scale_log2, m_run, l_run, oacc);
        }
        const float l = xor32_sum(l_run);
        int64_t qrow;
        int qh;
        const bool valid = query_of(qrow, qh);
        if (part.whole) {
            const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
            Tile::store_row(oacc, inv, p.o + qrow * p.so_t + qh * p.so_h, valid);
            if (valid && p.lse && hl == 0)
                p.lse[qrow * p.sl_t + qh * p.sl_h] = (m_run * p.scale_log2 + fast_log2(l)) * kLn2;
        } else if (valid) {
            const int64_t r = part_slot(sh) * ROWS + wave * 32 + q32;
            if (hl == 0) {
                p.part_m[r] = m_run * p.scale_log2;
                p.part_l[r] = l;
            }
            Tile::store_state(oacc, p.part_acc + r * D);
        }
        sh.u += part.b1 - part.b0;
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
static PagedShape paged_shape(int64_t max_rows, int64_t pairs, int hkv, int64_t capacity, int head_dim) {
    // A workgroup per item, where every one runs at once: two steps at most, or
    // four where the items fill half the chip by themselves (replays of a graph,
    // 128-wide heads, 8 kv heads, against runs: 2 x 500 keys 9.4 us and 11.3, 2 x 700
    // 12.0 and 11.3, 4 x 700 12.2 and 11.8, 8 x 700 15.6 and 15.5, 16 x 700 17.8 and
    // 20.9, 32 x 700 21.8 and 28.0, 8 x 1000 20.3 and 16.9, 16 x 1024 23.2 and 23.4,
    // 32 x 1024 29.5 and 35.6; eager calls give runs half a us more.  Longer ones
    // gain 5 us of 40 with equal contexts, and lose as much where they differ by a
    // factor of three, which runs even out).  The lengths stay on the device, so
    // capacity, what the table has columns for, stands for them: 2 x 300 keys take
    // 10.8 us with a table four times as wide, 12.5 with one of 32 times, 32 x 1024
    // 34.6 with either, 64 x 500 34.2 against 32.6.
    const int steps = pairs >= 128 ? 4 : 2;
    if (max_rows <= 16 && capacity <= steps * 32 * kItemWaves && pairs <= 256) return {1, 4, 8, 1, 1, true};
    if (max_rows <= 32) {
        const int qb = max_rows <= 16 ? 1 : 2;
        const int per_cu = narrow_waves(head_dim, qb);
        // Several kv heads per workgroup where the reading is most of the time:
        // few rows, at least 16 steps per workgroup and no more than 16 parts
        // per row, since each part leaves a state per head (64 x 8000 keys: 380 us
        // with one head, 363 with four; 8 x 3000 keys, 32 rows: 27.1 against 36.6).
        int heads = hkv % 4 == 0 ? 4 : hkv % 2 == 0 ? 2 : 1;
        const int64_t work = pairs * (((int64_t)capacity + 127) / 128);
        if (max_rows > 8 || pairs / heads * 16 < 256 * per_cu || work < 16 * 256 * per_cu) heads = 1;
        return {qb, qb == 1 ? 4 : 5, heads == 4 ? 5 : heads == 2 ? 6 : 7, heads, per_cu, false};
    }
    return {0, 7, 6, 1, 2, false};
}

template <typename T, int D>
static int launch_paged(const PagedParams& p, const PagedShape& sh, hipStream_t st) {
    const dim3 grid(p.nwg), block(kPagedThreads);
    if (sh.items) {
        hipLaunchKernelGGL((paged_attn_kernel<T, D, 1, kItemWaves, 1, false>), dim3((uint32_t)(p.B * p.tiles * p.Hkv)),
                           dim3(64 * kItemWaves), 0, st, p);
        return launch_status("paged_attn_kernel, a workgroup per item");
    }
#define QATTN_NARROW(QB, HW) hipLaunchKernelGGL((paged_attn_kernel<T, D, QB, kNarrowWaves, HW, true>), grid, block, 0, st, p)
    switch (8 * sh.qb + sh.heads) {
        case 8 + 1: QATTN_NARROW(1, 1); break;
        case 8 + 2: QATTN_NARROW(1, 2); break;
        case 8 + 4: QATTN_NARROW(1, 4); break;
        case 16 + 1: QATTN_NARROW(2, 1); break;
        default: hipLaunchKernelGGL((paged_wide_kernel<T, D>), grid, block, 0, st, p);
    }
#undef QATTN_NARROW
    const int rc = launch_status(sh.qb ? "paged_attn_kernel" : "paged_wide_kernel");
    return rc ? rc : launch_merge<T, D>(p, st);
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int64_t qattn_prefix_paged_workspace_bytes(int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int32_t pt_cols, int32_t page_size) {
    return paged_workspace(paged_shape, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim, pt_cols,
                           page_size);
}

int qattn_prefix_paged_fwd(const void* q, const int64_t q_stride[3], const void* k_cache, const int64_t k_stride[4],
                           const void* v_cache, const int64_t v_stride[4], const int32_t* page_table,
                           int32_t pt_cols, int32_t num_pages, int32_t page_size, const int32_t* context_lens,
                           void* o, const int64_t o_stride[3], float* lse, const int64_t lse_stride[2],
                           const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale, int32_t dtype,
                           void* workspace, int64_t workspace_size, void* stream) {
    clear_error();
    PagedParams p{};
    PagedPlan plan;
    const int rc = paged_setup(p, plan, paged_shape, q, q_stride, k_cache, k_stride, v_cache, v_stride, page_table,
                               pt_cols, num_pages, page_size, context_lens, o, o_stride, lse, lse_stride, cu_seqlens,
                               batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim, scale, dtype,
                               workspace, workspace_size);
    if (rc || plan.nothing) return rc;
    hipStream_t st = (hipStream_t)stream;
    if (dtype == QATTN_DTYPE_F16)
        return head_dim == 32   ? launch_paged<F16, 32>(p, plan.shape, st)
               : head_dim == 64 ? launch_paged<F16, 64>(p, plan.shape, st)
                                : launch_paged<F16, 128>(p, plan.shape, st);
    return head_dim == 32   ? launch_paged<BF16, 32>(p, plan.shape, st)
           : head_dim == 64 ? launch_paged<BF16, 64>(p, plan.shape, st)
                            : launch_paged<BF16, 128>(p, plan.shape, st);
}

}  // extern "C"
