// paged_attn.hip -- attention of query tokens over their sequence's context in
// a paged K/V cache, with LSE.
//
// Row r of sequence s and kv head g is query token r / group, q head
// g * group + r % group; every row attends keys 0 .. context - 1:
//   o = sum_j softmax_j(scale q.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// in one pass with a running maximum m and sum l.
//
// Work: units of 32 to 128 keys of one (sequence, kv heads, row tile), numbered
// sequence by sequence, heads, tiles and keys innermost.  The workgroups of the
// launch take equal runs of all units, whatever the contexts' lengths (no host
// knows them: the lengths stay on the device), so a run may end inside an item.
// A run's whole items are finished in the workgroup; of a cut item every part
// leaves its state (m, l, numerator, fp32) in the workspace and
// paged_merge_kernel joins them in key order, without atomics: results do not
// depend on timing.
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
#include <algorithm>

#include "dense_tiles.h"
#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kPagedThreads = 256;

// Waves per SIMD of the narrow kernel: two, but one with 128-wide heads from 32
// rows on, whose accumulators, K operand and loads in flight take the registers
// of both.
constexpr int narrow_waves(int d, int qb) { return d == 128 && qb > 1 ? 1 : 2; }

struct PagedParams {
    const uint16_t* q;
    const uint16_t* kc;
    const uint16_t* vc;
    uint16_t* o;
    float* lse;
    const int32_t* cu;     // null: row s belongs to sequence s
    const int32_t* table;  // [B, pt_cols]
    const int32_t* ctx;    // [B]
    int64_t sq_t, sq_h, so_t, so_h, sl_t, sl_h;
    int64_t sk_page, sk_slot, sk_head, sv_page, sv_slot, sv_head;
    int64_t total_tokens;
    int32_t B, Hq, Hkv, group, max_seqlen;
    int32_t pt_cols, num_pages, page_size, capacity;
    int32_t nwg;          // workgroups that share the units (a multiple of 8)
    int32_t least;        // units that are worth a workgroup
    int32_t tiles;        // tiles of the longest sequence (a workgroup per item)
    Divider pdiv, gdiv;   // page_size, group
    // kv heads of a workgroup and groups of them; log2 of the rows of a tile and
    // of the keys of a unit (of one kv head)
    int32_t heads, head_shift, groups, row_shift, key_shift;
    Divider groupdiv, tilediv;  // groups, tiles
    float scale_log2;
    // what the merge needs of the work's order, written by the main kernel:
    // the first unit of each sequence [B + 1], or (cuts not null) the item that
    // each run's first unit lies in
    int32_t* base;
    struct RunStart* cuts;  // [nwg]
    float* part_m;        // [nwg][2][heads][rows of a tile], in log2 units
    float* part_l;
    float* part_acc;      // [nwg][2][heads][rows of a tile][D]
};

// Rows and blocks of a sequence; unit (group of kv heads, tile, block) of it is
// number (group * tiles + tile) * blocks + block.
struct SeqWork {
    int32_t s0, rows, tiles, ctx, blocks;
    __device__ __forceinline__ int32_t units(int groups) const { return groups * tiles * blocks; }
};
__device__ __forceinline__ SeqWork seq_work(const PagedParams& p, int s) {
    SeqWork w;
    w.s0 = p.cu ? p.cu[s] : s;
    const int32_t s1 = p.cu ? p.cu[s + 1] : s + 1;
    int32_t n = s1 - w.s0;
    if (w.s0 < 0 || s1 < w.s0 || (int64_t)s1 > p.total_tokens) n = 0;
    n = min(n, p.max_seqlen);
    w.rows = n * p.group;
    w.tiles = (w.rows + (1 << p.row_shift) - 1) >> p.row_shift;
    w.ctx = max(0, min(p.ctx[s], p.capacity));
    // (rows without a context are a block without keys: 0 and -inf)
    w.blocks = max(1, (w.ctx + (1 << p.key_shift) - 1) >> p.key_shift);
    return w;
}

// The item that a run starts in; b0: the blocks of it that runs before hold.
struct RunStart {
    int32_t s0, rows, tile, group, b0, blocks, first, total;  // first: the item's first unit
};

// Equal runs of the units: run w starts at first(w).  (The host checks that
// the units of the longest contexts stay below 2^31.)
struct Runs {
    int32_t n, q, rem;
    __device__ __forceinline__ Runs(int32_t total, int nwg, int least) {
        n = max(1, min(nwg, total / least));
        q = (int32_t)((uint32_t)total / (uint32_t)n);
        rem = total - q * n;
    }
    __device__ __forceinline__ int32_t first(int w) const { return w * q + min(w, rem); }
    __device__ __forceinline__ int of(int32_t unit) const {
        const int32_t big = rem * (q + 1);
        return unit < big ? (int)((uint32_t)unit / (uint32_t)(q + 1)) : rem + (int)((uint32_t)(unit - big) / (uint32_t)q);
    }
};

// This workgroup's run [u, end): the sequence that holds u and its first unit.
// Workgroup 0 leaves the sequences' first units to the merge.  Every thread
// calls it; false: no unit.
struct Share {
    int32_t u, end, start, seq, seq_base, total;
    SeqWork sw;  // of seq
};
__device__ __forceinline__ bool no_share(const PagedParams& p, int wg) {
    if (p.cuts && threadIdx.x == 0) p.cuts[wg] = RunStart{};
    return false;
}
__device__ __forceinline__ bool find_share(const PagedParams& p, Share& sh) {
    __shared__ int32_t sums[4];
    __shared__ int32_t found[2];
    __shared__ SeqWork found_work;
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    // consecutive runs on one XCD: tiles of one item share its L2
    const int per = gridDim.x >> 3;
    const int wg = (blockIdx.x & 7) * per + (blockIdx.x >> 3);
    if (p.B <= 64) {
        // every wave for itself: a sequence per lane, no barrier ahead of the
        // first load (1 x 1000 keys, both kernels in a graph: 10.4 -> 10.1 us)
        SeqWork work{};
        if (lane < p.B) work = seq_work(p, lane);
        const int32_t mine = lane < p.B ? work.units(p.groups) : 0;
        int32_t inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t up = __shfl_up(inc, d);
            if (lane >= d) inc += up;
        }
        const int32_t total = __builtin_amdgcn_readlane(inc, 63);
        if (wg == 0 && wave == 0) {
            if (lane < p.B) p.base[lane] = inc - mine;
            if (lane == 0) p.base[p.B] = total;
        }
        const Runs runs(total, p.nwg, p.least);
        if (wg >= runs.n || total == 0) return no_share(p, wg);
        sh.u = sh.start = runs.first(wg);
        sh.end = runs.first(wg + 1);
        sh.total = total;
        const int at = __builtin_ctzll(__ballot(sh.u < inc));  // the first sequence that ends past u
        sh.seq = at;
        sh.seq_base = __builtin_amdgcn_readlane(inc - mine, at);
        sh.sw.s0 = __builtin_amdgcn_readlane(work.s0, at);
        sh.sw.rows = __builtin_amdgcn_readlane(work.rows, at);
        sh.sw.tiles = __builtin_amdgcn_readlane(work.tiles, at);
        sh.sw.ctx = __builtin_amdgcn_readlane(work.ctx, at);
        sh.sw.blocks = __builtin_amdgcn_readlane(work.blocks, at);
        return true;
    }
    // exclusive prefix of `mine` over the workgroup, and the sum
    auto scan = [&](int32_t mine, int32_t& sum) {
        int32_t inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int32_t up = __shfl_up(inc, d);
            if (lane >= d) inc += up;
        }
        __syncthreads();
        if (lane == 63) sums[wave] = inc;
        __syncthreads();
        int32_t before = 0;
        sum = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            before += w < wave ? sums[w] : 0;
            sum += sums[w];
        }
        return before + inc - mine;
    };
    int32_t total = 0, mine = 0, excl = 0;
    SeqWork work{};
    for (int c = 0; c < p.B; c += kPagedThreads) {
        int32_t sum;
        if (c + tid < p.B) work = seq_work(p, c + tid);
        mine = c + tid < p.B ? work.units(p.groups) : 0;
        excl = total + scan(mine, sum);
        if (wg == 0 && c + tid < p.B) p.base[c + tid] = excl;
        total += sum;
    }
    total = __builtin_amdgcn_readfirstlane(total);  // (what follows from it stays in scalar registers)
    if (wg == 0 && tid == 0) p.base[p.B] = total;
    const Runs runs(total, p.nwg, p.least);
    if (wg >= runs.n || total == 0) return no_share(p, wg);
    sh.u = sh.start = runs.first(wg);
    sh.end = runs.first(wg + 1);
    sh.total = total;
    if (p.B <= kPagedThreads) {
        if (sh.u >= excl && sh.u < excl + mine) found[0] = tid, found[1] = excl, found_work = work;
    } else {
        int32_t before = 0;
        for (int c = 0; c < p.B; c += kPagedThreads) {
            int32_t sum;
            if (c + tid < p.B) work = seq_work(p, c + tid);
            mine = c + tid < p.B ? work.units(p.groups) : 0;
            excl = before + scan(mine, sum);
            if (sh.u >= excl && sh.u < excl + mine) found[0] = c + tid, found[1] = excl, found_work = work;
            before += sum;
        }
    }
    __syncthreads();
    sh.seq = __builtin_amdgcn_readfirstlane(found[0]);
    sh.seq_base = __builtin_amdgcn_readfirstlane(found[1]);
    sh.sw.s0 = __builtin_amdgcn_readfirstlane(found_work.s0);
    sh.sw.rows = __builtin_amdgcn_readfirstlane(found_work.rows);
    sh.sw.tiles = __builtin_amdgcn_readfirstlane(found_work.tiles);
    sh.sw.ctx = __builtin_amdgcn_readfirstlane(found_work.ctx);
    sh.sw.blocks = __builtin_amdgcn_readfirstlane(found_work.blocks);
    return true;
}

// Workspace state of the part that starts at the run's unit u: 0 for the run's
// first part, 1 for another (its last: parts in between are whole items).
__device__ __forceinline__ int64_t part_slot(const Share& sh) {
    const int per = gridDim.x >> 3;
    return 2 * (int64_t)((blockIdx.x & 7) * per + (blockIdx.x >> 3)) + (sh.u == sh.start ? 0 : 1);
}

// The part of an item that starts at the run's unit u: blocks b0 .. b1 - 1 of
// (seq, group, tile); moves the share on to it and returns the sequence's work.
struct Part {
    int32_t group, tile, b0, b1;
    bool whole;
};
__device__ __forceinline__ SeqWork next_part(const PagedParams& p, Share& sh, Part& part) {
    SeqWork& sw = sh.sw;
    while (sh.u >= sh.seq_base + sw.units(p.groups)) {  // (empty sequences are passed over)
        sh.seq_base += sw.units(p.groups);
        sw = seq_work(p, ++sh.seq);
    }
    const uint32_t in = (uint32_t)(sh.u - sh.seq_base);
    const uint32_t item = in / (uint32_t)sw.blocks;
    part.b0 = (int32_t)(in - item * (uint32_t)sw.blocks);
    part.group = (int32_t)(item / (uint32_t)sw.tiles);
    part.tile = (int32_t)(item - (uint32_t)part.group * (uint32_t)sw.tiles);
    part.b1 = min(sw.blocks, part.b0 + (sh.end - sh.u));
    part.whole = part.b0 == 0 && part.b1 == sw.blocks;
    if (p.cuts && sh.u == sh.start && threadIdx.x == 0) {
        const int per = gridDim.x >> 3;
        p.cuts[(blockIdx.x & 7) * per + (blockIdx.x >> 3)] =
            RunStart{sw.s0, sw.rows, part.tile, part.group, part.b0, sw.blocks, sh.u - part.b0, sh.total};
    }
    return sw;
}

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

        // ---- the waves' states joined, row block by row block ----
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            l_run[q] = col4_sum(l_run[q]);
            if (lq == 0) {
                ml[0][wave][16 * q + l16] = m_run[q];
                ml[1][wave][16 * q + l16] = l_run[q];
            }
        }
        // a head's waves: [waves][16 rows][D / 4], float4 c of row r at c ^ (r & 7)
        float4* const os = reinterpret_cast<float4*>(vlds + wave / WPH * WPH * WBLK);
        constexpr int C4 = D / 4;
        constexpr int PASS = 64 * WPH / DV;  // rows that a head's threads take at a time
        const int ht = tid % (64 * WPH), hw = wave / WPH * WPH;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            __syncthreads();  // (q = 0: the key loops are done; later: the block before has been read)
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
                os[(wave % WPH * 16 + l16) * C4 + ((4 * dt + lq) ^ (l16 & 7))] =
                    make_float4(oacc[q][dt][0], oacc[q][dt][1], oacc[q][dt][2], oacc[q][dt][3]);
            __syncthreads();
            const int ch = ht % DV;
            for (int row = ht / DV; row < 16; row += PASS) {
                int64_t qrow;
                int qh;
                if (!query_of(16 * q + row, qrow, qh)) break;
                float m = -INFINITY, l = 0.f, acc[8] = {};
#pragma unroll
                for (int w = 0; w < WPH; ++w) m = fmaxf(m, ml[0][hw + w][16 * q + row]);
                const float mc = m == -INFINITY ? 0.f : m * p.scale_log2;
#pragma unroll
                for (int w = 0; w < WPH; ++w) {
                    const float f = fast_exp2(__builtin_fmaf(ml[0][hw + w][16 * q + row], p.scale_log2, -mc));
                    l += f * ml[1][hw + w][16 * q + row];
                    const float4 x = os[(w * 16 + row) * C4 + ((2 * ch) ^ (row & 7))];
                    const float4 y = os[(w * 16 + row) * C4 + ((2 * ch + 1) ^ (row & 7))];
                    acc[0] += f * x.x, acc[1] += f * x.y, acc[2] += f * x.z, acc[3] += f * x.w;
                    acc[4] += f * y.x, acc[5] += f * y.y, acc[6] += f * y.z, acc[7] += f * y.w;
                }
                if (part.whole) {
                    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
                    for (int j = 0; j < 8; ++j) acc[j] = in_range<T>(acc[j] * inv);
                    st16(p.o + qrow * p.so_t + qh * p.so_h + 8 * ch, pack8<T>(acc));
                    if (p.lse && ch == 0) p.lse[qrow * p.sl_t + qh * p.sl_h] = (mc + fast_log2(l)) * kLn2;
                } else {
                    const int64_t r = (part_slot(sh) * HW + wave / WPH) * ROWS + 16 * q + row;
                    if (ch == 0) {
                        p.part_m[r] = m * p.scale_log2;
                        p.part_l[r] = l;
                    }
                    float4* a = reinterpret_cast<float4*>(p.part_acc + r * D + 8 * ch);
                    a[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                    a[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
                }
            }
        }
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
// Joins the parts of cut items.  WPR waves per row, each with an equal share of
// the parts: one part's maximum and sum per lane, the numerators with lanes
// across the head dim.  What bounds it is its chain of dependent loads (lengths
// and units, then the states): four waves per row where few rows leave the chip
// empty.  Waves are dealt to every row that the call may have (sequence, query
// token, q head) or, where most sequences are far shorter than the longest, to
// the rows of the item that each run starts in: the first run that starts inside
// an item joins it.  (64 sequences, one of 2048 tokens and the others of one,
// contexts of 500, 32 / 8 heads: 500 us for rows that are not there, 67 so.)
// ---------------------------------------------------------------------------
template <typename T, int D, int WPR>
__global__ __launch_bounds__(kPagedThreads) void paged_merge_kernel(PagedParams p, int32_t n_rows, Divider hqdiv,
                                                                    Divider msdiv) {
    constexpr int E = D / 64 ? D / 64 : 1;  // floats of a lane (D = 32: lanes 0 .. 31)
    __shared__ float wm[WPR], wl[WPR], wacc[WPR > 1 ? WPR * D : 1];
    const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
    const int row = WPR == 1 ? blockIdx.x * 4 + wave : blockIdx.x;
    const int sub = WPR == 1 ? 0 : wave;
    if (row >= n_rows) return;
    int32_t s0, rows, tile, grp, hl, rr, a, blocks, total;  // hl, rr: kv head of the group, row of the tile
    if (p.cuts) {
        const int w = row >> (p.row_shift + p.head_shift);
        const int in = row - (w << (p.row_shift + p.head_shift));
        hl = in >> p.row_shift;
        rr = in - (hl << p.row_shift);
        const RunStart c = p.cuts[w];
        if (c.b0 == 0) return;
        s0 = c.s0, rows = c.rows, tile = c.tile, grp = c.group, a = c.first, blocks = c.blocks, total = c.total;
        if (w > 0 && Runs(total, p.nwg, p.least).first(w - 1) > a) return;
    } else {
        const int r0 = divide(row, hqdiv);
        const int qh = row - r0 * p.Hq;
        const int seq = divide(r0, msdiv);
        const int tok = r0 - seq * p.max_seqlen;
        total = p.base[p.B];
        const int32_t base = p.base[seq];  // (asked for with the sequence's lengths)
        const SeqWork sw = seq_work(p, seq);
        const int kvh = divide(qh, p.gdiv);
        rr = tok * p.group + (qh - kvh * p.group);
        s0 = sw.s0, rows = sw.rows, blocks = sw.blocks;
        tile = rr >> p.row_shift;
        rr -= tile << p.row_shift;
        grp = kvh >> p.head_shift;
        hl = kvh - (grp << p.head_shift);
        a = base + (grp * sw.tiles + tile) * blocks;
    }
    const int in_seq = (tile << p.row_shift) + rr;
    if (in_seq >= rows) return;
    const Runs runs(total, p.nwg, p.least);
    const int w0 = runs.of(a), w1 = runs.of(a + blocks - 1) + 1;
    if (w0 + 1 == w1) return;  // finished by its workgroup
    const int tok = divide(in_seq, p.gdiv);
    const int qh = ((grp << p.head_shift) + hl) * p.group + (in_seq - tok * p.group);
    uint16_t* const o = p.o + (int64_t)(s0 + tok) * p.so_t + qh * p.so_h;
    float* const lse = p.lse ? p.lse + (int64_t)(s0 + tok) * p.sl_t + qh * p.sl_h : nullptr;
    // row of the workspace that holds run w's part: a run that starts inside the
    // item, or with it, holds it in state 0
    auto at = [&](int w) {
        const int64_t state = 2 * (int64_t)w + (runs.first(w) >= a ? 0 : 1);
        return ((((state << p.head_shift) + hl) << p.row_shift)) + rr;
    };
    const int share = WPR == 1 ? w1 - w0 : (w1 - w0 + WPR - 1) / WPR;
    const int lo = w0 + sub * share, hi = min(w1, lo + share);
    const bool in = lane * E < D;
    float m = -INFINITY, l = 0.f, acc[E] = {};
    for (int c = lo; c < hi; c += 64) {
        const int n = min(64, hi - c);
        const bool mine = lane < n;
        const int64_t own = at(min(c + lane, hi - 1));
        const float mi = mine ? p.part_m[own] : -INFINITY;
        const float li = mine ? p.part_l[own] : 0.f;
        constexpr int U = 8;  // numerators requested together, the first ones before any maximum is known
        float x[U][E];
        auto request = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float* from = p.part_acc + at(min(c + i + u, hi - 1)) * D + (in ? lane * E : 0);
#pragma unroll
                for (int e = 0; e < E; ++e) x[u][e] = from[e];
            }
        };
        request(0);
        float mn = mi;
        for (int d = 32; d; d >>= 1) mn = fmaxf(mn, __shfl_xor(mn, d));
        mn = fmaxf(mn, m);
        const float mc = mn == -INFINITY ? 0.f : mn;
        const float old = fast_exp2(m - mc);
        const float f = mine ? fast_exp2(mi - mc) : 0.f;
        l = l * old + f * li;
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] *= old;
        for (int i = 0; i < n; i += U) {
            if (i) request(i);
#pragma unroll
            for (int u = 0; u < U; ++u) {
                const float fi = __builtin_bit_cast(
                    float, __builtin_amdgcn_readlane(__builtin_bit_cast(int, f), min(i + u, 63)));
#pragma unroll
                for (int e = 0; e < E; ++e) acc[e] = __builtin_fmaf(fi, i + u < n ? x[u][e] : 0.f, acc[e]);
            }
        }
        m = mn;
    }
    for (int d = 32; d; d >>= 1) l += __shfl_xor(l, d);
    if constexpr (WPR > 1) {
        if (lane == 0) wm[sub] = m, wl[sub] = l;
        if (in) {
#pragma unroll
            for (int e = 0; e < E; ++e) wacc[sub * D + lane * E + e] = acc[e];
        }
        __syncthreads();
        if (sub) return;
        m = -INFINITY, l = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) m = fmaxf(m, wm[w]);
#pragma unroll
        for (int e = 0; e < E; ++e) acc[e] = 0.f;
#pragma unroll
        for (int w = 0; w < WPR; ++w) {
            const float f = fast_exp2(wm[w] - (m == -INFINITY ? 0.f : m));
            l += f * wl[w];
#pragma unroll
            for (int e = 0; e < E; ++e) acc[e] += f * (in ? wacc[w * D + lane * E + e] : 0.f);
        }
    }
    const float mc = m == -INFINITY ? 0.f : m;
    const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
    if (in) {
        if constexpr (E == 2)
            *reinterpret_cast<uint32_t*>(o + 2 * lane) = MfmaOps<T>::pack2(in_range<T>(acc[0] * inv), in_range<T>(acc[1] * inv));
        else
            o[lane] = (uint16_t)MfmaOps<T>::pack2(in_range<T>(acc[0] * inv), 0.f);
    }
    if (lse && lane == 0) *lse = (mc + fast_log2(l)) * kLn2;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Kernel of a call: row blocks of a tile (0: the wide kernel), log2 of its rows
// and of a unit's keys, kv heads of a workgroup, workgroups per CU, and whether
// every item is one workgroup's.
struct PagedShape {
    int qb, row_shift, key_shift, heads, per_cu;
    bool items;
};
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

struct PagedSpace {
    int64_t base, cuts, m, l, acc, bytes;
};
static PagedSpace paged_space(int32_t batch, int nwg, const PagedShape& shape, int head_dim) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t rows = (2 * (int64_t)nwg * shape.heads) << shape.row_shift;
    PagedSpace s;
    s.base = 0;
    s.cuts = up(((int64_t)batch + 1) * 4);
    s.m = s.cuts + up(nwg * (int64_t)sizeof(RunStart));
    s.l = s.m + up(rows * 4);
    s.acc = s.l + up(rows * 4);
    s.bytes = s.acc + rows * head_dim * 4;
    return s;
}

template <typename T, int D>
static int launch_merge(const PagedParams& p, hipStream_t st) {
    const int64_t rows = p.cuts ? (int64_t)p.nwg * p.heads << p.row_shift : (int64_t)p.B * p.max_seqlen * p.Hq;
    const Divider hq = make_divider(p.Hq), ms = make_divider(p.max_seqlen);
    if (rows <= 512)
        hipLaunchKernelGGL((paged_merge_kernel<T, D, 4>), dim3((uint32_t)rows), dim3(kPagedThreads), 0, st, p,
                           (int32_t)rows, hq, ms);
    else
        hipLaunchKernelGGL((paged_merge_kernel<T, D, 1>), dim3((uint32_t)((rows + 3) / 4)),
                           dim3(kPagedThreads), 0, st, p, (int32_t)rows, hq, ms);
    return launch_status("paged_merge_kernel");
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

// What the workspace size and the launch agree on; false: nothing to launch.
struct PagedPlan {
    int32_t max_seqlen;
    PagedShape shape;
    int nwg, least, tiles;
    bool too_many;  // units past 32 bits
};
static bool paged_plan(PagedPlan& plan, int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t hq,
                       int32_t hkv, int32_t head_dim, int32_t pt_cols, int32_t page_size) {
    if (batch <= 0 || total_tokens <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || pt_cols < 0 || page_size < 1 ||
        (int64_t)pt_cols * page_size > kMaxPositions)
        return false;
    plan.max_seqlen = (int32_t)std::min<int64_t>(max_seqlen, total_tokens);
    if (plan.max_seqlen <= 0) return false;
    const int64_t rows = (int64_t)plan.max_seqlen * (hq / hkv);
    plan.shape = paged_shape(rows, (int64_t)batch * hkv, hkv, (int64_t)pt_cols * page_size, head_dim);
    // As many workgroups as run at once, no more than the units that the page
    // table has room for.
    const int64_t tiles = ((rows - 1) >> plan.shape.row_shift) + 1;
    const int64_t blocks =
        std::max<int64_t>(1, ((int64_t)pt_cols * page_size + (1 << plan.shape.key_shift) - 1) >> plan.shape.key_shift);
    const double units = (double)batch * (hkv / plan.shape.heads) * tiles * blocks;
    plan.too_many = units >= 2147483648.0;
    plan.tiles = (int)std::min<int64_t>(tiles, INT32_MAX);
    plan.nwg = (int)std::min<double>(256.0 * plan.shape.per_cu, std::max(1.0, units));
    plan.nwg = (plan.nwg + 7) / 8 * 8;
    plan.least = plan.shape.qb ? 1 : 2;
    return true;
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int64_t qattn_prefix_paged_workspace_bytes(int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim,
                                           int32_t pt_cols, int32_t page_size) {
    PagedPlan plan;
    if (head_dim <= 0 || !paged_plan(plan, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, head_dim,
                                     pt_cols, page_size))
        return 0;
    return plan.shape.items ? 0 : paged_space(batch, plan.nwg, plan.shape, head_dim).bytes;
}

int qattn_prefix_paged_fwd(const void* q, const int64_t q_stride[3], const void* k_cache, const int64_t k_stride[4],
                           const void* v_cache, const int64_t v_stride[4], const int32_t* page_table,
                           int32_t pt_cols, int32_t num_pages, int32_t page_size, const int32_t* context_lens,
                           void* o, const int64_t o_stride[3], float* lse, const int64_t lse_stride[2],
                           const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                           int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale, int32_t dtype,
                           void* workspace, int64_t workspace_size, void* stream) {
    clear_error();
    const int rc = check_common(dtype, head_dim, batch, max_seqlen, total_tokens, num_q_heads, num_kv_heads, 0);
    if (rc) return rc;
    if (page_size < 1 || pt_cols < 0 || num_pages < 0 || (int64_t)pt_cols * page_size > kMaxPositions) {
        set_error("bad paged arguments: page_size=%d pt_cols=%d num_pages=%d", page_size, pt_cols, num_pages);
        return QATTN_ERR_ARG;
    }
    if (!(scale > 0.f) || !(scale < INFINITY)) {
        set_error("scale must be positive and finite");
        return QATTN_ERR_ARG;
    }
    PagedPlan plan;
    if (!paged_plan(plan, batch, cu_seqlens ? max_seqlen : 1, total_tokens, num_q_heads, num_kv_heads, head_dim,
                    pt_cols, page_size))
        return QATTN_OK;  // nothing to compute
    const bool keys = pt_cols > 0 && num_pages > 0;
    if (!q || !o || !q_stride || !o_stride || !k_stride || !v_stride || !context_lens || (lse && !lse_stride) ||
        (pt_cols > 0 && !page_table) || (keys && (!k_cache || !v_cache))) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    if (plan.too_many || (int64_t)plan.max_seqlen * (num_q_heads / num_kv_heads) > INT32_MAX / 2) {
        set_error("sizes too large: batch=%d num_kv_heads=%d max_seqlen=%d group=%d pt_cols=%d page_size=%d", batch,
                  num_kv_heads, plan.max_seqlen, num_q_heads / num_kv_heads, pt_cols, page_size);
        return QATTN_ERR_ARG;
    }
    if (!row_aligned(q, q_stride, 2) || !row_aligned(o, o_stride, 2)) {
        set_error("q/o rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    if (!row_aligned(k_cache, k_stride, 3) || !row_aligned(v_cache, v_stride, 3)) {
        set_error("k/v cache rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    if (keys) {
        for (const int64_t* st : {k_stride, v_stride}) {
            // a row's offset (kv head aside) in 16-byte units is 32 bits wide
            if (st[0] < 0 || st[1] < 0 || st[0] > (int64_t(1) << 40) || st[1] > (int64_t(1) << 32) ||
                ((num_pages - 1) * (st[0] / 8) + (page_size - 1) * (st[1] / 8)) >= (int64_t(1) << 32)) {
                set_error("cache strides must be non-negative and a cache span less than 64 GiB");
                return QATTN_ERR_LAYOUT;
            }
        }
    }
    const PagedSpace sp = paged_space(batch, plan.nwg, plan.shape, head_dim);
    if (!plan.shape.items && (!workspace || workspace_size < sp.bytes)) {
        set_error("workspace of %lld bytes needed, %lld given", (long long)sp.bytes, (long long)workspace_size);
        return QATTN_ERR_WORKSPACE;
    }
    if (!plan.shape.items && (uintptr_t)workspace & 255u) {
        set_error("workspace must be 256-byte aligned");
        return QATTN_ERR_WORKSPACE;
    }
    PagedParams p{};
    p.q = (const uint16_t*)q;
    p.kc = (const uint16_t*)k_cache;
    p.vc = (const uint16_t*)v_cache;
    p.o = (uint16_t*)o;
    p.lse = lse;
    p.cu = cu_seqlens;
    p.table = page_table;
    p.ctx = context_lens;
    p.sq_t = q_stride[0], p.sq_h = q_stride[1];
    p.so_t = o_stride[0], p.so_h = o_stride[1];
    if (lse) p.sl_t = lse_stride[0], p.sl_h = lse_stride[1];
    p.sk_page = k_stride[0], p.sk_slot = k_stride[1], p.sk_head = k_stride[2];
    p.sv_page = v_stride[0], p.sv_slot = v_stride[1], p.sv_head = v_stride[2];
    p.total_tokens = total_tokens;
    p.B = batch, p.Hq = num_q_heads, p.Hkv = num_kv_heads, p.group = num_q_heads / num_kv_heads;
    p.max_seqlen = plan.max_seqlen;
    p.pt_cols = pt_cols, p.num_pages = num_pages, p.page_size = page_size;
    p.capacity = keys ? pt_cols * page_size : 0;  // (without pages no key exists)
    p.nwg = plan.nwg;
    p.least = plan.least;
    p.tiles = plan.tiles;
    p.heads = plan.shape.heads;
    p.groups = num_kv_heads / p.heads;
    p.row_shift = plan.shape.row_shift;
    p.key_shift = plan.shape.key_shift;
    p.groupdiv = make_divider(p.groups);
    p.tilediv = make_divider(plan.tiles);
    p.head_shift = p.heads == 4 ? 2 : p.heads == 2 ? 1 : 0;
    p.pdiv = make_divider(page_size);
    p.gdiv = make_divider(p.group);
    p.scale_log2 = scale * kLog2e;
    char* const ws = (char*)workspace;
    p.base = (int32_t*)(ws + sp.base);
    // (a wave of the merge that finds no row costs a fraction of one that joins
    // parts, and a run's rows may be none of a cut item)
    if ((double)batch * plan.max_seqlen * num_q_heads > 2.0 * ((int64_t)plan.nwg * p.heads << p.row_shift))
        p.cuts = (RunStart*)(ws + sp.cuts);
    p.part_m = (float*)(ws + sp.m);
    p.part_l = (float*)(ws + sp.l);
    p.part_acc = (float*)(ws + sp.acc);
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
