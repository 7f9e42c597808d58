// paged_work.h -- attention of query tokens over their sequence's context in
// pages: parameters, the deal of the work to workgroups, the join of cut items,
// and the host's checks, for the kernels over 16-bit caches (paged_attn.hip) and
// over quantised ones (quant_attn.hip).
//
// Work: units of 32 to 128 keys of one (sequence, kv heads, row tile), numbered
// sequence by sequence, heads, tiles and keys innermost.  The workgroups of the
// launch take equal runs of all units, whatever the contexts' lengths (no host
// knows them: the lengths stay on the device), so a run may end inside an item.
// A run's whole items are finished in the workgroup; of a cut item every part
// leaves its state (m, l, numerator, fp32) in the workspace and
// paged_merge_kernel joins them in key order, without atomics: results do not
// depend on timing.
#pragma once

#include <algorithm>

#include "dense_tiles.h"
#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kPagedThreads = 256;

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
// Workgroup 0 leaves the sequences' first units to the merge.  Every one of the
// workgroup's NT threads calls it; false: no unit.
struct Share {
    int32_t u, end, start, seq, seq_base, total;
    SeqWork sw;  // of seq
};
__device__ __forceinline__ bool no_share(const PagedParams& p, int wg) {
    if (p.cuts && threadIdx.x == 0) p.cuts[wg] = RunStart{};
    return false;
}
template <int NT = kPagedThreads>
__device__ __forceinline__ bool find_share(const PagedParams& p, Share& sh) {
    __shared__ int32_t sums[NT / 64];
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
        for (int w = 0; w < NT / 64; ++w) {
            before += w < wave ? sums[w] : 0;
            sum += sums[w];
        }
        return before + inc - mine;
    };
    int32_t total = 0, mine = 0, excl = 0;
    SeqWork work{};
    for (int c = 0; c < p.B; c += NT) {
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
    if (p.B <= NT) {
        if (sh.u >= excl && sh.u < excl + mine) found[0] = tid, found[1] = excl, found_work = work;
    } else {
        int32_t before = 0;
        for (int c = 0; c < p.B; c += NT) {
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
// The states of a workgroup's NW waves (NW / HW for each of HW kv heads, 16 QB
// rows each) joined row block by row block: the part's output, or its state in
// the workspace.  oacc element i of tile dt is row l16, column 16 dt + 4 lq + i;
// column chunk ch (8 columns) holds head dims 8 dims_of(ch) .. + 7; row r's state lies
// at row state_of(r) of its part's in the workspace.  lds: NW x 32 x D elements of 16
// bits that no wave uses any more after the first barrier.  part_rows: rows of a part.
// ---------------------------------------------------------------------------
template <typename T, int D, int QB, int NW, int HW, class Query, class Dims, class State>
__device__ __forceinline__ void join_waves(const PagedParams& p, const Share& sh, const Part& part, Query query_of,
                                           const float (&m_run)[QB], float (&l_run)[QB], const f4_t (&oacc)[QB][D / 16],
                                           uint16_t* lds, float (&ml)[2][NW][16 * QB], Dims dims_of, int part_rows,
                                           State state_of) {
    constexpr int DV = D / 8, ND = D / 16, WBLK = 32 * D, WPH = NW / HW;
    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int l16 = lane & 15, lq = lane >> 4;
#pragma unroll
    for (int q = 0; q < QB; ++q) {
        l_run[q] = col4_sum(l_run[q]);
        if (lq == 0) {
            ml[0][wave][16 * q + l16] = m_run[q];
            ml[1][wave][16 * q + l16] = l_run[q];
        }
    }
    // a head's waves: [waves][16 rows][D / 4], float4 c of row r at c ^ (r & 7)
    float4* const os = reinterpret_cast<float4*>(lds + wave / WPH * WPH * WBLK);
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
        const int ch = ht % DV, dim = 8 * dims_of(ch);
        for (int row = ht / DV; row < 16; row += PASS) {
            int64_t qrow;
            int qh;
            if (!query_of(16 * q + row, qrow, qh)) continue;
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
                st16(p.o + qrow * p.so_t + qh * p.so_h + dim, pack8<T>(acc));
                if (p.lse && ch == 0) p.lse[qrow * p.sl_t + qh * p.sl_h] = (mc + fast_log2(l)) * kLn2;
            } else {
                const int64_t r = part_slot(sh) * part_rows + state_of(16 * q + row);
                if (ch == 0) {
                    p.part_m[r] = m * p.scale_log2;
                    p.part_l[r] = l;
                }
                float4* a = reinterpret_cast<float4*>(p.part_acc + r * D + dim);
                a[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
                a[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            }
        }
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
        const int n = __builtin_amdgcn_readfirstlane(min(64, hi - c));
        const bool mine = lane < n;
        const int64_t own = at(min(c + lane, hi - 1));
        const float mi = mine ? p.part_m[own] : -INFINITY;
        const float li = mine ? p.part_l[own] : 0.f;
        // numerators requested together (in eights that are there), the first ones before any
        // maximum is known (eight alone: 1 x 30000 keys in 4 bits 22.9 us, with sixteen 22.3;
        // 32: 22.1, but 1 x 131072 43.0 against 42.5)
        constexpr int U = 16;
        float x[U][E];
        auto request = [&](int i) {
#pragma unroll
            for (int u = 0; u < U; ++u) {
                if (u >= 8 && i + u / 8 * 8 >= n) break;
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
                if (u >= 8 && i + u / 8 * 8 >= n) break;
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
// and of a unit's keys, kv heads of a workgroup, workgroups per CU, whether every
// item is one workgroup's.
struct PagedShape {
    int qb, row_shift, key_shift, heads, per_cu;
    bool items;
    int wave_heads;  // quantised caches: kv heads of a wave
};

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

// What the workspace size and the launch agree on; shape_of chooses the kernel.
// false: nothing to launch.
struct PagedPlan {
    int32_t max_seqlen;
    PagedShape shape;
    int nwg, least, tiles;
    bool too_many;  // units past 32 bits
    bool nothing;   // no row: nothing to launch
};
template <class ShapeOf>
static bool paged_plan(PagedPlan& plan, ShapeOf shape_of, int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t hq,
                       int32_t hkv, int32_t head_dim, int32_t pt_cols, int32_t page_size) {
    if (head_dim <= 0 || batch <= 0 || total_tokens <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || pt_cols < 0 || page_size < 1 ||
        (int64_t)pt_cols * page_size > kMaxPositions)
        return false;
    plan.max_seqlen = (int32_t)std::min<int64_t>(max_seqlen, total_tokens);
    if (plan.max_seqlen <= 0) return false;
    const int64_t rows = (int64_t)plan.max_seqlen * (hq / hkv);
    plan.shape = shape_of(rows, (int64_t)batch * hkv, hkv, (int64_t)pt_cols * page_size, head_dim);
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

template <class ShapeOf>
static int64_t paged_workspace(ShapeOf shape_of, int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t hq,
                               int32_t hkv, int32_t head_dim, int32_t pt_cols, int32_t page_size) {
    PagedPlan plan;
    if (!paged_plan(plan, shape_of, batch, max_seqlen, total_tokens, hq, hkv, head_dim, pt_cols, page_size)) return 0;
    return plan.shape.items ? 0 : paged_space(batch, plan.nwg, plan.shape, head_dim).bytes;
}

// A call's checks, plan and parameters.  Strides of the caches {page, slot, head,
// dim} in elements of two bytes.
template <class ShapeOf>
static int paged_setup(PagedParams& p, PagedPlan& plan, ShapeOf shape_of, const void* q, const int64_t* q_stride,
                       const void* k_cache, const int64_t* k_stride, const void* v_cache, const int64_t* v_stride,
                       const int32_t* page_table, int32_t pt_cols, int32_t num_pages, int32_t page_size,
                       const int32_t* context_lens, void* o, const int64_t* o_stride, float* lse,
                       const int64_t* lse_stride, const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen,
                       int64_t total_tokens, int32_t num_q_heads, int32_t num_kv_heads, int32_t head_dim, float scale,
                       int32_t dtype, void* workspace, int64_t workspace_size) {
    plan.nothing = false;
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
    plan.nothing = !paged_plan(plan, shape_of, batch, cu_seqlens ? max_seqlen : 1, total_tokens, num_q_heads,
                               num_kv_heads, head_dim, pt_cols, page_size);
    if (plan.nothing) return QATTN_OK;
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
    p.head_shift = __builtin_ctz((unsigned)p.heads);
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
    return QATTN_OK;
}

}  // namespace qattn
