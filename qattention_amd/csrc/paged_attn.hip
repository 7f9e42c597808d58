// paged_attn.hip -- attention of query tokens over their sequence's context in
// a paged K/V cache, with LSE.
//
// Row r of sequence s and kv head g is query token r / group, q head
// g * group + r % group; every row attends keys 0 .. context - 1:
//   o = sum_j softmax_j(scale q.k_j) v_j,  lse = m + ln sum_j exp(s_j - m)
// in one pass with a running maximum m and sum l.
//
// Work: units of 128 keys of one (sequence, kv head, tile of 16 QB rows),
// numbered sequence by sequence, heads, tiles and keys innermost.  The
// workgroups of the launch take equal runs of all units, whatever the
// contexts' lengths (no host knows them: the lengths stay on the device), so a
// run may end inside an item.  A run's whole items are finished in the
// workgroup; of a cut item every part leaves its state (m, l, numerator, fp32)
// in the workspace and paged_merge_kernel joins them in key order, without
// atomics: results do not depend on timing.
//
// A unit's 128 keys are 32 per wave.  Per step a wave forms
//   S^T = K Q^T      2 key tiles x D/32 products of v_mfma_f32_16x16x32
//   O^T += V^T P^T   D/16 products
// with K rows loaded from the cache straight into the A operand's layout and
// V rows through a wave-private LDS block that the transposing reads
// (ds_read_b64_tr_b16) take as V^T; S^T has one row (query) per lane column,
// and its registers are the P^T operand.  The loads of the next step are
// requested before the products of this one; page numbers one step earlier.
#include <algorithm>

#include "kv_tiles.h"
#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kPagedThreads = 256;
constexpr int kUnit = 128;  // keys per unit: 4 waves x 32

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
    int32_t slots;        // rows of one workspace state: 16 QB
    Divider pdiv, gdiv;   // page_size, group
    float scale_log2;
    int64_t* base;        // [B + 1] first unit of each sequence (written by the main kernel)
    float* part_m;        // [nwg][2][slots]
    float* part_l;
    float* part_acc;      // [nwg][2][slots][D]
};

// Waves per SIMD: two, but one with 128-wide heads from 32 rows on, whose
// accumulators, K operand and loads in flight take the registers of both.
constexpr int paged_waves(int d, int qb) { return d == 128 && qb > 1 ? 1 : 2; }

// Rows, tiles and units of a sequence.
struct SeqWork {
    int32_t s0, rows, tiles, ctx, blocks;
    __device__ __forceinline__ int64_t units(int hkv) const { return (int64_t)hkv * tiles * blocks; }
};
template <int QB>
__device__ __forceinline__ SeqWork seq_work(const PagedParams& p, int s) {
    SeqWork w;
    w.s0 = p.cu ? p.cu[s] : s;
    const int32_t s1 = p.cu ? p.cu[s + 1] : s + 1;
    int32_t n = s1 - w.s0;
    if (w.s0 < 0 || s1 < w.s0 || (int64_t)s1 > p.total_tokens) n = 0;
    n = min(n, p.max_seqlen);
    w.rows = n * p.group;
    w.tiles = (w.rows + 16 * QB - 1) / (16 * QB);
    w.ctx = max(0, min(p.ctx[s], p.capacity));
    w.blocks = (w.ctx + kUnit - 1) / kUnit;
    return w;
}

// Workgroups that take units, and the first unit of workgroup w of them.
__device__ __forceinline__ int64_t run_first(int64_t total, int nwg, int w) { return total * w / nwg; }
__device__ __forceinline__ int runs_of(int64_t total, int nwg) { return (int)(total < nwg ? total : nwg); }

template <typename T, int D, int QB>
__global__ __launch_bounds__(kPagedThreads)
    __attribute__((amdgpu_waves_per_eu(paged_waves(D, QB)))) void paged_attn_kernel(PagedParams p) {
    constexpr int NC = D / 32;     // k-steps of S^T over the head dim
    constexpr int ND = D / 16;     // d-tiles of O^T
    constexpr int DV = D / 8;      // 16-byte chunks per row
    constexpr int RPI = 512 / D;   // V rows per load instruction of a wave
    constexpr int NV = 32 / RPI;   // V loads per lane and step
    constexpr int WBLK = 32 * D;   // elements of a wave's V block
    // The waves' V blocks; after the key loop, the waves' numerators of one
    // row block (4 x 16 rows x D floats, the same size).
    __shared__ __attribute__((aligned(1024))) uint16_t vlds[4 * WBLK];
    __shared__ float ml[2][4][16 * QB];
    __shared__ int64_t scan[4];
    __shared__ int found_seq;
    __shared__ int64_t found_base;

    const int tid = threadIdx.x;
    const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const int lane = tid & 63;
    const int l16 = lane & 15, lq = lane >> 4;
    // consecutive runs on one XCD: tiles of one item share its L2
    const int per = gridDim.x >> 3;
    const int wg = (blockIdx.x & 7) * per + (blockIdx.x >> 3);

    // ---- units of every sequence: their sum, then the sequence that holds
    // this run's first unit.  Workgroup 0 leaves the table to the merge. ----
    auto chunk_scan = [&](int s, int64_t& sum) {  // exclusive prefix within the chunk, and its sum
        const int64_t mine = s < p.B ? seq_work<QB>(p, s).units(p.Hkv) : 0;
        int64_t inc = mine;
#pragma unroll
        for (int d = 1; d < 64; d <<= 1) {
            const int64_t up = __shfl_up(inc, d);
            if (lane >= d) inc += up;
        }
        __syncthreads();
        if (lane == 63) scan[wave] = inc;
        __syncthreads();
        int64_t before = 0;
        sum = 0;
#pragma unroll
        for (int w = 0; w < 4; ++w) {
            before += w < wave ? scan[w] : 0;
            sum += scan[w];
        }
        return before + inc - mine;
    };
    int64_t total = 0, excl0 = 0;
    for (int c = 0; c < p.B; c += kPagedThreads) {
        int64_t sum;
        const int64_t e = chunk_scan(c + tid, sum);
        if (c == 0) excl0 = e;
        if (wg == 0 && c + tid < p.B) p.base[c + tid] = total + e;
        total += sum;
    }
    if (wg == 0 && tid == 0) p.base[p.B] = total;
    const int nrun = runs_of(total, p.nwg);
    if (wg >= nrun) return;
    int64_t u = run_first(total, nrun, wg);
    const int64_t u_end = run_first(total, nrun, wg + 1);
    {
        int64_t before = 0;
        for (int c = 0; c < p.B; c += kPagedThreads) {
            int64_t sum;
            const bool one = p.B <= kPagedThreads;
            const int64_t e = one ? excl0 : before + chunk_scan(c + tid, sum);
            const int s = c + tid;
            if (s < p.B) {
                const int64_t mine = seq_work<QB>(p, s).units(p.Hkv);
                if (u >= e && u < e + mine) {
                    found_seq = s;
                    found_base = e;
                }
            }
            if (!one) before += sum;
        }
        __syncthreads();
    }
    int seq = __builtin_amdgcn_readfirstlane(found_seq);
    int64_t seq_base = found_base;

    // wave-private V block: chunk c of row r at c ^ kv_swz(r)
    uint16_t* const vblk = vlds + wave * WBLK;
    const int vr = 4 * lq + (l16 >> 2);
    const int vaddr0 = vr * D + 8 * (((l16 & 3) >> 1) ^ kv_swz(vr, DV)) + 4 * (l16 & 1);

    while (u < u_end) {
        SeqWork sw = seq_work<QB>(p, seq);
        while (u >= seq_base + sw.units(p.Hkv)) {  // (empty sequences are passed over)
            seq_base += sw.units(p.Hkv);
            sw = seq_work<QB>(p, ++seq);
        }
        const int64_t in = u - seq_base;
        const int item = (int)(in / sw.blocks);  // kv head * tiles + tile
        const int b0 = (int)(in - (int64_t)item * sw.blocks);
        const int kvh = item / sw.tiles;
        const int tile = item - kvh * sw.tiles;
        const int b1 = (int)min((int64_t)sw.blocks, b0 + (u_end - u));
        const int ctx = sw.ctx;

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

        // key lane % 32 of step b: its page, or -1 (past the context)
        auto key_at = [&](int b) { return kUnit * b + 32 * wave + (lane & 31); };
        auto page_of = [&](int b) {
            const int pos = key_at(b);
            return pos < ctx && b < b1 ? pt[divide(pos, p.pdiv)] : -1;
        };
        // the step's loads: K rows in the A operand's layout, V rows by row
        // (load n: row n RPI + lane / DV, chunk lane % DV).  Keys that do not
        // exist read the cache's first row and count for nothing below.
        Vec16 kx[2][NC], vx[NV];
        uint32_t have = 0;  // bit j: key j of the step exists
        auto issue = [&](int b, int page) {
            const bool ok = (uint32_t)page < (uint32_t)p.num_pages;
            have = (uint32_t)__ballot(ok);
            const int pos = key_at(b);
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
        issue(b0, page);
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

        // ---- the four waves' states joined, row block by row block ----
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            l_run[q] = col4_sum(l_run[q]);
            if (lq == 0) {
                ml[0][wave][16 * q + l16] = m_run[q];
                ml[1][wave][16 * q + l16] = l_run[q];
            }
        }
        const bool whole = b0 == 0 && b1 == sw.blocks;
        const int64_t slot = 2 * (int64_t)wg + (u == run_first(total, nrun, wg) ? 0 : 1);
        float4* const os = reinterpret_cast<float4*>(vlds);  // [4 waves][16 rows][D / 4], float4 c of row r at c ^ (r & 7)
        constexpr int C4 = D / 4;
#pragma unroll
        for (int q = 0; q < QB; ++q) {
            __syncthreads();  // (q = 0: the key loops are done; later: the block before has been read)
#pragma unroll
            for (int dt = 0; dt < ND; ++dt)
                os[(wave * 16 + l16) * C4 + ((4 * dt + lq) ^ (l16 & 7))] =
                    make_float4(oacc[q][dt][0], oacc[q][dt][1], oacc[q][dt][2], oacc[q][dt][3]);
            __syncthreads();
            const int row = tid / DV, ch = tid % DV;
            if (row < 16) {
                float m = -INFINITY, l = 0.f, acc[8] = {};
#pragma unroll
                for (int w = 0; w < 4; ++w) m = fmaxf(m, ml[0][w][16 * q + row]);
                const float mc = m == -INFINITY ? 0.f : m * p.scale_log2;
#pragma unroll
                for (int w = 0; w < 4; ++w) {
                    const float f = fast_exp2(__builtin_fmaf(ml[0][w][16 * q + row], p.scale_log2, -mc));
                    l += f * ml[1][w][16 * q + row];
                    const float4 x = os[(w * 16 + row) * C4 + ((2 * ch) ^ (row & 7))];
                    const float4 y = os[(w * 16 + row) * C4 + ((2 * ch + 1) ^ (row & 7))];
                    acc[0] += f * x.x, acc[1] += f * x.y, acc[2] += f * x.z, acc[3] += f * x.w;
                    acc[4] += f * y.x, acc[5] += f * y.y, acc[6] += f * y.z, acc[7] += f * y.w;
                }
                int64_t qrow;
                int qh;
                if (query_of(16 * q + row, qrow, qh)) {
                    if (whole) {
                        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
#pragma unroll
                        for (int j = 0; j < 8; ++j) acc[j] *= inv;
                        st16(p.o + qrow * p.so_t + qh * p.so_h + 8 * ch, pack8<T>(acc));
                        if (p.lse && ch == 0) p.lse[qrow * p.sl_t + qh * p.sl_h] = (mc + fast_log2(l)) * kLn2;
                    } else {
                        const int64_t r = slot * p.slots + 16 * q + row;
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
        }
        __syncthreads();  // the LDS is free for the next item
        u += b1 - b0;
    }
}

// ---------------------------------------------------------------------------
// Joins the parts of cut items, and answers rows without a context (o = 0,
// lse = -inf).  Workgroup (sequence, query token, q head); wave w takes every
// fourth part.
// ---------------------------------------------------------------------------
template <typename T, int D, int QB>
__global__ __launch_bounds__(kPagedThreads) void paged_merge_kernel(PagedParams p, Divider hqdiv, Divider msdiv) {
    constexpr int E = D / 32;  // floats of a lane (lanes past D / E = 32 idle in the sums)
    __shared__ float wm[4], wl[4];
    __shared__ float wacc[4][D];
    const int r0 = divide(blockIdx.x, hqdiv);
    const int qh = blockIdx.x - r0 * p.Hq;
    const int seq = divide(r0, msdiv);
    const int tok = r0 - seq * p.max_seqlen;
    const SeqWork sw = seq_work<QB>(p, seq);
    const int kvh = divide(qh, p.gdiv);
    const int rr = tok * p.group + (qh - kvh * p.group);
    if (rr >= sw.rows) return;
    uint16_t* const o = p.o + (int64_t)(sw.s0 + tok) * p.so_t + qh * p.so_h;
    const int tid = threadIdx.x;
    if (sw.blocks == 0) {
        if (tid < D / 8) st16(o + 8 * tid, Vec16{{0u, 0u, 0u, 0u}});
        if (p.lse && tid == 0) p.lse[(int64_t)(sw.s0 + tok) * p.sl_t + qh * p.sl_h] = -INFINITY;
        return;
    }
    const int64_t total = p.base[p.B];
    const int nrun = runs_of(total, p.nwg);
    const int tile = rr / (16 * QB);
    const int64_t a = p.base[seq] + (int64_t)(kvh * sw.tiles + tile) * sw.blocks, b = a + sw.blocks;
    // runs that hold the first and the last unit of the item
    auto run_of = [&](int64_t x) {
        int w = (int)(((x + 1) * nrun - 1) / total);
        while (run_first(total, nrun, w) > x) --w;
        while (run_first(total, nrun, w + 1) <= x) ++w;
        return w;
    };
    const int w0 = run_of(a), w1 = run_of(b - 1);
    if (w0 == w1) return;  // finished by its workgroup
    const int wave = tid >> 6, lane = tid & 63;
    const int r = rr - tile * 16 * QB;
    auto at = [&](int w) {  // row of the workspace that holds run w's part
        return (2 * (int64_t)w + (run_first(total, nrun, w) >= a ? 0 : 1)) * p.slots + r;
    };
    // (a run that starts inside the item, or with it, holds its part in slot 0)
    float m = -INFINITY;
    for (int w = w0 + lane; w <= w1; w += 64) m = fmaxf(m, p.part_m[at(w)]);
    for (int d = 32; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
    const float mc = m == -INFINITY ? 0.f : m;
    float l = 0.f, acc[E] = {};
    for (int w = w0 + wave; w <= w1; w += 4) {
        const int64_t row = at(w);
        const float f = fast_exp2(p.part_m[row] - mc);
        l += f * p.part_l[row];
        if (lane < 32) {
#pragma unroll
            for (int j = 0; j < E; ++j) acc[j] += f * p.part_acc[row * D + lane * E + j];
        }
    }
    if (lane == 0) wl[wave] = l;
    if (lane < 32) {
#pragma unroll
        for (int j = 0; j < E; ++j) wacc[wave][lane * E + j] = acc[j];
    }
    __syncthreads();
    if (tid < D / 8) {
        l = wl[0] + wl[1] + wl[2] + wl[3];
        const float inv = l > 0.f ? 1.f / l : (l == 0.f ? 0.f : l);
        float x[8];
#pragma unroll
        for (int j = 0; j < 8; ++j)
            x[j] = (wacc[0][8 * tid + j] + wacc[1][8 * tid + j] + wacc[2][8 * tid + j] + wacc[3][8 * tid + j]) * inv;
        st16(o + 8 * tid, pack8<T>(x));
        if (p.lse && tid == 0)
            p.lse[(int64_t)(sw.s0 + tok) * p.sl_t + qh * p.sl_h] = (mc + fast_log2(l)) * kLn2;
    }
    (void)wm;
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Row blocks of a workgroup's tile: as many as the longest sequence fills.
static int row_blocks(int64_t max_rows) { return max_rows <= 16 ? 1 : max_rows <= 32 ? 2 : 4; }

// Workgroups of the launch: as many as run at once, no more than the units that
// the page table has room for.
static int paged_workgroups(int32_t batch, int64_t max_rows, int32_t hkv, int32_t capacity, int qb, int head_dim) {
    const int64_t tiles = (max_rows + 16 * qb - 1) / (16 * qb);
    const int64_t blocks = ((int64_t)capacity + kUnit - 1) / kUnit;
    const int64_t most = 256 * paged_waves(head_dim, qb);
    // batch * hkv * tiles * blocks, without passing 2^63
    int64_t units = std::min<int64_t>((int64_t)batch * hkv, most);
    units = std::min<int64_t>(units * std::min<int64_t>(tiles, most), most);
    units = std::min<int64_t>(units * std::min<int64_t>(blocks, most), most);
    return (int)((std::max<int64_t>(units, 1) + 7) / 8 * 8);
}

struct PagedSpace {
    int64_t base, m, l, acc, bytes;
};
static PagedSpace paged_space(int32_t batch, int nwg, int qb, int head_dim) {
    auto up = [](int64_t x) { return (x + 255) / 256 * 256; };
    const int64_t rows = 2 * (int64_t)nwg * 16 * qb;
    PagedSpace s;
    s.base = 0;
    s.m = up(((int64_t)batch + 1) * 8);
    s.l = s.m + up(rows * 4);
    s.acc = s.l + up(rows * 4);
    s.bytes = s.acc + rows * head_dim * 4;
    return s;
}

template <typename T, int D, int QB>
static int launch_paged_qb(const PagedParams& p, hipStream_t st) {
    hipLaunchKernelGGL((paged_attn_kernel<T, D, QB>), dim3(p.nwg), dim3(kPagedThreads), 0, st, p);
    const int rc = launch_status("paged_attn_kernel");
    if (rc) return rc;
    const int64_t blocks = (int64_t)p.B * p.max_seqlen * p.Hq;
    if (blocks > INT32_MAX) {
        set_error("grid too large (%lld blocks)", (long long)blocks);
        return QATTN_ERR_ARG;
    }
    hipLaunchKernelGGL((paged_merge_kernel<T, D, QB>), dim3((uint32_t)blocks), dim3(kPagedThreads), 0, st, p,
                       make_divider(p.Hq), make_divider(p.max_seqlen));
    return launch_status("paged_merge_kernel");
}

template <typename T>
static int launch_paged(const PagedParams& p, int head_dim, int qb, hipStream_t st) {
    switch (head_dim * 8 + qb) {
        case 32 * 8 + 1: return launch_paged_qb<T, 32, 1>(p, st);
        case 32 * 8 + 2: return launch_paged_qb<T, 32, 2>(p, st);
        case 32 * 8 + 4: return launch_paged_qb<T, 32, 4>(p, st);
        case 64 * 8 + 1: return launch_paged_qb<T, 64, 1>(p, st);
        case 64 * 8 + 2: return launch_paged_qb<T, 64, 2>(p, st);
        case 64 * 8 + 4: return launch_paged_qb<T, 64, 4>(p, st);
        case 128 * 8 + 1: return launch_paged_qb<T, 128, 1>(p, st);
        case 128 * 8 + 2: return launch_paged_qb<T, 128, 2>(p, st);
        default: return launch_paged_qb<T, 128, 4>(p, st);
    }
}

// What the workspace size and the launch agree on; false: nothing to launch.
struct PagedPlan {
    int32_t max_seqlen;
    int qb, nwg;
};
static bool paged_plan(PagedPlan& plan, int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t hq,
                       int32_t hkv, int32_t head_dim, int32_t pt_cols, int32_t page_size) {
    if (batch <= 0 || total_tokens <= 0 || hq <= 0 || hkv <= 0 || hq % hkv || pt_cols < 0 || page_size < 1 ||
        (int64_t)pt_cols * page_size > kMaxPositions)
        return false;
    plan.max_seqlen = (int32_t)std::min<int64_t>(max_seqlen, total_tokens);
    if (plan.max_seqlen <= 0) return false;
    const int64_t rows = (int64_t)plan.max_seqlen * (hq / hkv);
    plan.qb = row_blocks(rows);
    plan.nwg = paged_workgroups(batch, rows, hkv, pt_cols * page_size, plan.qb, head_dim);
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
    return paged_space(batch, plan.nwg, plan.qb, head_dim).bytes;
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
    if ((int64_t)plan.max_seqlen * (num_q_heads / num_kv_heads) > INT32_MAX / 2) {
        set_error("max_seqlen %d with %d q heads per kv head is too large", plan.max_seqlen, num_q_heads / num_kv_heads);
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
    const PagedSpace sp = paged_space(batch, plan.nwg, plan.qb, head_dim);
    if (!workspace || workspace_size < sp.bytes) {
        set_error("workspace of %lld bytes needed, %lld given", (long long)sp.bytes, (long long)workspace_size);
        return QATTN_ERR_WORKSPACE;
    }
    if ((uintptr_t)workspace & 255u) {
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
    p.slots = 16 * plan.qb;
    p.pdiv = make_divider(page_size);
    p.gdiv = make_divider(p.group);
    p.scale_log2 = scale * kLog2e;
    char* const ws = (char*)workspace;
    p.base = (int64_t*)(ws + sp.base);
    p.part_m = (float*)(ws + sp.m);
    p.part_l = (float*)(ws + sp.l);
    p.part_acc = (float*)(ws + sp.acc);
    return dtype == QATTN_DTYPE_F16 ? launch_paged<F16>(p, head_dim, plan.qb, (hipStream_t)stream)
                                    : launch_paged<BF16>(p, head_dim, plan.qb, (hipStream_t)stream);
}

}  // extern "C"
