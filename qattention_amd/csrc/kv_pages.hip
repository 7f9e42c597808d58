// kv_pages.hip -- moving K/V rows and pages of a paged cache: the rows of new
// tokens into the pages behind each context, the rows of an accepted draft
// path together, whole pages to other pages.
//
// All three only move 16-byte chunks: what bounds a large call is HBM (each
// byte read and written once), a small one its launch and one chain of
// dependent loads (sequence offsets, context length, page, row).  A row is
// addressed as page * stride_page + slot * stride_slot + head * stride_head
// in 64 bits, so caches of any size work; positions inside a sequence are 32
// bits (the host checks pt_cols * page_size).
#include <algorithm>

#include "qattn_common.h"
#include "qattn_device.h"

namespace qattn {

constexpr int kMoveThreads = 256;

struct PageParams {
    uint16_t* kc;
    uint16_t* vc;
    int64_t sk_layer, sk_page, sk_slot, sk_head;
    int64_t sv_layer, sv_page, sv_slot, sv_head;
    const int32_t* table;  // [B, pt_cols]
    const int32_t* ctx;    // [B]
    int32_t* new_lens;     // [B]
    int32_t pt_cols, num_pages, page_size, capacity;  // capacity: pt_cols * page_size
    int32_t B, chunks;                                // chunks: 16-byte chunks of one token's K row (all heads)
    Divider pdiv, cdiv;                               // page_size, chunks
    int32_t dvshift;                                  // chunks of one head's row: 1 << dvshift
};

// Loads and stores of append and copy, past the caches where they can be: for
// large moves (8 x 4003 rows of 8 x 128: 57.0 us with plain ones, 51.1 so; 256
// pages in 16 layers: 108.6 and 100.8), which run at the rate of a large copy.
// The attention that reads the rows next finds them further away: append and
// attention of a layer in a graph, 32 new rows over contexts of 100 tokens 9.1 us
// with plain ones, 9.3 so; 2048 rows that 64 tokens attend 31.5 and 32.6; 8 x 500
// rows, 4 x 60 over 2000 tokens, 32 over 2000: no difference.
typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Vec16 ld16_once(const void* p) {
    const u4_t x = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(p));
    return Vec16{{x[0], x[1], x[2], x[3]}};
}
__device__ __forceinline__ void st16_once(void* p, const Vec16& v) {
    const u4_t x = {v.w[0], v.w[1], v.w[2], v.w[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<u4_t*>(p));
}

// Element offset of position pos of sequence seq (head 0) in K and V, or
// false where its page does not exist.
__device__ __forceinline__ bool slot_of(const PageParams& p, int seq, int32_t pos, int64_t& ko, int64_t& vo) {
    const int32_t col = divide(pos, p.pdiv);
    const int32_t page = p.table[(int64_t)seq * p.pt_cols + col];
    const int32_t slot = pos - col * p.page_size;
    ko = (int64_t)page * p.sk_page + (int64_t)slot * p.sk_slot;
    vo = (int64_t)page * p.sv_page + (int64_t)slot * p.sv_slot;
    return (uint32_t)page < (uint32_t)p.num_pages;
}

// ---------------------------------------------------------------------------
// append: workgroup (sequence, run of `rows` new rows), or `rows` packed rows,
// of whichever sequences, where most sequences are far shorter than the longest
// (one of 2048 rows among 63 of one row, 8 heads of 128: 15.4 us for runs that
// are not there, 5.7 so); a thread moves one 16-byte chunk of K and of V at a
// time, kU of them requested before the first is stored.
// ---------------------------------------------------------------------------
constexpr int kU = 2;  // (8 x 4003 rows: 48.9 us, with four 50.3)

struct AppendParams {
    PageParams pg;
    const uint16_t* k;
    const uint16_t* v;
    int64_t sk_t, sk_h, sv_t, sv_h;
    const int32_t* cu;  // null: row s belongs to sequence s
    int64_t total_tokens;
    int32_t max_seqlen, rows, runs;  // runs: of the longest sequence (PACKED: of all rows)
    Divider rdiv;                    // runs
};
constexpr int kMaxRows = kU * kMoveThreads / 4;  // of a workgroup: 4 chunks a row at least

// First row and rows of a sequence that the page table has a place for.
__device__ __forceinline__ int32_t new_rows(const AppendParams& p, int seq, int32_t ctx, int32_t& s0) {
    s0 = p.cu ? p.cu[seq] : seq;
    const int32_t s1 = p.cu ? p.cu[seq + 1] : seq + 1;
    int32_t n = s1 - s0;
    if (s0 < 0 || s1 < s0 || (int64_t)s1 > p.total_tokens || ctx < 0) n = 0;
    n = min(n, p.max_seqlen);
    return max(0, min(n, p.pg.capacity - ctx));
}

template <bool PACKED>

__global__ __launch_bounds__(kMoveThreads) void kv_append_kernel(AppendParams p) {
    const PageParams& g = p.pg;
    __shared__ int32_t at_seq[PACKED ? kMaxRows : 1], at_pos[PACKED ? kMaxRows : 1];  // the rows' sequences, positions
    int32_t seq = 0, ctx = 0, s0 = 0, first, todo;
    if constexpr (PACKED) {
        first = blockIdx.x * p.rows;
        const int rows = (int)min((int64_t)p.rows, p.total_tokens - first);
        for (int r = threadIdx.x; r < rows; r += kMoveThreads) at_seq[r] = -1;
        __syncthreads();
        // a lane per sequence, every wave its part of the rows
        const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
        for (int c = 0; c < g.B; c += 64) {
            const int s = c + lane;
            int32_t x0 = 0, x = 0, n = 0;
            if (s < g.B) {
                x = g.ctx[s];
                n = new_rows(p, s, x, x0);
                if (blockIdx.x == 0 && wave == 0) g.new_lens[s] = x + n;
            }
            if (!__any(x0 < first + rows && x0 + n > first)) continue;
            for (int r = wave; r < rows; r += kMoveThreads / 64) {
                const int32_t i = first + r - x0;
                if (i >= 0 && i < n) at_seq[r] = s, at_pos[r] = x + i;
            }
        }
        __syncthreads();
        todo = rows * g.chunks;
    } else {
        seq = divide(blockIdx.x, p.rdiv);
        const int run = blockIdx.x - seq * p.runs;
        ctx = g.ctx[seq];
        const int32_t n = new_rows(p, seq, ctx, s0);
        if (run == 0 && threadIdx.x == 0) g.new_lens[seq] = ctx + n;
        first = run * p.rows;
        todo = min(n - first, p.rows) * g.chunks;
    }
    for (int32_t e0 = threadIdx.x; e0 < todo; e0 += kU * kMoveThreads) {
        Vec16 kv[kU], vv[kU];
        int64_t ko[kU], vo[kU];
        bool ok[kU];
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            const int32_t e = e0 + u * kMoveThreads;
            ok[u] = e < todo;
            if (ok[u]) {
                const int32_t row = divide(e, g.cdiv);
                const int32_t rest = e - row * g.chunks;
                const int32_t h = rest >> g.dvshift, c = 8 * (rest & ((1 << g.dvshift) - 1));
                const int64_t t = (int64_t)s0 + first + row;
                kv[u] = ld16_once(p.k + t * p.sk_t + h * p.sk_h + c);
                vv[u] = ld16_once(p.v + t * p.sv_t + h * p.sv_h + c);
                if constexpr (PACKED) {
                    seq = at_seq[row];
                    ok[u] = seq >= 0 && slot_of(g, seq, at_pos[row], ko[u], vo[u]);
                } else {
                    ok[u] = slot_of(g, seq, ctx + first + row, ko[u], vo[u]);
                }
                ko[u] += h * g.sk_head + c;
                vo[u] += h * g.sv_head + c;
            }
        }
#pragma unroll
        for (int u = 0; u < kU; ++u) {
            if (ok[u]) {
                st16_once(g.kc + ko[u], kv[u]);
                st16_once(g.vc + vo[u], vv[u]);
            }
        }
    }
}

// ---------------------------------------------------------------------------
// compact: workgroup (layer, sequence, run of 2 * chunks K and V chunks); a
// thread owns one 16-byte column of the sequence's rows and moves it down the
// path, kStep rows requested before the first is stored.  The path is
// strictly increasing, so node j >= j: a row is read before any row at or
// above it is written, and threads share no byte.
//
// Lane j of every wave holds step j of the path, its rows' pages and offsets:
// the path is one load and the pages are two, side by side.  (Read one after
// the other by all lanes they took most of the call: 48 paths of up to 8 nodes
// in 32 layers 16.0 us, so 11.7.)
// ---------------------------------------------------------------------------
struct CompactParams {
    PageParams pg;
    const int32_t* path;  // [B, cols]
    int32_t cols, parts;
    Divider ptdiv, bdiv;  // parts, B
};

// Lane i's value to all lanes (i uniform).
__device__ __forceinline__ int64_t from_lane(int64_t x, int i) {
    const uint32_t lo = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)x, i);
    const uint32_t hi = (uint32_t)__builtin_amdgcn_readlane((int)(uint32_t)((uint64_t)x >> 32), i);
    return (int64_t)((uint64_t)hi << 32 | lo);
}

__global__ __launch_bounds__(kMoveThreads) void kv_compact_kernel(CompactParams p) {
    const PageParams& g = p.pg;
    const int r0 = divide(blockIdx.x, p.ptdiv);
    const int part = blockIdx.x - r0 * p.parts;
    const int layer = divide(r0, p.bdiv);
    const int seq = r0 - layer * p.pg.B;
    const int32_t ctx = g.ctx[seq];
    const int32_t* path = p.path + (int64_t)seq * p.cols;
    const int lane = threadIdx.x & 63;
    const int32_t e = part * kMoveThreads + threadIdx.x;
    const bool is_v = e >= g.chunks;
    const bool live = e < 2 * g.chunks;
    const int32_t rest = is_v ? e - g.chunks : e;
    const int32_t h = rest >> g.dvshift, c = 8 * (rest & ((1 << g.dvshift) - 1));
    uint16_t* const base = is_v ? g.vc + layer * g.sv_layer + h * g.sv_head + c
                                : g.kc + layer * g.sk_layer + h * g.sk_head + c;
    constexpr int kStep = 8;
    int32_t count = 0, last = -1;
    for (int32_t c0 = 0; c0 < p.cols && ctx >= 0; c0 += 64) {
        const int32_t node = c0 + lane < p.cols ? path[c0 + lane] : -1;
        int32_t before = __shfl_up(node, 1);
        if (lane == 0) before = last;
        // the path goes on as far as every entry rises and has a column
        // (positions stay below 2^30)
        const uint64_t rises = __ballot(node > before && node < g.capacity - ctx);
        const int n = ~rises ? __builtin_ctzll(~rises) : 64;
        int64_t ks = 0, vs = 0, kd = 0, vd = 0;
        bool have = false;
        if (lane < n) {
            have = slot_of(g, seq, ctx + node, ks, vs);
            have = slot_of(g, seq, ctx + c0 + lane, kd, vd) && have && node != c0 + lane;
        }
        const uint64_t moves = __ballot(have);
        for (int j = 0; j < n; j += kStep) {
            Vec16 x[kStep];
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                if (j + u < n && moves >> (j + u) & 1) {
                    const int64_t k = from_lane(ks, j + u), v = from_lane(vs, j + u);
                    if (live) x[u] = ld16(base + (is_v ? v : k));
                }
            }
#pragma unroll
            for (int u = 0; u < kStep; ++u) {
                if (j + u < n && moves >> (j + u) & 1) {
                    const int64_t k = from_lane(kd, j + u), v = from_lane(vd, j + u);
                    if (live) st16(base + (is_v ? v : k), x[u]);
                }
            }
        }
        count += n;
        if (n < 64) break;
        last = __builtin_amdgcn_readlane(node, 63);
    }
    if (layer == 0 && part == 0 && threadIdx.x == 0) g.new_lens[seq] = ctx + count;
}

// ---------------------------------------------------------------------------
// copy: workgroup (layer, pair of pages, run of 16-byte chunks of the page)
// ---------------------------------------------------------------------------
struct CopyParams {
    PageParams pg;
    const int32_t* src;
    const int32_t* dst;
    int32_t n, page_chunks, parts;  // page_chunks: 16-byte chunks of one K page
    Divider ptdiv, ndiv;            // parts, n
};

constexpr int kCopyU = 2;

__global__ __launch_bounds__(kMoveThreads) void kv_copy_kernel(CopyParams p) {
    const PageParams& g = p.pg;
    const int r0 = divide(blockIdx.x, p.ptdiv);
    const int part = blockIdx.x - r0 * p.parts;
    const int layer = divide(r0, p.ndiv);
    const int i = r0 - layer * p.n;
    const int32_t a = p.src[i], b = p.dst[i];
    if ((uint32_t)a >= (uint32_t)g.num_pages || (uint32_t)b >= (uint32_t)g.num_pages || a == b) return;
    const uint16_t* ks = g.kc + layer * g.sk_layer + a * g.sk_page;
    const uint16_t* vs = g.vc + layer * g.sv_layer + a * g.sv_page;
    uint16_t* kd = g.kc + layer * g.sk_layer + b * g.sk_page;
    uint16_t* vd = g.vc + layer * g.sv_layer + b * g.sv_page;
    Vec16 kv[kCopyU], vv[kCopyU];
    int64_t ko[kCopyU], vo[kCopyU];
#pragma unroll
    for (int u = 0; u < kCopyU; ++u) {
        const int32_t e = (part * kCopyU + u) * kMoveThreads + threadIdx.x;
        if (e < p.page_chunks) {
            const int32_t slot = divide(e, g.cdiv);
            const int32_t rest = e - slot * g.chunks;
            const int32_t h = rest >> g.dvshift, c = 8 * (rest & ((1 << g.dvshift) - 1));
            ko[u] = slot * g.sk_slot + h * g.sk_head + c;
            vo[u] = slot * g.sv_slot + h * g.sv_head + c;
            kv[u] = ld16_once(ks + ko[u]);
            vv[u] = ld16_once(vs + vo[u]);
        }
    }
#pragma unroll
    for (int u = 0; u < kCopyU; ++u) {
        if ((part * kCopyU + u) * kMoveThreads + (int32_t)threadIdx.x < p.page_chunks) {
            st16_once(kd + ko[u], kv[u]);
            st16_once(vd + vo[u], vv[u]);
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
// Checks and fills what the three calls share.  stride: {layer, page, slot,
// head, dim}.
static int fill_pages(PageParams& p, void* kc, const int64_t* ks, void* vc, const int64_t* vs, int32_t num_layers,
                      int32_t num_pages, int32_t page_size, int32_t hkv, int32_t head_dim, int32_t dtype) {
    if (dtype != QATTN_DTYPE_F16 && dtype != QATTN_DTYPE_BF16) {
        set_error("dtype %d is not fp16 (0) or bf16 (1)", dtype);
        return QATTN_ERR_DTYPE;
    }
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) {
        set_error("head_dim %d not in {32, 64, 128}", head_dim);
        return QATTN_ERR_HEAD_DIM;
    }
    if (num_layers < 0 || num_pages < 0 || page_size < 1 || hkv < 1 || hkv > (1 << 16)) {
        set_error("bad cache sizes: num_layers=%d num_pages=%d page_size=%d num_kv_heads=%d", num_layers, num_pages,
                  page_size, hkv);
        return QATTN_ERR_ARG;
    }
    if (!ks || !vs) {
        set_error("null stride array");
        return QATTN_ERR_ARG;
    }
    p = PageParams{};
    p.chunks = hkv * (head_dim / 8);
    if ((int64_t)page_size * p.chunks >= (int64_t(1) << 30)) {
        set_error("a page of %d rows of %d heads is too large", page_size, hkv);
        return QATTN_ERR_ARG;
    }
    if ((num_layers > 0 && num_pages > 0) && (!kc || !vc)) {
        set_error("null cache pointer");
        return QATTN_ERR_ARG;
    }
    if (!row_aligned(kc, ks, 4) || !row_aligned(vc, vs, 4)) {
        set_error("k/v cache rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    p.kc = (uint16_t*)kc;
    p.vc = (uint16_t*)vc;
    p.sk_layer = ks[0], p.sk_page = ks[1], p.sk_slot = ks[2], p.sk_head = ks[3];
    p.sv_layer = vs[0], p.sv_page = vs[1], p.sv_slot = vs[2], p.sv_head = vs[3];
    p.num_pages = num_pages;
    p.page_size = page_size;
    p.pdiv = make_divider(page_size);
    p.cdiv = make_divider(p.chunks);
    p.dvshift = head_dim == 32 ? 2 : head_dim == 64 ? 3 : 4;
    return QATTN_OK;
}

static int fill_table(PageParams& p, const int32_t* table, int32_t pt_cols, const int32_t* ctx, int32_t* new_lens,
                      int32_t batch) {
    if (batch < 0 || pt_cols < 0 || (int64_t)pt_cols * p.page_size > kMaxPositions) {
        set_error("bad page table: batch=%d pt_cols=%d page_size=%d", batch, pt_cols, p.page_size);
        return QATTN_ERR_ARG;
    }
    if (batch > 0 && (!ctx || !new_lens || (!table && pt_cols > 0))) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    p.table = table;
    p.ctx = ctx;
    p.new_lens = new_lens;
    p.pt_cols = pt_cols;
    p.capacity = pt_cols * p.page_size;
    p.B = batch;
    return QATTN_OK;
}

static int grid_of(int64_t blocks) {
    if (blocks > INT32_MAX) {
        set_error("grid too large (%lld blocks)", (long long)blocks);
        return -1;
    }
    return (int)blocks;
}

}  // namespace qattn

using namespace qattn;

extern "C" {

int qattn_kv_append(const void* k, const int64_t k_stride[3], const void* v, const int64_t v_stride[3],
                    void* k_cache, const int64_t kc_stride[5], void* v_cache, const int64_t vc_stride[5],
                    const int32_t* page_table, int32_t pt_cols, int32_t num_pages, int32_t page_size,
                    const int32_t* context_lens, int32_t* new_lens, const int32_t* cu_seqlens, int32_t batch,
                    int32_t max_seqlen, int64_t total_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                    void* stream) {
    clear_error();
    if (!kc_stride || !vc_stride || !k_stride || !v_stride) {
        set_error("null stride array");
        return QATTN_ERR_ARG;
    }
    AppendParams p{};
    int rc = fill_pages(p.pg, k_cache, kc_stride, v_cache, vc_stride, 1, num_pages, page_size, num_kv_heads, head_dim, dtype);
    if (rc) return rc;
    rc = fill_table(p.pg, page_table, pt_cols, context_lens, new_lens, batch);
    if (rc) return rc;
    if (max_seqlen < 0 || total_tokens < 0 || total_tokens >= (int64_t(1) << 31)) {
        set_error("bad sizes: max_seqlen=%d total_tokens=%lld", max_seqlen, (long long)total_tokens);
        return QATTN_ERR_ARG;
    }
    if (batch == 0) return QATTN_OK;
    if (total_tokens > 0 && (!k || !v)) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    if (!row_aligned(k, k_stride, 2) || !row_aligned(v, v_stride, 2)) {
        set_error("k/v rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    p.k = (const uint16_t*)k;
    p.v = (const uint16_t*)v;
    p.sk_t = k_stride[0], p.sk_h = k_stride[1];
    p.sv_t = v_stride[0], p.sv_h = v_stride[1];
    p.cu = cu_seqlens;
    p.total_tokens = total_tokens;
    p.max_seqlen = (int32_t)std::min<int64_t>({cu_seqlens ? max_seqlen : 1, total_tokens, p.pg.capacity});
    // a workgroup's rows: one round of kU chunks of K and V per thread, at least one row
    p.rows = std::max(1, kU * kMoveThreads / p.pg.chunks);
    p.runs = std::max(1, (int32_t)(((int64_t)p.max_seqlen + p.rows - 1) / p.rows));
    p.rdiv = make_divider(p.runs);
    const int64_t packed = (total_tokens + p.rows - 1) / p.rows;
    if (cu_seqlens && packed > 0 && (int64_t)batch * p.runs > 4 * packed) {
        hipLaunchKernelGGL(kv_append_kernel<true>, dim3((uint32_t)packed), dim3(kMoveThreads), 0, (hipStream_t)stream, p);
        return launch_status("kv_append_kernel, packed rows");
    }
    const int grid = grid_of((int64_t)batch * p.runs);
    if (grid < 0) return QATTN_ERR_ARG;
    hipLaunchKernelGGL(kv_append_kernel<false>, dim3(grid), dim3(kMoveThreads), 0, (hipStream_t)stream, p);
    return launch_status("kv_append_kernel");
}

int qattn_kv_compact(void* k_cache, const int64_t kc_stride[5], void* v_cache, const int64_t vc_stride[5],
                     int32_t num_layers, const int32_t* page_table, int32_t pt_cols, int32_t num_pages,
                     int32_t page_size, const int32_t* context_lens, const int32_t* accepted, int32_t path_cols,
                     int32_t* new_lens, int32_t batch, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                     void* stream) {
    clear_error();
    CompactParams p{};
    int rc = fill_pages(p.pg, k_cache, kc_stride, v_cache, vc_stride, num_layers, num_pages, page_size, num_kv_heads,
                        head_dim, dtype);
    if (rc) return rc;
    rc = fill_table(p.pg, page_table, pt_cols, context_lens, new_lens, batch);
    if (rc) return rc;
    if (path_cols < 0 || (path_cols > 0 && batch > 0 && !accepted) || num_layers < 1) {
        set_error("bad path: path_cols=%d num_layers=%d", path_cols, num_layers);
        return QATTN_ERR_ARG;
    }
    if (batch == 0) return QATTN_OK;
    p.path = accepted;
    p.cols = path_cols;
    p.parts = (2 * p.pg.chunks + kMoveThreads - 1) / kMoveThreads;
    p.ptdiv = make_divider(p.parts);
    p.bdiv = make_divider(batch);
    const int grid = grid_of((int64_t)num_layers * batch * p.parts);
    if (grid < 0) return QATTN_ERR_ARG;
    hipLaunchKernelGGL(kv_compact_kernel, dim3(grid), dim3(kMoveThreads), 0, (hipStream_t)stream, p);
    return launch_status("kv_compact_kernel");
}

int qattn_kv_copy_pages(void* k_cache, const int64_t kc_stride[5], void* v_cache, const int64_t vc_stride[5],
                        int32_t num_layers, int32_t num_pages, int32_t page_size, const int32_t* src_pages,
                        const int32_t* dst_pages, int32_t n, int32_t num_kv_heads, int32_t head_dim, int32_t dtype,
                        void* stream) {
    clear_error();
    CopyParams p{};
    const int rc = fill_pages(p.pg, k_cache, kc_stride, v_cache, vc_stride, num_layers, num_pages, page_size,
                              num_kv_heads, head_dim, dtype);
    if (rc) return rc;
    if (n < 0 || (n > 0 && (!src_pages || !dst_pages))) {
        set_error("bad page list (n=%d)", n);
        return QATTN_ERR_ARG;
    }
    if (n == 0 || num_layers == 0 || num_pages == 0) return QATTN_OK;
    p.src = src_pages;
    p.dst = dst_pages;
    p.n = n;
    p.page_chunks = page_size * p.pg.chunks;
    p.parts = (p.page_chunks + kCopyU * kMoveThreads - 1) / (kCopyU * kMoveThreads);
    p.ptdiv = make_divider(p.parts);
    p.ndiv = make_divider(n);
    const int grid = grid_of((int64_t)num_layers * n * p.parts);
    if (grid < 0) return QATTN_ERR_ARG;
    hipLaunchKernelGGL(kv_copy_kernel, dim3(grid), dim3(kMoveThreads), 0, (hipStream_t)stream, p);
    return launch_status("kv_copy_kernel");
}

}  // extern "C"
