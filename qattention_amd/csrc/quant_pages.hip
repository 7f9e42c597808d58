// quant_pages.hip -- rows into and out of a paged cache that is held in 4 or 8
// bits (quant_format.h): new K/V rows quantised behind each context, positions
// of a context read back as 16-bit rows.
//
// A thread has 8 elements of K and of V at a time, a quad of lanes a block of 32
// with its scale.  Both directions are bound by HBM in large calls (16 bits per
// element on one side, 4.25 or 8.25 on the other: 8 x 4003 rows of 8 heads of 128
// in 4 bits, 166 MB, are written in 31.5 us, 5.3 TB/s, what a copy reaches; 16
// contexts of 10007 read back, 835 MB, in 144) and by their launch and one chain of
// dependent loads (offsets, context length, page, row) in small ones (32 x 1 rows:
// 2.7 and 2.5 us).
#include <algorithm>

#include "qattn_common.h"
#include "quant_format.h"

namespace qattn {

constexpr int kRowThreads = 256;

struct QuantPageParams {
    uint8_t *kc, *vc, *ks, *vs;             // elements and scales of the cache
    int64_t sc_page, sc_slot, sc_head;      // bytes; K and V alike
    int64_t ss_page, ss_slot, ss_head;
    uint16_t *k, *v;                        // packed 16-bit rows
    int64_t sk_t, sk_h, sv_t, sv_h;
    const int32_t* table;                   // [B, pt_cols]
    const int32_t* ctx;                     // [B]: the position of each sequence's first row
    const int32_t* cu;                      // null: row s belongs to sequence s
    int32_t* new_lens;                      // [B]
    int64_t total_tokens;
    int32_t B, pt_cols, num_pages, page_size, capacity, max_seqlen;
    int32_t chunks;                         // 8-element chunks of one token's K row (all heads)
    int32_t dvshift;                        // chunks of one head's row: 1 << dvshift
    int32_t rows, runs;                     // of a workgroup; workgroups of the longest sequence
    Divider pdiv, cdiv, rdiv;               // page_size, chunks, runs
};

typedef uint32_t u4_t __attribute__((ext_vector_type(4)));
__device__ __forceinline__ Vec16 ld16_once(const void* p) {
    const u4_t x = __builtin_nontemporal_load(reinterpret_cast<const u4_t*>(p));
    return Vec16{{x[0], x[1], x[2], x[3]}};
}
__device__ __forceinline__ void st16_once(void* p, const Vec16& v) {
    const u4_t x = {v.w[0], v.w[1], v.w[2], v.w[3]};
    __builtin_nontemporal_store(x, reinterpret_cast<u4_t*>(p));
}

// Rows of a sequence and its first packed row; bad offsets give none.
__device__ __forceinline__ int32_t rows_of(const QuantPageParams& p, int seq, int32_t& s0) {
    s0 = p.cu ? p.cu[seq] : seq;
    const int32_t s1 = p.cu ? p.cu[seq + 1] : seq + 1;
    if (s0 < 0 || s1 < s0 || (int64_t)s1 > p.total_tokens) return 0;
    return min(s1 - s0, p.max_seqlen);
}

// The workgroup's packed rows: first + r, r < count, of sequence seq(r) at
// position pos(r).  PACKED: `rows` rows of whichever sequences (seq -1: of none);
// otherwise a run of one sequence's rows.
// Chunks of K and of V per thread and round.  (Two keep more loads in flight, 16 x 10007
// rows read back: 144 us, with one 151, with four 151.  Calls of fewer than kFull
// workgroups get half the rows per workgroup and leave the second chunk out: append 1 x
// 731: 3.2 us, with two 4.1; 63 x 1 and one of 2000: 5.3, 5.8; from there on the other
// way round, 7 x 1 and one of 8000: 11.9, 11.1.)
constexpr int kUnits = 2;
constexpr int kFull = 1024;
constexpr int kMaxRows = kUnits * kRowThreads / 4;          // of a workgroup: 4 chunks a row at least
template <bool PACKED, bool APPEND>
struct WorkRows {
    int64_t first;
    int32_t count, seq0, pos0;
    const int32_t *at_seq, *at_pos;

    __device__ __forceinline__ WorkRows(const QuantPageParams& p, int32_t* seqs, int32_t* poss) {
        at_seq = seqs, at_pos = poss;
        // rows that are there; a position that the table has no column for takes none
        auto there = [&](int32_t n, int32_t ctx) {
            if constexpr (APPEND) return ctx < 0 ? 0 : max(0, min(n, p.capacity - ctx));
            return n;
        };
        if constexpr (PACKED) {
            first = (int64_t)blockIdx.x * p.rows;
            count = (int32_t)min((int64_t)p.rows, p.total_tokens - first);
            for (int r = threadIdx.x; r < count; r += kRowThreads) seqs[r] = -1;
            __syncthreads();
            // a lane per sequence, every wave its part of the rows
            const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
            for (int c = 0; c < p.B; c += 64) {
                const int s = c + lane;
                int32_t x0 = 0, x = 0, n = 0;
                if (s < p.B) {
                    x = p.ctx[s];
                    n = there(rows_of(p, s, x0), x);
                    if (APPEND && blockIdx.x == 0 && wave == 0) p.new_lens[s] = x + n;
                }
                if (!__any(n > 0 && x0 < first + count && (int64_t)x0 + n > first)) continue;
                for (int r = wave; r < count; r += kRowThreads / 64) {
                    const int64_t i = first + r - x0;
                    if (i >= 0 && i < n) seqs[r] = s, poss[r] = (int32_t)((uint32_t)x + (uint32_t)i);
                }
            }
            __syncthreads();
        } else {
            seq0 = divide(blockIdx.x, p.rdiv);
            const int run = blockIdx.x - seq0 * p.runs;
            const int32_t ctx = p.ctx[seq0];
            int32_t s0;
            const int32_t n = there(rows_of(p, seq0, s0), ctx);
            if (APPEND && run == 0 && threadIdx.x == 0) p.new_lens[seq0] = ctx + n;
            const int32_t from = run * p.rows;
            first = (int64_t)s0 + from;
            pos0 = (int32_t)((uint32_t)ctx + (uint32_t)from);
            count = max(0, min(n - from, p.rows));
        }
    }
    __device__ __forceinline__ int32_t seq(int r) const {
        if constexpr (PACKED) return at_seq[r];
        return seq0;
    }
    // (a position that wraps is negative or past the capacity, at most 2^30: no place)
    __device__ __forceinline__ int32_t pos(int r) const {
        if constexpr (PACKED) return at_pos[r];
        return (int32_t)((uint32_t)pos0 + (uint32_t)r);
    }
};

// Byte offsets of position pos of sequence seq (head 0) among the elements and
// the scales; false: it has no place in the cache.
__device__ __forceinline__ bool place_of(const QuantPageParams& p, int seq, int32_t pos, int64_t& at, int64_t& scale) {
    if ((uint32_t)pos >= (uint32_t)p.capacity) return false;
    const int32_t col = divide(pos, p.pdiv);
    const int32_t page = p.table[(int64_t)seq * p.pt_cols + col];
    const int32_t slot = pos - col * p.page_size;
    at = (int64_t)page * p.sc_page + (int64_t)slot * p.sc_slot;
    scale = (int64_t)page * p.ss_page + (int64_t)slot * p.ss_slot;
    return (uint32_t)page < (uint32_t)p.num_pages;
}

template <int BITS>
struct Words {
    uint32_t w[BITS / 4];
};
template <int BITS>
__device__ __forceinline__ Words<BITS> ld_words(const uint8_t* p) {
    Words<BITS> r;
    if constexpr (BITS == 4) {
        r.w[0] = *reinterpret_cast<const uint32_t*>(p);
    } else {
        const uint2 x = *reinterpret_cast<const uint2*>(p);
        r.w[0] = x.x, r.w[1] = x.y;
    }
    return r;
}
template <int BITS>
__device__ __forceinline__ void st_words(uint8_t* p, const Words<BITS>& x) {
    if constexpr (BITS == 4)
        *reinterpret_cast<uint32_t*>(p) = x.w[0];
    else
        *reinterpret_cast<uint2*>(p) = make_uint2(x.w[0], x.w[1]);
}

template <typename T, int BITS, bool PACKED>
__global__ __launch_bounds__(kRowThreads) void quant_append_kernel(QuantPageParams p) {
    __shared__ int32_t seqs[PACKED ? kMaxRows : 1], poss[PACKED ? kMaxRows : 1];
    const WorkRows<PACKED, true> rows(p, seqs, poss);
    const int32_t todo = rows.count * p.chunks;
    // (chunks of a row are a multiple of 4, so a quad of lanes is one block or idle)
    for (int32_t e0 = threadIdx.x; e0 < todo; e0 += kUnits * kRowThreads) {
        Vec16 x[2][kUnits];
        int64_t at[kUnits], sc[kUnits];
        bool ok[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int32_t e = e0 + u * kRowThreads;
            ok[u] = e < todo;
            if (ok[u]) {
                const int32_t row = divide(e, p.cdiv);
                const int32_t rest = e - row * p.chunks;
                const int32_t h = rest >> p.dvshift, c = rest & ((1 << p.dvshift) - 1);
                const int64_t t = rows.first + row;
                x[0][u] = ld16_once(p.k + t * p.sk_t + h * p.sk_h + 8 * c);
                x[1][u] = ld16_once(p.v + t * p.sv_t + h * p.sv_h + 8 * c);
                const int32_t seq = rows.seq(row);
                ok[u] = seq >= 0 && place_of(p, seq, rows.pos(row), at[u], sc[u]);
                at[u] += h * p.sc_head + c * BITS;
                sc[u] += h * p.ss_head + (c >> 2);
            }
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (ok[u]) {
                Words<BITS> w;
                uint32_t code = narrow8<T, BITS>(x[0][u], w.w);
                st_words<BITS>(p.kc + at[u], w);
                if ((threadIdx.x & 3) == 0) p.ks[sc[u]] = (uint8_t)code;
                code = narrow8<T, BITS>(x[1][u], w.w);
                st_words<BITS>(p.vc + at[u], w);
                if ((threadIdx.x & 3) == 0) p.vs[sc[u]] = (uint8_t)code;
            }
        }
    }
}

template <typename T, int BITS, bool PACKED>
__global__ __launch_bounds__(kRowThreads) void quant_read_kernel(QuantPageParams p) {
    __shared__ int32_t seqs[PACKED ? kMaxRows : 1], poss[PACKED ? kMaxRows : 1];
    const WorkRows<PACKED, false> rows(p, seqs, poss);
    const int32_t todo = rows.count * p.chunks;
    for (int32_t e0 = threadIdx.x; e0 < todo; e0 += kUnits * kRowThreads) {
        Words<BITS> w[2][kUnits];
        uint32_t code[2][kUnits];
        int64_t ko[kUnits], vo[kUnits];
        bool ok[kUnits];
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            const int32_t e = e0 + u * kRowThreads;
            ok[u] = e < todo;
            if (ok[u]) {
                const int32_t row = divide(e, p.cdiv);
                const int32_t rest = e - row * p.chunks;
                const int32_t h = rest >> p.dvshift, c = rest & ((1 << p.dvshift) - 1);
                const int64_t t = rows.first + row;
                ko[u] = t * p.sk_t + h * p.sk_h + 8 * c;
                vo[u] = t * p.sv_t + h * p.sv_h + 8 * c;
                const int32_t seq = rows.seq(row);
                ok[u] = seq >= 0;
                int64_t at, sc;
#pragma unroll
                for (int i = 0; i < BITS / 4; ++i) w[0][u].w[i] = w[1][u].w[i] = 0;
                code[0][u] = code[1][u] = 127;  // (a position without a place reads as zeros)
                if (ok[u] && place_of(p, seq, rows.pos(row), at, sc)) {
                    at += h * p.sc_head + c * BITS;
                    sc += h * p.ss_head + (c >> 2);
                    w[0][u] = ld_words<BITS>(p.kc + at);
                    w[1][u] = ld_words<BITS>(p.vc + at);
                    code[0][u] = p.ks[sc];
                    code[1][u] = p.vs[sc];
                }
            }
        }
#pragma unroll
        for (int u = 0; u < kUnits; ++u) {
            if (ok[u]) {
                st16_once(p.k + ko[u], widen8<T, BITS>(w[0][u].w, scale_of(code[0][u])));
                st16_once(p.v + vo[u], widen8<T, BITS>(w[1][u].w, scale_of(code[1][u])));
            }
        }
    }
}

// ---------------------------------------------------------------------------
// Host side
// ---------------------------------------------------------------------------
int check_quant(const void* kc, const void* vc, const int64_t* cs, const void* ks, const void* vs, const int64_t* ss,
                int32_t pt_cols, int32_t num_pages, int32_t page_size, int32_t hkv, int32_t head_dim, int32_t dtype,
                int32_t bits) {
    if (dtype != QATTN_DTYPE_F16 && dtype != QATTN_DTYPE_BF16) {
        set_error("dtype %d is not fp16 (0) or bf16 (1)", dtype);
        return QATTN_ERR_DTYPE;
    }
    if (bits != 4 && bits != 8) {
        set_error("a cache of %d bits: neither 4 nor 8", bits);
        return QATTN_ERR_DTYPE;
    }
    if (head_dim != 32 && head_dim != 64 && head_dim != 128) {
        set_error("head_dim %d not in {32, 64, 128}", head_dim);
        return QATTN_ERR_HEAD_DIM;
    }
    if (num_pages < 0 || page_size < 1 || hkv < 1 || hkv > (1 << 16) || pt_cols < 0 ||
        (int64_t)pt_cols * page_size > kMaxPositions) {
        set_error("bad cache sizes: num_pages=%d page_size=%d num_kv_heads=%d pt_cols=%d", num_pages, page_size, hkv,
                  pt_cols);
        return QATTN_ERR_ARG;
    }
    if (!cs || !ss || (num_pages > 0 && (!kc || !vc || !ks || !vs))) {
        set_error("null cache pointer or stride array");
        return QATTN_ERR_ARG;
    }
    const int64_t unit = head_dim / kQuantBlock;  // bytes of one head's scales: read together
    if (cs[3] != 1 || (cs[0] | cs[1] | cs[2]) & 15 || ((uintptr_t)kc | (uintptr_t)vc) & 15) {
        set_error("elements of the cache must be 16-byte aligned rows with stride_byte 1");
        return QATTN_ERR_LAYOUT;
    }
    if (ss[3] != 1 || (ss[0] | ss[1] | ss[2]) & (unit - 1) || ((uintptr_t)ks | (uintptr_t)vs) & (unit - 1)) {
        set_error("scales must be %lld-byte aligned rows with stride_byte 1", (long long)unit);
        return QATTN_ERR_LAYOUT;
    }
    return QATTN_OK;
}

// Checks and fills what both calls share.  Strides of the cache: {page, slot,
// head, byte}.
static int fill_quant(QuantPageParams& p, const void* kc, const void* vc, const int64_t* cs, const void* ks,
                      const void* vs, const int64_t* ss, const int32_t* table, int32_t pt_cols, int32_t num_pages,
                      int32_t page_size, const int32_t* ctx, const void* k, const int64_t* kst, const void* v,
                      const int64_t* vst, const int32_t* cu, int32_t batch, int32_t max_seqlen, int64_t total_tokens,
                      int32_t hkv, int32_t head_dim, int32_t dtype, int32_t bits) {
    const int rc = check_quant(kc, vc, cs, ks, vs, ss, pt_cols, num_pages, page_size, hkv, head_dim, dtype, bits);
    if (rc) return rc;
    if (batch < 0 || max_seqlen < 0 || total_tokens < 0 || total_tokens >= (int64_t(1) << 31)) {
        set_error("bad sizes: batch=%d max_seqlen=%d total_tokens=%lld", batch, max_seqlen, (long long)total_tokens);
        return QATTN_ERR_ARG;
    }
    if (!kst || !vst || (batch > 0 && (!ctx || (!table && pt_cols > 0))) || (total_tokens > 0 && (!k || !v))) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    if (!row_aligned(k, kst, 2) || !row_aligned(v, vst, 2)) {
        set_error("k/v rows must be 16-byte aligned with stride_dim 1");
        return QATTN_ERR_LAYOUT;
    }
    p = QuantPageParams{};
    p.kc = (uint8_t*)kc, p.vc = (uint8_t*)vc, p.ks = (uint8_t*)ks, p.vs = (uint8_t*)vs;
    p.sc_page = cs[0], p.sc_slot = cs[1], p.sc_head = cs[2];
    p.ss_page = ss[0], p.ss_slot = ss[1], p.ss_head = ss[2];
    p.k = (uint16_t*)k, p.v = (uint16_t*)v;
    p.sk_t = kst[0], p.sk_h = kst[1], p.sv_t = vst[0], p.sv_h = vst[1];
    p.table = table, p.ctx = ctx, p.cu = cu;
    p.total_tokens = total_tokens;
    p.B = batch, p.pt_cols = pt_cols, p.num_pages = num_pages, p.page_size = page_size;
    p.capacity = num_pages > 0 ? pt_cols * page_size : 0;
    p.max_seqlen = (int32_t)std::min<int64_t>(cu ? max_seqlen : 1, total_tokens);
    p.chunks = hkv * (head_dim / 8);
    p.dvshift = head_dim == 32 ? 2 : head_dim == 64 ? 3 : 4;
    const bool full = total_tokens * p.chunks >= (int64_t)kFull * kUnits * kRowThreads;
    p.rows = std::max(1, (full ? kUnits : 1) * kRowThreads / p.chunks);
    p.pdiv = make_divider(page_size);
    p.cdiv = make_divider(p.chunks);
    return QATTN_OK;
}

// Workgroups of one sequence's rows each, or of packed rows, of whichever
// sequences, where most sequences are far shorter than the longest.  (Packed ones
// look every sequence up: append 32 x 1 rows 3.7 us, by sequences 2.7; 8 x 4003 36.9
// and 33.3.  By sequences most workgroups find nothing: 63 x 1 and one of 2000 16.0,
// packed 5.8; 7 x 1 and one of 8000 15.3 and 11.1; 31 x 1 and one of 300 4.4 and 3.9.)
static int row_grid(QuantPageParams& p, int32_t longest, bool& packed, uint32_t& grid) {
    p.runs = std::max(1, (int32_t)(((int64_t)longest + p.rows - 1) / p.rows));
    p.rdiv = make_divider(p.runs);
    const int64_t all = (p.total_tokens + p.rows - 1) / p.rows, each = (int64_t)p.B * p.runs;
    packed = p.cu && all > 0 && each > 4 * all;
    const int64_t n = packed ? all : each;
    if (n > INT32_MAX) {
        set_error("grid too large (%lld blocks)", (long long)n);
        return QATTN_ERR_ARG;
    }
    grid = (uint32_t)n;
    return QATTN_OK;
}

#define QATTN_ROWS(KERNEL, T, BITS)                                                                        \
    do {                                                                                                   \
        if (packed)                                                                                        \
            hipLaunchKernelGGL((KERNEL<T, BITS, true>), dim3(grid), dim3(kRowThreads), 0, st, p);          \
        else                                                                                               \
            hipLaunchKernelGGL((KERNEL<T, BITS, false>), dim3(grid), dim3(kRowThreads), 0, st, p);         \
    } while (0)
#define QATTN_ROWS_ALL(KERNEL)                                                                             \
    do {                                                                                                   \
        if (dtype == QATTN_DTYPE_F16 && bits == 4) QATTN_ROWS(KERNEL, F16, 4);                             \
        else if (dtype == QATTN_DTYPE_F16) QATTN_ROWS(KERNEL, F16, 8);                                     \
        else if (bits == 4) QATTN_ROWS(KERNEL, BF16, 4);                                                   \
        else QATTN_ROWS(KERNEL, BF16, 8);                                                                  \
    } while (0)

}  // namespace qattn

using namespace qattn;

extern "C" {

int qattn_quant_append(const void* k, const int64_t k_stride[3], const void* v, const int64_t v_stride[3],
                       void* k_cache, void* v_cache, const int64_t cache_stride[4], void* k_scale, void* v_scale,
                       const int64_t scale_stride[4], const int32_t* page_table, int32_t pt_cols, int32_t num_pages,
                       int32_t page_size, const int32_t* context_lens, int32_t* new_lens, const int32_t* cu_seqlens,
                       int32_t batch, int32_t max_seqlen, int64_t total_tokens, int32_t num_kv_heads, int32_t head_dim,
                       int32_t dtype, int32_t bits, void* stream) {
    clear_error();
    QuantPageParams p;
    int rc = fill_quant(p, k_cache, v_cache, cache_stride, k_scale, v_scale, scale_stride, page_table, pt_cols,
                        num_pages, page_size, context_lens, k, k_stride, v, v_stride, cu_seqlens, batch, max_seqlen,
                        total_tokens, num_kv_heads, head_dim, dtype, bits);
    if (rc || batch == 0) return rc;
    if (!new_lens) {
        set_error("null pointer argument");
        return QATTN_ERR_ARG;
    }
    // (positions count where the table has a column, whatever pages there are)
    p.capacity = pt_cols * page_size;
    p.new_lens = new_lens;
    bool packed;
    uint32_t grid;
    rc = row_grid(p, std::min(p.max_seqlen, p.capacity), packed, grid);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    QATTN_ROWS_ALL(quant_append_kernel);
    return launch_status("quant_append_kernel");
}

int qattn_quant_read(const void* k_cache, const void* v_cache, const int64_t cache_stride[4], const void* k_scale,
                     const void* v_scale, const int64_t scale_stride[4], const int32_t* page_table, int32_t pt_cols,
                     int32_t num_pages, int32_t page_size, const int32_t* starts, void* k, const int64_t k_stride[3],
                     void* v, const int64_t v_stride[3], const int32_t* cu_seqlens, int32_t batch, int32_t max_seqlen,
                     int64_t total_tokens, int32_t num_kv_heads, int32_t head_dim, int32_t dtype, int32_t bits,
                     void* stream) {
    clear_error();
    QuantPageParams p;
    int rc = fill_quant(p, k_cache, v_cache, cache_stride, k_scale, v_scale, scale_stride, page_table, pt_cols,
                        num_pages, page_size, starts, k, k_stride, v, v_stride, cu_seqlens, batch, max_seqlen,
                        total_tokens, num_kv_heads, head_dim, dtype, bits);
    if (rc || batch == 0 || p.max_seqlen == 0) return rc;
    bool packed;
    uint32_t grid;
    rc = row_grid(p, p.max_seqlen, packed, grid);
    if (rc) return rc;
    hipStream_t st = (hipStream_t)stream;
    QATTN_ROWS_ALL(quant_read_kernel);
    return launch_status("quant_read_kernel");
}

}  // extern "C"
