// kv_tiles.h -- K/V blocks in LDS, as the dense attention kernels share them:
// the 16-byte chunk swizzles and the global -> LDS load.
#pragma once

#include "qattn_device.h"

namespace qattn {

// 16-byte chunk swizzle of the K/V blocks in LDS: chunk c of key row r sits at
// position c ^ kv_swz(r) of its (unpadded) row.  With 256-byte rows both
// operand reads are bank-conflict free on gfx950 (probed with
// SQ_LDS_BANK_CONFLICT): the K reads (ds_read_b128, rows 16 mt + l16, chunk
// 4 c + lq) and the V^T reads (ds_read_b64_tr_b16, 8 rows of 32 bytes per
// 32-lane pass).  Smaller head dims keep the low bits (correct, not probed).
__device__ __forceinline__ int kv_swz(int r, int dv) {
    const int b2 = (r >> 2) & 1, b3 = (r >> 3) & 1;
    return ((2 * (r & 3)) | (8 * (b3 ^ b2)) | b2) & (dv - 1);
}

// Chunk swizzle of the K/V blocks of the 32x32x16 prefix kernel: chunk c of
// key row r sits at c ^ kv_swz32(r).  Its K operand reads (ds_read_b128, 16
// consecutive rows at one chunk per 16-lane pass) need 16 distinct positions
// for rows r..r+15, which a bijection on r & 15 gives; its V^T operand reads
// (ds_read_b64_tr_b16, per 32-lane pass 4 consecutive rows x one aligned
// group of 4 chunks) need the 4 rows in distinct groups, which 4 (r & 3)
// gives.  (Positions checked on the CPU for every pass at D = 128.)
__device__ __forceinline__ int kv_swz32(int r, int dv) { return ((4 * (r & 3)) | ((r >> 2) & 3)) & (dv - 1); }

// s_waitcnt immediate (gfx9 encoding): vmcnt N, expcnt and lgkmcnt unconstrained
constexpr int kWaitVm(int n) { return (n & 15) | ((n >> 4) << 14) | (7 << 4) | (15 << 8); }

// One 1 KB global -> LDS load: global_load_lds_dwordx4 with a wave-uniform
// base in SGPRs and a 32-bit per-lane byte offset (lane i writes bytes
// [16 i, 16 i + 16) of the LDS run at dst), so issuing it costs no vector ALU
// work.  Written as an asm statement, which also keeps the compiler's wait
// analysis precise: it treats a pending LDS-DMA load as an out-of-order LDS
// event and would otherwise wait for every LDS read in flight
// (lgkmcnt(0)) before each use of one.  The kernel orders these loads itself
// (s_waitcnt vmcnt + barrier before a buffer is read, barrier before it is
// overwritten).
// RFL: take the base and destination through readfirstlane, for code where
// the compiler cannot prove them wave-uniform on its own (each 32-bit half
// widened as unsigned: readfirstlane returns int).
template <bool RFL = false>
__device__ __forceinline__ void lds_dma16(uint32_t voff, const char* sbase, void* dst) {
    uint32_t lds = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) void*)dst;
    if constexpr (RFL) {
        const uint64_t a = (uint64_t)(uintptr_t)sbase;
        const uint32_t lo = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)a);
        const uint32_t hi = (uint32_t)__builtin_amdgcn_readfirstlane((int)(uint32_t)(a >> 32));
        sbase = (const char*)(uintptr_t)(((uint64_t)hi << 32) | (uint64_t)lo);
        lds = (uint32_t)__builtin_amdgcn_readfirstlane((int)lds);
    }
    // M0 (the LDS destination) is an operand the compiler allocates ("{m0}"),
    // so it writes M0 itself and knows its value afterwards
    asm volatile("global_load_lds_dwordx4 %0, %1" ::"v"(voff), "s"(sbase), "{m0}"(lds) : "memory");
}

}  // namespace qattn
