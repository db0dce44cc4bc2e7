// Device building blocks shared by the kernels with packed INT4 weight rows
// (i4w_gemm.hpp, moe_w4a16.hip): LDS reads and LDS DMA, the nibble unpack, the
// swizzles of the LDS rows.
#pragma once

#include "common.hpp"
#include "f16_dma_gemm.hpp"

namespace clove {
namespace i4w {

using namespace hw;
using dma::dma16;
using dma::make_rsrc;
using dma::vmcnt_imm;

typedef __attribute__((address_space(3))) u32x4 lds_u32x4;
typedef __attribute__((address_space(3))) unsigned lds_u32;

__device__ __forceinline__ u32x4 lds_read16(unsigned addr) {
    return *reinterpret_cast<const lds_u32x4*>((size_t)addr);
}
__device__ __forceinline__ unsigned lds_read4(unsigned addr) {
    return *reinterpret_cast<const lds_u32*>((size_t)addr);
}

// (the wait state after the M0 write, as in dma16)
__device__ __forceinline__ void dma4(const u32x4& rsrc, unsigned lds_addr, int voff, int soff) {
    asm volatile("s_nop 0\n\tbuffer_load_dword %0, %1, %2 offen lds"
                 :
                 : "v"(voff), "s"(rsrc), "s"(soff), "{m0}"(lds_addr)
                 : "memory");
}

// (q - z) * 2^-9 for the 8 nibbles of one dword, in k order; zz = -z * 2^-9, mul what
// takes the two subnormals of a byte to q * 2^-9 (0, and zz 0: makes all of them 0).
// Byte b holds k = 2b and 2b + 1: in the high and low nibble (the weights'
// packing), or with LO_FIRST in the low and high nibble (the order in which
// ds_read_b64_tr_b4 returns k rows)
template <bool LO_FIRST = false>
__device__ __forceinline__ f16x8 unpack8(unsigned w, f16x2 mul, f16x2 zz) {
    const unsigned hr = w & 0xf0f0f0f0u, lo = w & 0x0f0f0f0fu;
    f16x2 v[4];
#pragma unroll
    for (int b = 0; b < 4; ++b) {
        const unsigned sel = LO_FIRST ? 0x0c000c00u | (unsigned)(4 + b) | ((unsigned)b << 16)
                                      : 0x0c000c00u | (unsigned)b | ((unsigned)(4 + b) << 16);
        const f16x2 sub = bitcast<f16x2>(__builtin_amdgcn_perm(lo, hr, sel));
        v[b] = __builtin_elementwise_fma(sub, mul, zz);
    }
    f16x8 r;
    r.s01 = v[0];
    r.s23 = v[1];
    r.s45 = v[2];
    r.s67 = v[3];
    return r;
}
template <bool LO_FIRST = false>
__device__ __forceinline__ f16x8 unpack8(unsigned w, f16x2 zz) {
    return unpack8<LO_FIRST>(w,
                             LO_FIRST ? f16x2{(_Float16)32768.0f, (_Float16)2048.0f}
                                      : f16x2{(_Float16)2048.0f, (_Float16)32768.0f},
                             zz);
}

// A 16-byte LDS read serves 16 lanes per clock from one 256-byte window of
// banks.  The 16 lanes of a fragment read take 16 consecutive rows, one chunk
// each, so the chunk is swizzled by the row bits above those that already
// separate rows within a window:
//   weight rows of 64 bytes (whole group: 4 rows per window) or 32 bytes
//   (half: 8 per window): chunk c at c ^ ((r >> 2) & 3) or c ^ ((r >> 3) & 1)
//   X rows of 256 bytes (one per window) or 128 bytes (two): chunk c at
//   c ^ (x & 15) or c ^ ((x >> 1) & 7)
// so rows r .. r + 15 reading one chunk hit 16 distinct 16-byte bank slots.
template <int KS>
__device__ __forceinline__ int swz_w(int r) {
    return KS == 8 ? ((r >> 2) & 3) : ((r >> 3) & 1);
}
template <int KS>
__device__ __forceinline__ int swz_x(int x) {
    return KS == 8 ? (x & 15) : ((x >> 1) & 7);
}

template <int IMM>
__device__ __forceinline__ void wait_vm() {
    __builtin_amdgcn_s_waitcnt(IMM);
}

}  // namespace i4w
}  // namespace clove
