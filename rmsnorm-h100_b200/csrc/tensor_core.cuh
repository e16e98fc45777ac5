// tensor_core.cuh -- tcgen05 products of e4m3 operands in shared memory, their accumulators in
// tensor memory, and the tiled TMA copies that bring the operands (no multicast).
#pragma once

#include <cuda.h>

#include "device_common.cuh"

namespace rmsb200 {

// An operand tile in shared memory: rows of 128 bytes (128 values along k), eight rows to a
// 1024-byte atom with the 128-byte swizzle, atoms one after the other. TMA writes it, the
// product reads it.
constexpr int kTileK = 128;

// The matrix descriptor of a tile at a 1024-byte boundary: addresses in 16-byte units, 1024
// bytes from one group of eight rows to the next, 128-byte swizzle. 32 values further along k
// are 32 bytes further.
__device__ __forceinline__ uint64_t operand_desc(uint32_t addr) {
  return static_cast<uint64_t>((addr & 0x3ffffu) >> 4) | (uint64_t{1} << 16) | (uint64_t{1024 >> 4} << 32) |
         (uint64_t{1} << 46) | (uint64_t{2} << 61);
}

// The instruction descriptor of an M x N product: e4m3 operands, both with k contiguous, fp32
// accumulators.
__host__ __device__ constexpr uint32_t product_desc(int m, int n) {
  return (1u << 4) | (static_cast<uint32_t>(n >> 3) << 17) | (static_cast<uint32_t>(m >> 4) << 24);
}

// One lane of a whole warp, always the same. Unlike a test of the lane's number it tells the
// compiler that a single thread follows, whose operands can lie in uniform registers.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(yes));
  return yes != 0;
}

// One thread of the CTA (of the pair): D (+)= A B^T over 32 values of k.
template <bool kPair>
__device__ __forceinline__ void mma_e4m3(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool add) {
  if constexpr (kPair)
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::2.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
  else
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f8f6f4 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
        "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add))
        : "memory");
}

// The same for block-scaled operands: an exponent (8 bits, as a power of two in fp32 has it) for
// every 32 values of k of every row, in tensor memory; the tensor cores apply them.
__host__ __device__ constexpr uint32_t scaled_product_desc(int m, int n) {
  return (static_cast<uint32_t>(n >> 3) << 17) | (1u << 23) | (static_cast<uint32_t>(m >> 4) << 24);
}

// By a pair. Every 32 rows of a CTA's a take a column at scale_a (lane: row % 32), of all of b at
// scale_b, in both CTAs; byte 0 of a cell is read.
__device__ __forceinline__ void mma_e4m3_scaled(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, uint32_t scale_a,
                                                uint32_t scale_b, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\tsetp.ne.u32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::2.kind::mxf8f6f4.block_scale [%0], %1, %2, %3, [%5], [%6], p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "r"(scale_a), "r"(scale_b)
      : "memory");
}

// 32 rows of 16 bytes, one behind the other in shared memory, into four columns of 32 lanes and
// their copies in the other 96; in both CTAs of a pair, each from its own shared memory.
__device__ __forceinline__ void scales_to_tmem(uint32_t taddr, uint32_t smem_addr) {
  const uint64_t desc = static_cast<uint64_t>((smem_addr & 0x3ffffu) >> 4) | (uint64_t{1} << 16) | (uint64_t{128 >> 4} << 32) |
                        (uint64_t{1} << 46);
  asm volatile("tcgen05.cp.cta_group::2.32x128b.warpx4 [%0], %1;" ::"r"(taddr), "l"(desc) : "memory");
}

// `bar` gets one arrival when this thread's products so far are complete; of a pair, both CTAs'.
template <bool kPair>
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  if constexpr (kPair)
    asm volatile(
        "tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(
            smem_u32(bar)),
        "h"(static_cast<uint16_t>(3))
        : "memory");
  else
    asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
                 : "memory");
}

// A box of a [rows][k] byte matrix into shared memory; outside the matrix zeros. x: byte of a
// row (a multiple of 16), y: row. Of a pair, the bytes count on the first CTA's barrier: the
// bit of a shared-memory address that tells the two apart is cleared.
template <bool kPair>
__device__ __forceinline__ void tile_load(void* dst, const CUtensorMap* map, int x, int y, uint64_t* bar) {
  if constexpr (kPair)
    asm volatile(
        "cp.async.bulk.tensor.2d.cta_group::2.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, "
        "%4}], [%2];" ::"r"(smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar) & 0xfeffffffu), "r"(x), "r"(y)
        : "memory");
  else
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4}], [%2];" ::"r"(
            smem_u32(dst)),
        "l"(map), "r"(smem_u32(bar)), "r"(x), "r"(y)
        : "memory");
}

__device__ __forceinline__ void prefetch_map(const CUtensorMap* map) {
  asm volatile("prefetch.tensormap [%0];" ::"l"(map) : "memory");
}

// One arrival at the barrier of CTA `rank` of the cluster.
__device__ __forceinline__ void mbar_arrive_peer(uint64_t* bar, uint32_t rank) {
  asm volatile("mbarrier.arrive.shared::cluster.b64 _, [%0];" ::"r"(map_peer(smem_u32(bar), rank))
               : "memory");
}

__device__ __forceinline__ float4 ld_peer4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared::cluster.v4.f32 {%0, %1, %2, %3}, [%4];"
               : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w)
               : "r"(addr)
               : "memory");
  return v;
}

// Tensor memory of a pair: one warp of each of its CTAs.
__device__ __forceinline__ void tmem_alloc_pair(uint32_t* dst, uint32_t ncols) {
  asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(dst)), "r"(ncols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc_pair(uint32_t taddr, uint32_t ncols) {
  asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(ncols) : "memory");
}

// Consecutive columns of this lane: asked for, and (every load so far) landed. The registers
// pass through the wait, so that nothing that uses them moves before it.
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float2 (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
               : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x),
                 "=f"(v[3].y), "=f"(v[4].x), "=f"(v[4].y), "=f"(v[5].x), "=f"(v[5].y), "=f"(v[6].x), "=f"(v[6].y),
                 "=f"(v[7].x), "=f"(v[7].y)
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_landed(float2 (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0].x), "+f"(v[0].y), "+f"(v[1].x), "+f"(v[1].y), "+f"(v[2].x), "+f"(v[2].y), "+f"(v[3].x),
                 "+f"(v[3].y), "+f"(v[4].x), "+f"(v[4].y), "+f"(v[5].x), "+f"(v[5].y), "+f"(v[6].x), "+f"(v[6].y),
                 "+f"(v[7].x), "+f"(v[7].y)::"memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t taddr, float2 (&v)[16]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x32.b32 "
               "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, "
               "%21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
               : "=f"(v[0].x), "=f"(v[0].y), "=f"(v[1].x), "=f"(v[1].y), "=f"(v[2].x), "=f"(v[2].y), "=f"(v[3].x),
                 "=f"(v[3].y), "=f"(v[4].x), "=f"(v[4].y), "=f"(v[5].x), "=f"(v[5].y), "=f"(v[6].x), "=f"(v[6].y),
                 "=f"(v[7].x), "=f"(v[7].y), "=f"(v[8].x), "=f"(v[8].y), "=f"(v[9].x), "=f"(v[9].y), "=f"(v[10].x),
                 "=f"(v[10].y), "=f"(v[11].x), "=f"(v[11].y), "=f"(v[12].x), "=f"(v[12].y), "=f"(v[13].x),
                 "=f"(v[13].y), "=f"(v[14].x), "=f"(v[14].y), "=f"(v[15].x), "=f"(v[15].y)
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_landed(float2 (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0].x), "+f"(v[0].y), "+f"(v[1].x), "+f"(v[1].y), "+f"(v[2].x), "+f"(v[2].y), "+f"(v[3].x),
                 "+f"(v[3].y), "+f"(v[4].x), "+f"(v[4].y), "+f"(v[5].x), "+f"(v[5].y), "+f"(v[6].x), "+f"(v[6].y),
                 "+f"(v[7].x), "+f"(v[7].y), "+f"(v[8].x), "+f"(v[8].y), "+f"(v[9].x), "+f"(v[9].y), "+f"(v[10].x),
                 "+f"(v[10].y), "+f"(v[11].x), "+f"(v[11].y), "+f"(v[12].x), "+f"(v[12].y), "+f"(v[13].x),
                 "+f"(v[13].y), "+f"(v[14].x), "+f"(v[14].y), "+f"(v[15].x), "+f"(v[15].y)::"memory");
}

template <int kRegs>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs));
}
template <int kRegs>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs));
}

}  // namespace rmsb200
