// What the tensor-core kernels of the packed attention share: tensor maps of [tokens, heads, D] tensors, operand descriptors,
// tensor-memory stores, packed arithmetic.
#pragma once

#include <cuda.h>

#include "gw_packed.cuh"
#include "gw_tc.cuh"

namespace gw {

constexpr int kTile = 128;                     // rows of an operand tile = TMEM lanes
constexpr int kBoxBytes = kTile * 64 * 2;      // 128 rows x 64 16-bit columns: one TMA box, rows of 128 bytes, 128-byte swizzle

__device__ __forceinline__ void tma_load_3d(void* dst, const CUtensorMap* map, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];" ::"r"(
          smem_u32(dst)),
      "l"(map), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}
// all DP columns of ROWS rows of one head, as DP / 64 boxes one behind the other
template <int DP, int ROWS = kTile>
__device__ __forceinline__ void load_rows(unsigned char* dst, const CUtensorMap* map, int head, int row, uint64_t* bar) {
#pragma unroll
  for (int b = 0; b < DP / 64; ++b) tma_load_3d(dst + b * ROWS * 128, map, 64 * b, head, row, bar);
}

// Operand tile read along its rows (the contraction runs over the tokens): 64 columns are one swizzle atom wide, further
// columns start one box behind; groups of eight rows are 1024 bytes apart.
__device__ __forceinline__ uint64_t make_smem_desc_mn(uint32_t saddr) {
  uint64_t d = 0;
  d |= static_cast<uint64_t>((saddr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(kBoxBytes >> 4) << 16;  // leading byte offset: the next 64 columns
  d |= static_cast<uint64_t>(1024 >> 4) << 32;       // stride byte offset: the next eight rows
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}
constexpr uint32_t kBMajorMN = 1u << 16;  // instruction descriptor: B is read along its rows

// D = A . B^T over DP columns, both operands row tiles in shared memory (K-major)
template <int DP>
__device__ __forceinline__ void mma_rows(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc) {
#pragma unroll
  for (int s = 0; s < DP / 16; ++s) {
    const uint64_t at = (s / 4) * (kBoxBytes >> 4) + (s % 4) * 2;
    tc_mma_f16(d, a + at, b + at, idesc, s > 0 ? 1u : 0u);
  }
}
__device__ __forceinline__ void tc_mma_f16_ts(uint32_t d_tmem, uint32_t a_tmem, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "l"(bdesc), "r"(idesc), "r"(accumulate)
      : "memory");
}

__device__ __forceinline__ void tmem_load32(uint32_t taddr, float* v) {
  uint32_t* r = reinterpret_cast<uint32_t*>(v);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]), "=r"(r[9]),
        "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]),
        "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(taddr)
      : "memory");
}
__device__ __forceinline__ void tmem_store32(uint32_t taddr, const uint32_t* r) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]),
      "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_store8(uint32_t taddr, const uint32_t (&r)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8};" ::"r"(taddr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]),
               "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7])
               : "memory");
}
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// two fp32 values in one 64-bit register: one instruction for both
__device__ __forceinline__ uint64_t pack_f2(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void unpack_f2(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_f2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t add_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ uint64_t mul_f2(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float exp2_fast(float x) {  // 2 ulp; results below 2^-126 are zero
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
template <typename T> __device__ __forceinline__ uint32_t pack_half2(float lo, float hi);
template <> __device__ __forceinline__ uint32_t pack_half2<__nv_bfloat16>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}
template <> __device__ __forceinline__ uint32_t pack_half2<__half>(float lo, float hi) {
  uint32_t d;
  asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(hi), "f"(lo));
  return d;
}

// Waits of a whole warp.  Every lane asks the barrier, and one lane's wait may run out where another's last try succeeds; the warp
// decides as one, or it would split in front of the next warp-wide instruction (shuffle, elect, tcgen05), which then waits for the
// missing lanes without end.  A wait also ends, as if it had run out, when another warp of the block has given up (`abort`, nullable): looked
// at between tries only, where the time is not missed (with a look at each tile the wide-head forward took 4 % longer).  Against lanes
// that decide alone: 33 312 tokens, 16 heads of 64 5.43 ms both, 8328 tokens' training step 1563 -> 1594 us, of 128 columns 2187 -> 2208.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, const volatile int* abort, unsigned long long limit_ns = kWaitLimitNs) {
  if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
  const unsigned long long t0 = global_timer_ns();
  for (;;) {
#pragma unroll 1
    for (int i = 0; i < 256; ++i)
      if (__all_sync(0xffffffffu, mbar_try_wait(bar, parity))) return true;
    if (__any_sync(0xffffffffu, global_timer_ns() - t0 > limit_ns || (abort != nullptr && *abort != 0))) return false;
  }
}
__device__ __forceinline__ bool warp_sees(const volatile int& flag) { return __any_sync(0xffffffffu, flag != 0); }

// One lane of a whole warp, the same one every time.  The compiler knows of this form that a single lane follows, and feeds the
// products' descriptors from uniform registers; behind `lane == 0` it moves each of them over first, which cost the wide-head
// forward 6 % and the narrow one 2 to 6 %.
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(is));
  return is != 0;
}
// a value read from memory that is the same in all lanes, made known as such to the compiler
__device__ __forceinline__ int uniform(int v) { return __shfl_sync(0xffffffffu, v, 0); }

// 32 16-bit values of one row, as many of them as lie below `left`: whole 32-byte sectors where the row allows it
__device__ __forceinline__ void store_row32(void* dst, const uint32_t (&e)[16], int left, bool sectors) {
  if (sectors) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      if (16 * i < left)
        asm volatile("st.global.v8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"l"(static_cast<char*>(dst) + 32 * i), "r"(e[8 * i]),
                     "r"(e[8 * i + 1]), "r"(e[8 * i + 2]), "r"(e[8 * i + 3]), "r"(e[8 * i + 4]), "r"(e[8 * i + 5]), "r"(e[8 * i + 6]),
                     "r"(e[8 * i + 7])
                     : "memory");
  } else {
#pragma unroll
    for (int i = 0; i < 4; ++i)
      if (8 * i < left) reinterpret_cast<uint4*>(dst)[i] = make_uint4(e[4 * i], e[4 * i + 1], e[4 * i + 2], e[4 * i + 3]);
  }
}
__device__ __forceinline__ bool row_sectors(const void* base, int D) { return D % 16 == 0 && (reinterpret_cast<uintptr_t>(base) & 31) == 0; }

// Rows from `from` on of an operand tile become zero (whole warp): the rows behind a sequence's end belong to its
// neighbour or to nobody, and zero times whatever stands there need not be zero.
template <int DP, int ROWS = kTile>
__device__ __forceinline__ void zero_rows_from(unsigned char* tile, int from) {
  const int lane = threadIdx.x & 31;
  for (int b = 0; b < DP / 64; ++b)
    for (int i = from * 8 + lane; i < ROWS * 8; i += 32) *reinterpret_cast<uint4*>(tile + b * ROWS * 128 + i * 16) = make_uint4(0, 0, 0, 0);
  fence_proxy_async_smem();
  __syncwarp();
}

// [tokens, heads, D] tensor of 16-bit elements with any 16-byte strides; a box is 64 columns of `rows` tokens of one head, what lies
// outside the tensor reads as zero (a side without tokens is never loaded)
int make_token_map(CUtensorMap* map, const void* base, int dtype, int64_t tokens, int heads, int D, int64_t token_stride, int64_t head_stride,
                   int rows);

}  // namespace gw
