// Tensor-core and tensor-copy primitives for sm_100a as inline PTX: tensor
// maps and tiled bulk copies, tcgen05 matrix products with accumulators in
// tensor memory, their shared-memory descriptors, and the bounded wait of the
// kernels that hand tiles between warps.
//
// Tiles. A 16-bit operand tile of R rows and D columns lies in shared memory
// as D / 64 blocks of [R][64] elements (128 bytes a row), each written by
// tiled copies with the 128-byte swizzle, 1024-byte aligned. The same tile
// serves as an operand whose contracted index runs along its columns or along
// its rows.
#pragma once

#include <cuda.h>

#include "bulk.cuh"

namespace bloth {

// ------------------------------------------------------------- arithmetic
// 2^x; 2 ulp, results below the normal range are 0.
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}
// Two floats rounded to T in one register, the first in the lower half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  uint32_t r;
  if constexpr (std::is_same<T, __nv_bfloat16>::value)
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  else
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(r) : "f"(hi), "f"(lo));
  return r;
}

// Two floats y rounded to T, and what that took off them, times UP, rounded to T.
template <typename T, int UP = 1>
__device__ __forceinline__ void split2(float y0, float y1, uint32_t& hi, uint32_t& lo) {
  hi = pack2<T>(y0, y1);
  if constexpr (std::is_same<T, __nv_bfloat16>::value) {
    lo = pack2<T>((y0 - __uint_as_float(hi << 16)) * UP,
                  (y1 - __uint_as_float(hi & 0xffff0000u)) * UP);
  } else {
    __half2 h;
    memcpy(&h, &hi, 4);
    lo = pack2<T>((y0 - __half2float(h.x)) * UP, (y1 - __half2float(h.y)) * UP);
  }
}

// --------------------------------------------------------------- barriers
// Barriers are named by their 32-bit shared-memory address: the warps that
// issue copies and products run little else than waits and address
// arithmetic, one after the other, and every instruction there costs the
// tensor core its latency.
__device__ __forceinline__ void bar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void bar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void bar_expect(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
// One test of phase `parity`: at once (bar_test), or suspended for the default
// time at most (bar_try).
__device__ __forceinline__ bool bar_test(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.test_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}
__device__ __forceinline__ bool bar_try(uint32_t bar, uint32_t parity) {
  uint32_t done;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(done)
      : "r"(bar), "r"(parity)
      : "memory");
  return done != 0;
}

// What a CTA's waits share: the flag (in shared memory) by which a thread
// whose wait took longer than kWaitLimitNs makes all others give up, and the
// device's fault word, where that is recorded.
struct Waits {
  volatile int* stop;
  unsigned int* fault;
};
static __device__ __noinline__ bool bar_wait_slow(uint32_t bar, uint32_t parity, Waits w) {
  unsigned long long t0 = 0;
  for (int i = 1;; ++i) {
    if (bar_try(bar, parity)) return true;
    // the time is read now and then only: reading it takes longer than most waits
    if ((i & 63) != 0) continue;
    if (*w.stop) return false;
    const unsigned long long t = global_ns();
    if (t0 == 0) t0 = t;
    if (t - t0 > kWaitLimitNs) {
      *w.stop = 1;
      if (w.fault != nullptr) atomicOr(w.fault, kFaultCopyTimeout);
      return false;
    }
  }
}
// Waits for phase `parity` of `bar`; false once the CTA has given up.
__device__ __forceinline__ bool bar_wait(uint32_t bar, uint32_t parity, const Waits& w) {
  if (bar_try(bar, parity)) return true;
  return bar_wait_slow(bar, parity, w);
}
// After giving up: waits, as long again, for a copy or product in flight.
__device__ __forceinline__ void bar_drain(uint32_t bar, uint32_t parity, const Waits& w) {
  const unsigned long long t0 = global_ns();
  while (!bar_try(bar, parity)) {
    if (global_ns() - t0 > kWaitLimitNs) {
      if (w.fault != nullptr) atomicOr(w.fault, kFaultDrainTimeout);
      return;
    }
  }
}

// Stage and phase of a ring of barriers, advanced without a division.
template <int STAGES>
struct Ring {
  uint32_t at = 0, phase = 0;
  __device__ __forceinline__ void next() {
    if (++at == STAGES) {
      at = 0;
      phase ^= 1u;
    }
  }
};

// True in one lane of a converged warp. The issuing warps run their loops as
// a whole and let this lane issue, so that addresses and descriptors are
// computed in uniform registers, where the instructions take them from.
__device__ __forceinline__ bool elect() {
  uint32_t p;
  asm volatile(
      "{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(p));
  return p != 0;
}

// ----------------------------------------------------------- tiled copies
// One box of a 4-D tensor map (column, row, head, batch) into shared memory.
__device__ __forceinline__ void tma_load(uint32_t dst, const CUtensorMap* map, int col, int row,
                                         int head, int batch, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%2, %3, %4, %5}], [%6];" ::"r"(dst),
      "l"(map), "r"(col), "r"(row), "r"(head), "r"(batch), "r"(bar)
      : "memory");
}
// `bytes` consecutive bytes, both addresses and the size multiples of 16.
__device__ __forceinline__ void run_load(uint32_t dst, const void* src, uint32_t bytes,
                                         uint32_t bar) {
  asm volatile(
      "cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(
          dst),
      "l"(src), "r"(bytes), "r"(bar)
      : "memory");
}
// An operand tile of ROWS rows r0.. of a head: boxes of 64 rows x 64 columns.
template <int D, int ROWS>
__device__ __forceinline__ void load_tile(uint32_t dst, const CUtensorMap* map, int r0, int h,
                                          int b, uint32_t bar) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c)
#pragma unroll
    for (int r = 0; r < ROWS; r += 64)
      tma_load(dst + c * ROWS * 128 + r * 128, map, c * 64, r0 + r, h, b, bar);
}

// ------------------------------------------------------------ descriptors
// Shared-memory operand descriptor, addresses and offsets in 16-byte units.
// Upper word, the same for every tile here: groups of 8 rows are 1024 bytes
// apart (bits 32-45), version 1 (bit 46), 128-byte swizzle (2 in bits 61-63).
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// Lower word: the address, and the offset between blocks of 64 columns (bits
// 16-29), which counts where the contracted index runs along the rows.
//   along the columns ("K-major"): a step of 16 columns is 32 bytes inside a
//   64-column block;
//   along the rows ("MN-major"): a step of 16 rows is 2048 bytes.
__device__ __forceinline__ uint32_t desc_lo(uint32_t addr, uint32_t block) {
  return ((addr & 0x3ffff) >> 4) | ((block >> 4) << 16);
}
// Instruction descriptor: fp32 accumulator, A and B of type T, M x N, B's
// contracted index along its rows (b_mn) or columns.
template <typename T>
__host__ __device__ constexpr uint32_t mma_desc(int m, int n, bool b_mn) {
  const uint32_t ty = std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return (1u << 4) | (ty << 7) | (ty << 10) | ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(n >> 3) << 17) |
         ((uint32_t)(m >> 4) << 24);
}

// --------------------------------------------------------- matrix products
// Tensor memory [d] (+)= A x B for 16 contracted elements; issued by one
// thread. A in shared memory (mma_ss) or in tensor memory (mma_ts).
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 da, {%1, %5};\n\tmov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((int)add), "r"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc,
                                       bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 db, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"((int)add), "r"(kDescHi)
      : "memory");
}

// d = A B^T, contracted over the D columns: A an operand tile of 128 rows, B of
// 64, at shared-memory addresses.
template <typename T, int D>
__device__ __forceinline__ void product_rows(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t id = mma_desc<T>(128, 64, false);
  const uint32_t la = desc_lo(a, 0), lb = desc_lo(b, 0);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    mma_ss(d, la + (((kk / 4) * (128 * 128) + (kk % 4) * 32) >> 4),
           lb + (((kk / 4) * (64 * 128) + (kk % 4) * 32) >> 4), id, kk > 0);
}
// The same with A in tensor memory (copy_operand).
template <typename T, int D>
__device__ __forceinline__ void product_rows_ts(uint32_t d, uint32_t a, uint32_t b) {
  constexpr uint32_t id = mma_desc<T>(128, 64, false);
  const uint32_t lb = desc_lo(b, 0);
#pragma unroll
  for (int kk = 0; kk < D / 16; ++kk)
    mma_ts(d, a + kk * 8, lb + (((kk / 4) * (64 * 128) + (kk % 4) * 32) >> 4), id, kk > 0);
}
// d (+)= W B, contracted over the 64 rows of operand tile B: W 128 x 64 of
// 16-bit elements in 32 columns of tensor memory.
template <typename T, int D>
__device__ __forceinline__ void product_cols(uint32_t d, uint32_t w, uint32_t b, bool add) {
  constexpr uint32_t id = mma_desc<T>(128, D, true);
  const uint32_t lb = desc_lo(b, 64 * 128);
#pragma unroll
  for (int kk = 0; kk < 4; ++kk) mma_ts(d, w + kk * 8, lb + kk * (2048 >> 4), id, add || kk > 0);
}
// `bar` completes a phase when every product issued so far has completed.
__device__ __forceinline__ void mma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(
                   bar)
               : "memory");
}

// ----------------------------------------------------------- tensor memory
// Whole-warp allocation of `cols` columns; the address goes to *dst.
__device__ __forceinline__ void tmem_alloc(uint32_t* dst, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                   smem_addr(dst)),
               "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols)
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld() {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_wait_st() {
  asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}

// 32 columns of the warp's 32 lanes: lane l gets row l. The address carries
// the warp's first lane in its upper half.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]),
        "=r"(r[21]), "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]),
        "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]),
        "=r"(r[7]), "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]),
        "=r"(r[14]), "=r"(r[15])
      : "r"(addr)
      : "memory");
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, "
      "%17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(
          addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
      "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]),
      "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]),
      "r"(r[30]), "r"(r[31])
      : "memory");
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
      "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}

// 64 columns of the thread's row, and 64 values rounded to T in 32 columns
// (not waited for).
__device__ __forceinline__ void load64(uint32_t at, float (&x)[64]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t r[32];
    tmem_ld32(at + c * 32, r);
#pragma unroll
    for (int i = 0; i < 32; ++i) x[c * 32 + i] = __uint_as_float(r[i]);
  }
  tmem_wait_ld();
}
template <typename T>
__device__ __forceinline__ void store64(uint32_t at, const float (&x)[64]) {
  uint32_t r[32];
#pragma unroll
  for (int i = 0; i < 32; ++i) r[i] = pack2<T>(x[2 * i], x[2 * i + 1]);
  tmem_st32(at, r);
}
// What that rounding took off, rounded in its turn.
template <typename T>
__device__ __forceinline__ void store64_rest(uint32_t at, const float (&x)[64]) {
#pragma unroll
  for (int c = 0; c < 2; ++c) {
    uint32_t r[16], hi;
#pragma unroll
    for (int i = 0; i < 16; ++i) split2<T>(x[32 * c + 2 * i], x[32 * c + 2 * i + 1], hi, r[i]);
    tmem_st16(at + 16 * c, r);
  }
}

// Row `r` of an operand tile of 128 rows, from shared memory to the thread's row
// of D / 2 tensor-memory columns, two elements each: a first operand there
// leaves the products half of their shared-memory reads.
template <int D>
__device__ __forceinline__ void copy_operand(const unsigned char* tile, int r, uint32_t at) {
#pragma unroll
  for (int c = 0; c < D / 64; ++c) {
    uint32_t w[32];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      const uint4 v = *reinterpret_cast<const uint4*>(tile + c * (128 * 128) + r * 128 +
                                                      ((i ^ (r & 7)) * 16));
      w[4 * i] = v.x;
      w[4 * i + 1] = v.y;
      w[4 * i + 2] = v.z;
      w[4 * i + 3] = v.w;
    }
    tmem_st32(at + c * 32, w);
  }
  tmem_wait_st();
}

// Rows [r0, r1) of an operand tile of 64 in shared memory become zeros, before
// later products read them (128 threads).
template <int D>
__device__ __forceinline__ void zero_rows(unsigned char* tile, int r0, int r1) {
  for (int c = threadIdx.x & 127; c < (r1 - r0) * (D / 8); c += 128) {
    const int r = r0 + c / (D / 8), b = c % (D / 8);
    *reinterpret_cast<uint4*>(tile + (b / 8) * (64 * 128) + r * 128 + (b % 8) * 16) =
        make_uint4(0, 0, 0, 0);
  }
  fence_proxy_async_smem();
}
// All but rows [r0, r1), which may reach past the tile, become zeros. Few blocks need
// it, so in the backward it is a call, which leaves the loops their registers (64 x
// 128 rows of 32/8 heads of 128, forward and backward: 344 us, in line 354; the
// forward's one loop is 1% slower with the call).
template <int D>
__device__ __noinline__ void keep_rows(unsigned char* tile, int r0, int r1) {
  if (r0 > 0) zero_rows<D>(tile, 0, r0);
  if (r1 < 64) zero_rows<D>(tile, r1, 64);
}

// Host: tensor map of a head tensor [B, S, H, D] of 16-bit elements, boxes of
// `rows` rows x 64 columns of one head, 128-byte swizzle, zeros outside.
int head_map(CUtensorMap* map, const void* p, int64_t sb, int64_t ss, int64_t sh, int B, int64_t S,
             int H, int D, int rows, int dtype);

}  // namespace bloth
