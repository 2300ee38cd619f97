// 5th-generation tensor-core building blocks of the many-query attention kernels: shared-memory
// and instruction descriptors, tcgen05 products and tensor-memory moves, bounded barrier waits.
//
// Both kernels hold 128 query rows per tile.  A row is one tensor-memory lane, so a softmax thread
// owns a whole row and the running maximum and sum need no exchange between threads.
//   S = Q K^T   Q, K: [rows][128] 16-bit in shared memory, two halves of 64 channels, each row 128
//               bytes with the 128-byte XOR swizzle; float32 scores in tensor memory
//   O += P V    P: 16-bit in tensor memory over the scores it was made from; V: [keys][128] in the
//               layout of K, read with the channels as the leading axis (no transposed copy)
#pragma once

#include <cuda.h>
#include <cudaTypedefs.h>

#include <cmath>
#include <mutex>

#include "tp_common.cuh"

namespace tp {

// ----------------------------------------------------------------------------- host side
inline int device_sms() {
  static int sms[64] = {};
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess || dev < 0 || dev >= 64) {
    cudaGetLastError();
    return 148;
  }
  if (!sms[dev]) {
    int n = 0;
    if (cudaDeviceGetAttribute(&n, cudaDevAttrMultiProcessorCount, dev) != cudaSuccess || n <= 0) {
      cudaGetLastError();
      return 148;
    }
    sms[dev] = n;
  }
  return sms[dev];
}

// Allow a kernel its dynamic shared memory on the current device.  `wg_regs`: the registers per
// thread that its warpgroups ask for, summed over the warpgroups; a warpgroup that asked for more than the block
// was launched with would wait for good, so a build whose register count differs is refused here.
inline int allow_kernel(const void* fn, int smem, int threads, int wg_regs, const char* what) {
  cudaFuncAttributes attr;
  cudaError_t e = cudaFuncGetAttributes(&attr, fn);
  if (e == cudaSuccess) e = cudaFuncSetAttribute(fn, cudaFuncAttributeMaxDynamicSharedMemorySize, smem);
  if (e != cudaSuccess) {
    cudaGetLastError();
    return fail(TP_ERR_CUDA, std::string(what) + ": " + cudaGetErrorString(e));
  }
  if (attr.numRegs * (threads / 128) < wg_regs)
    return fail(TP_ERR_CUDA, std::string(what) + ": built with " + std::to_string(attr.numRegs) + " registers per thread");
  return TP_OK;
}

// ----------------------------------------------------------------------------- descriptors
constexpr int kTile = 128;               // query rows of a tile
constexpr int kHalfTile = kTile * 128;   // bytes of 128 rows x 64 channels
constexpr int kTileBytes = 2 * kHalfTile;

// Byte offset of 16-byte chunk c (0..15) of row r in a tile of `rows` rows.
__device__ __forceinline__ uint32_t tile_chunk(int r, int c, int rows) {
  return uint32_t((c >> 3) * rows * 128 + r * 128 + (((c & 7) ^ (r & 7)) << 4));
}

// Shared-memory operand descriptor, 128-byte swizzle.  Low word: bits 0-13 address / 16, 16-29
// leading-axis offset / 16.  High word, the same for every operand here: bits 0-13 stride between
// groups of 8 rows (1024) / 16, 14-15 version 1, 29-31 swizzle 2.  Moving along a tile adds to the
// low word only.
constexpr uint32_t kDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
// Rows of 64 channels, channels contracted.
__device__ __forceinline__ uint32_t rows_lo(uint32_t addr) { return (addr >> 4) | (1u << 16); }
// Rows contracted, channels the output axis: halves of 64 channels `half` bytes apart.
__device__ __forceinline__ uint32_t cols_lo(uint32_t addr, uint32_t half) { return (addr >> 4) | ((half >> 4) << 16); }

// kind::f16 instruction descriptor, M = 128: float32 accumulator, both operands bf16 or both f16.
__host__ __device__ constexpr uint32_t mma_idesc(bool bf16, int n, bool b_cols) {
  return (1u << 4) | (uint32_t(bf16) << 7) | (uint32_t(bf16) << 10) | (uint32_t(b_cols) << 16) |
         (uint32_t(n >> 3) << 17) | (uint32_t(kTile >> 4) << 24);
}

// ----------------------------------------------------------------------------- tcgen05
__device__ __forceinline__ void tmem_alloc(uint32_t* slot, int cols) {  // one warp
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(slot)), "r"(cols)
               : "memory");
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
}
__device__ __forceinline__ void tmem_free(uint32_t addr, int cols) {  // the same warp
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(addr), "r"(cols));
}
// One thread of a warp, always the same one.  Issuing under this predicate inside code that the whole
// warp runs keeps descriptors and addresses in uniform registers, which the instruction needs; in
// code of a single lane each product took about 100 cycles to issue.
__device__ __forceinline__ bool elect_one() {
  uint32_t yes;
  asm volatile("{\n .reg .pred p;\n elect.sync _|p, 0xffffffff;\n selp.u32 %0, 1, 0, p;\n}\n" : "=r"(yes));
  return yes != 0;
}
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 da, db;\n setp.ne.u32 p, %4, 0;\n mov.b64 da, {%1, %5};\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %3, p;\n}\n" ::"r"(d),
      "r"(a_lo), "r"(b_lo), "r"(idesc), "r"(uint32_t(add)), "n"(kDescHi)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b_lo, uint32_t idesc, bool add) {
  asm volatile(
      "{\n .reg .pred p;\n .reg .b64 db;\n setp.ne.u32 p, %4, 0;\n mov.b64 db, {%2, %5};\n"
      " tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], db, %3, p;\n}\n" ::"r"(d),
      "r"(a), "r"(b_lo), "r"(idesc), "r"(uint32_t(add)), "n"(kDescHi)
      : "memory");
}
// Arrive on `bar` once every product issued by this thread so far has completed.
__device__ __forceinline__ void mma_commit(uint64_t* bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(smem_u32(bar))
               : "memory");
}
__device__ __forceinline__ void tmem_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tmem_wait_st() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// 32 columns of this warp's 32 lanes: thread i holds lane i.
__device__ __forceinline__ void tmem_ld32(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,%18,%19,"
      "%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%32];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15]), "=r"(u[16]),
        "=r"(u[17]), "=r"(u[18]), "=r"(u[19]), "=r"(u[20]), "=r"(u[21]), "=r"(u[22]), "=r"(u[23]), "=r"(u[24]),
        "=r"(u[25]), "=r"(u[26]), "=r"(u[27]), "=r"(u[28]), "=r"(u[29]), "=r"(u[30]), "=r"(u[31])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_ld16(uint32_t addr, float* r) {
  uint32_t* u = reinterpret_cast<uint32_t*>(r);
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
      : "=r"(u[0]), "=r"(u[1]), "=r"(u[2]), "=r"(u[3]), "=r"(u[4]), "=r"(u[5]), "=r"(u[6]), "=r"(u[7]), "=r"(u[8]),
        "=r"(u[9]), "=r"(u[10]), "=r"(u[11]), "=r"(u[12]), "=r"(u[13]), "=r"(u[14]), "=r"(u[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_st16(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%16], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(addr)
      : "memory");
}
// The registers of the loads above are valid after the wait; naming them as operands keeps the compiler
// from moving their uses before it.
__device__ __forceinline__ void after_wait16(float* r) {
  asm volatile(""
      : "+f"(r[0]), "+f"(r[1]), "+f"(r[2]), "+f"(r[3]), "+f"(r[4]), "+f"(r[5]), "+f"(r[6]), "+f"(r[7]),
        "+f"(r[8]), "+f"(r[9]), "+f"(r[10]), "+f"(r[11]), "+f"(r[12]), "+f"(r[13]), "+f"(r[14]), "+f"(r[15]));
}
template <int kCols>
__device__ __forceinline__ void tmem_wait_ld(float* r) {
  asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory");
#pragma unroll
  for (int c = 0; c < kCols; c += 16) after_wait16(r + c);
}
__device__ __forceinline__ void tmem_st32(uint32_t addr, const uint32_t* u) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%32], {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,%17,"
      "%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31};" ::"r"(u[0]),
      "r"(u[1]), "r"(u[2]), "r"(u[3]), "r"(u[4]), "r"(u[5]), "r"(u[6]), "r"(u[7]), "r"(u[8]), "r"(u[9]), "r"(u[10]),
      "r"(u[11]), "r"(u[12]), "r"(u[13]), "r"(u[14]), "r"(u[15]), "r"(u[16]), "r"(u[17]), "r"(u[18]), "r"(u[19]),
      "r"(u[20]), "r"(u[21]), "r"(u[22]), "r"(u[23]), "r"(u[24]), "r"(u[25]), "r"(u[26]), "r"(u[27]), "r"(u[28]),
      "r"(u[29]), "r"(u[30]), "r"(u[31]), "r"(addr)
      : "memory");
}

// Tiled 3-D tensor copy global -> shared memory at element coordinates (x, y, z).
__device__ __forceinline__ void tma_tile_3d(uint32_t dst, const void* tmap, int x, int y, int z, uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4}], [%5];\n" ::
          "r"(dst),
      "l"(reinterpret_cast<uint64_t>(tmap)), "r"(x), "r"(y), "r"(z), "r"(smem_u32(bar))
      : "memory");
}

// ----------------------------------------------------------------------------- bounded waits
constexpr long long kWaitCycles = 2000000000ll;  // about a second

// Wait for phase `parity` of `bar`.  False once the CTA has given up (`stop` set by any thread's
// wait that ran out): the caller leaves its loop.
__device__ __forceinline__ bool wait_bar(uint64_t* bar, uint32_t parity, volatile int* stop) {
  if (mbar_try_wait(bar, parity)) return true;
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity)) {
    if (*stop) return false;
    if (clock64() - t0 > kWaitCycles) {
      *stop = 1;
      return false;
    }
  }
  return true;
}
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* stop) {
  return __all_sync(0xffffffffu, wait_bar(bar, parity, stop));
}
// The same without giving up early, to drain copies and products in flight.
__device__ __forceinline__ void drain_bar(uint64_t* bar, uint32_t parity) {
  const long long t0 = clock64();
  while (!mbar_try_wait(bar, parity) && clock64() - t0 < kWaitCycles) {
  }
}

__device__ __forceinline__ uint32_t pack_bf2(float a, float b) {
  uint32_t d;
  asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
  return d;
}
template <bool kBf16>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
  return kBf16 ? pack_bf2(a, b) : pack_h2(a, b);
}

// Registers per thread of this warpgroup from here on (every warp of it executes this).
template <int kRegs>
__device__ __forceinline__ void more_registers() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegs)); }
template <int kRegs>
__device__ __forceinline__ void fewer_registers() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegs)); }

// ----------------------------------------------------------------------------- softmax of one row
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {  // two float32 each
  uint64_t d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
  return d;
}
__device__ __forceinline__ void split_pair(uint64_t p, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(p));
}

__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
  uint64_t d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
  float d;
  asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
  return d;
}

// The running softmax of a row: weights are 2^(s * scale_log2 - ref) with a reference 7 below the maximum that set
// it.  It moves only when a maximum exceeds that one by more than 8: weights up to 2^15 fit float16, sums and
// accumulators are float32, and the output accumulator, which lives in tensor memory, is rescaled a few times per row
// instead of once per tile.  The 7 are for small weights: float16 ends at 2^-24, so weights vanish from the product
// (not from the sum) under 2^-32 of the largest, where a reference at the maximum lost those under 2^-25: the whole
// of a flat background of keys behind one strong one.
constexpr float kRefBelow = 7.0f, kRefSlack = kRefBelow + 8.0f;
struct SoftmaxRow {
  float ref = -INFINITY;  // nothing seen yet
  float sum = 0.0f;
};

// Which columns of a tile a row sees: the first `n`, or those whose bit is set.
struct FirstN {
  int n;
  template <int kCols> __device__ __forceinline__ bool all() const { return n >= kCols; }
  __device__ __forceinline__ bool operator()(int c) const { return c < n; }
};
struct Bits64 {
  uint64_t bits;
  template <int kCols> __device__ __forceinline__ bool all() const { return ~bits == 0; }
  __device__ __forceinline__ bool operator()(int c) const { return bits >> c & 1; }
};

// One tile of kCols scores of this thread's row, in tensor memory at `s_addr` (the warp's lanes);
// columns that the row does not see are masked, whatever they hold.  Writes the 16-bit weights over the
// scores.  `o_addr`: the row's 128 accumulator columns, rescaled when the reference moves;
// `before_rescale()` waits until the products issued so far have completed (false: given up) and
// is not called for the first tile, when the accumulator holds nothing.
//
// The weights are made with the reference as it is while the maximum is found on another pipe, and
// made again in the few tiles that move the reference: the special-function unit, which needs 8 cycles
// for a warp's exponential (1,024 for 128 columns), does not wait for the maximum.
//
// Weights are rounded to the 16-bit input type (float16 for trees) for the product, the sum is of the unrounded ones:
// 0.00021 to 0.00027 of the norm from the 64-bit result where rounding the output alone gives 0.00021 (bfloat16 0.0020
// and 0.0016).  A second part of each would halve what the weights add and double the second product.
//
// kTwice: the scores of column c are the sum of columns c and c + kCols (a key in two parts) times `factors[c]` in
// shared memory, and its weight is written to both.  Where the factor is 0 the score is exact(c) instead.
struct NoExact {
  __device__ __forceinline__ float operator()(int) const { return 0.0f; }
};
template <int kCols, bool kBf16, bool kTwice = false, class Sees, class Wait, class Exact = NoExact>
__device__ __forceinline__ bool softmax_tile(SoftmaxRow& row, uint32_t s_addr, uint32_t o_addr, Sees sees,
                                             float scale_log2, bool first, Wait before_rescale,
                                             const float* factors = nullptr, Exact exact = Exact()) {
  float s[kCols];
#pragma unroll
  for (int c = 0; c < kCols; c += 32) tmem_ld32(s_addr + c, s + c);
  if constexpr (kTwice) {
    float rest[kCols];
#pragma unroll
    for (int c = 0; c < kCols; c += 32) tmem_ld32(s_addr + kCols + c, rest + c);
    tmem_wait_ld<kCols>(s);
    tmem_wait_ld<kCols>(rest);
    float least = 1.0f;
#pragma unroll
    for (int c = 0; c < kCols; c += 4) {
      const float4 f = *reinterpret_cast<const float4*>(factors + c);
      s[c] = (s[c] + rest[c]) * f.x, s[c + 1] = (s[c + 1] + rest[c + 1]) * f.y;
      s[c + 2] = (s[c + 2] + rest[c + 2]) * f.z, s[c + 3] = (s[c + 3] + rest[c + 3]) * f.w;
      least = fminf(fminf(fminf(least, f.x), fminf(f.y, f.z)), f.w);
    }
    if (least == 0.0f) {  // the same for all threads
#pragma unroll 1
      for (int i = 0; i < kCols; ++i) {
        if (factors[i] != 0.0f) continue;
        const float x = exact(i);
#pragma unroll
        for (int c = 0; c < kCols; ++c) s[c] = c == i ? x : s[c];
      }
    }
  } else {
    tmem_wait_ld<kCols>(s);
  }
  if (!__all_sync(0xffffffffu, sees.template all<kCols>())) {
#pragma unroll
    for (int c = 0; c < kCols; ++c) s[c] = sees(c) ? s[c] : -INFINITY;
  }
  if (first) {  // no reference to try: one pass of maxima costs less than a pass of weights
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < kCols; c += 2) top[c >> 1 & 3] = max3(top[c >> 1 & 3], s[c], s[c + 1]);
    row.ref = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * scale_log2 - kRefBelow;
  }
  const uint64_t scale2 = pair_of(scale_log2, scale_log2);
  uint64_t add[2];
  for (;;) {
    const float base = row.ref == -INFINITY ? 0.0f : -row.ref;
    const uint64_t base2 = pair_of(base, base);
    add[0] = add[1] = 0;
    float top[4] = {-INFINITY, -INFINITY, -INFINITY, -INFINITY};
#pragma unroll
    for (int c = 0; c < kCols; c += 32) {
      uint32_t w[16];
#pragma unroll
      for (int i = 0; i < 16; ++i) {
        const float x = s[c + 2 * i], y = s[c + 2 * i + 1];
        float e0, e1;
        split_pair(fma_pair(pair_of(x, y), scale2, base2), e0, e1);
        e0 = exp2_approx(e0);
        top[i & 3] = max3(top[i & 3], x, y);
        e1 = exp2_approx(e1);
        add[i & 1] = add_pair(add[i & 1], pair_of(e0, e1));
        w[i] = pack2<kBf16>(e0, e1);
      }
      tmem_st16(s_addr + c / 2, w);
      if (kTwice) tmem_st16(s_addr + kCols / 2 + c / 2, w);
    }
    const float m = max3(max3(top[0], top[1], top[2]), top[3], top[3]) * scale_log2;
    const bool moves = m > row.ref + kRefSlack;
    if (!__any_sync(0xffffffffu, moves)) break;
    const float to = moves ? m - kRefBelow : row.ref;
    const float f = moves ? exp2_approx(row.ref - to) : 1.0f;
    row.ref = to;
    row.sum *= f;
    if (!first) {
      if (!__all_sync(0xffffffffu, before_rescale())) return false;
      tmem_fence_after();
#pragma unroll
      for (int c = 0; c < 128; c += 16) {  // registers count more than speed
        float o[16];
        tmem_ld16(o_addr + c, o);
        tmem_wait_ld<16>(o);
#pragma unroll
        for (int i = 0; i < 16; ++i) o[i] *= f;
        tmem_st16(o_addr + c, reinterpret_cast<const uint32_t*>(o));
      }
    }
  }
  float a0, a1;
  split_pair(add_pair(add[0], add[1]), a0, a1);
  row.sum += a0 + a1;
  tmem_wait_st();
  return true;
}

// ----------------------------------------------------------------------------- rows in and out
// A warp's 32 rows of 64 bytes through 2 KB of shared memory, so that global memory is read and written
// four lanes to a row: chunk c (16 bytes) of row r sits at r * 64 + ((c ^ (r >> 1 & 3)) << 4), free of
// bank conflicts by rows and by columns.
constexpr int kStageRows = 2048;
__device__ __forceinline__ uint4* staged(uint8_t* buf, int row, int chunk) {
  return reinterpret_cast<uint4*>(buf + row * 64 + ((chunk ^ (row >> 1 & 3)) << 4));
}
// Write 64 bytes `w` per lane to the lane's own address `dst` (skipped where it is NULL).
__device__ __forceinline__ void store_rows64(uint8_t* buf, const uint32_t (&w)[16], uint8_t* dst) {
  const int lane = threadIdx.x & 31;
#pragma unroll
  for (int i = 0; i < 4; ++i) *staged(buf, lane, i) = make_uint4(w[4 * i], w[4 * i + 1], w[4 * i + 2], w[4 * i + 3]);
  __syncwarp();
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int row = 8 * i + (lane >> 2);
    uint8_t* to = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(dst), row));
    if (to) reinterpret_cast<uint4*>(to)[lane & 3] = *staged(buf, row, lane & 3);
  }
  __syncwarp();
}

// ----------------------------------------------------------------------------- merging split rows
// Partial records of rows whose keys were split over items: unnormalised outputs
// o[record][channel / 4][row][4] (a warp's 32 rows write whole lines) and (reference, sum) ml[record][row].
//   M = max ref_k, w_k = 2^(ref_k - M), out = sum w_k o_k / sum w_k sum_k, 0 where nothing was seen.
// Lane = row, so that a warp reads whole lines; `o`, `ml`: of the first record, the warp's first row and
// channel; `rows` live rows.  With few records (kFew) a warp merges 32 rows x 8 channels by itself, else
// the block's eight warps take every eighth record each and a second step adds their parts.  Either
// way the eight channels of a row end in one thread, which writes 16 bytes.
constexpr int kMergeThreads = 256, kFewRecords = 6;
struct MergePart {
  float ref = -INFINITY, sum = 0.0f, acc[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
  // Add records k, k + step, ... (at most kLoads, below n) with all their loads in flight.
  template <int kLoads>
  __device__ __forceinline__ void add(const float2* ml, const float4* o, int64_t ml_step, int64_t o_step, int64_t quad_step,
                                      int k, int step, int n) {
    float2 r[kLoads];
    float4 x[kLoads], y[kLoads];
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      r[i] = make_float2(-INFINITY, 0.0f);
      x[i] = y[i] = make_float4(0.f, 0.f, 0.f, 0.f);
      if (k + i * step < n) {
        r[i] = ml[(k + i * step) * ml_step];
        x[i] = o[(k + i * step) * o_step];
        y[i] = o[(k + i * step) * o_step + quad_step];
      }
    }
    float top = ref;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) top = fmaxf(top, r[i].x);
    const float base = top == -INFINITY ? 0.0f : top, f = exp2_approx(ref - base);
    ref = top;
    sum *= f;
#pragma unroll
    for (int c = 0; c < 8; ++c) acc[c] *= f;
#pragma unroll
    for (int i = 0; i < kLoads; ++i) {
      if (k + i * step >= n) break;
      const float w = exp2_approx(r[i].x - base);
      const float v[8] = {x[i].x, x[i].y, x[i].z, x[i].w, y[i].x, y[i].y, y[i].z, y[i].w};
      sum = fmaf(w, r[i].y, sum);
#pragma unroll
      for (int c = 0; c < 8; ++c) acc[c] = fmaf(w, v[c], acc[c]);
    }
  }
};
// Eight merged channels of this lane's row, in acc.  A warp of its own (kFew), or the first warp of a
// block; the others return false.
template <bool kFew>
__device__ __forceinline__ bool merge_records(MergePart& p, const float2* ml, const float4* o, int64_t ml_step,
                                              int64_t o_step, int64_t quad_step, int n, int rows) {
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (kFew) {
    if (lane < rows)
      for (int k = 0; k < n; k += kFewRecords) p.add<kFewRecords>(ml + lane, o + lane, ml_step, o_step, quad_step, k, 1, n);
  } else {
    __shared__ float part[7][10][32];
    if (lane < rows)
      for (int k = warp; k < n; k += 24) p.add<3>(ml + lane, o + lane, ml_step, o_step, quad_step, k, 8, n);
    if (warp) {
      part[warp - 1][0][lane] = p.ref;
      part[warp - 1][1][lane] = p.sum;
#pragma unroll
      for (int c = 0; c < 8; ++c) part[warp - 1][2 + c][lane] = p.acc[c];
    }
    __syncthreads();
    if (warp) return false;
    float top = p.ref;
#pragma unroll
    for (int k = 0; k < 7; ++k) top = fmaxf(top, part[k][0][lane]);
    const float base = top == -INFINITY ? 0.0f : top, f = exp2_approx(p.ref - base);
    p.sum *= f;
#pragma unroll
    for (int c = 0; c < 8; ++c) p.acc[c] *= f;
#pragma unroll
    for (int k = 0; k < 7; ++k) {
      const float w = exp2_approx(part[k][0][lane] - base);
      p.sum = fmaf(w, part[k][1][lane], p.sum);
#pragma unroll
      for (int c = 0; c < 8; ++c) p.acc[c] = fmaf(w, part[k][2 + c][lane], p.acc[c]);
    }
  }
  const float inv = p.sum == 0.0f ? 0.0f : 1.0f / p.sum;
#pragma unroll
  for (int c = 0; c < 8; ++c) p.acc[c] *= inv;
  return true;
}

// Launch a kernel as the programmatic dependent of the previous one in the stream (which lets it
// start, and which it waits for with griddepcontrol.wait).
template <class Params>
inline cudaError_t launch_dependent(void (*kernel)(Params), dim3 grid, int threads, cudaStream_t s, const Params& p) {
  cudaLaunchConfig_t cfg = {};
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.stream = s;
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  return cudaLaunchKernelEx(&cfg, kernel, p);
}

}  // namespace tp
