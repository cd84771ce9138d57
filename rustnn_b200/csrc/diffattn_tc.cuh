// Differential attention on the fifth-generation tensor cores: what its
// kernels share (PTX, descriptors, tensor maps).  bf16 operands come by tensor
// copies into 128-byte-swizzled tiles; accumulators and the maps between two
// products live in tensor memory.
#pragma once

#include <cuda.h>

#include "diffattn.cuh"
#include "tc_launch.cuh"

namespace rnn {
namespace diff {

using tc::elect_one;
using tc::fence_async_smem;
using tc::fence_barrier_init;
using tc::mbar_arrive;
using tc::mbar_arrive_expect_tx;
using tc::mbar_init;
using tc::smem_u32;
using tc::tc_fence_after;
using tc::tc_fence_before;
using tc::tmem_alloc;
using tc::tmem_dealloc;
using tc::tmem_relinquish;
using tc::tmem_wait_st;

// Tensor copies global -> shared (zero fill outside the tensor, no multicast).
__device__ __forceinline__ void tma_5d(uint32_t dst, const void* map, int c0, int c1, int c2, int c3, int c4,
                                       uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], "
      "[%7];" ::"r"(dst),
      "l"(map), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(smem_u32(bar))
      : "memory");
}

// D(tmem) (+)= A B^T, kind::f16 (bf16 operands, f32 accumulator), one CTA.
// _ss: A from shared memory; _ts: A from tensor memory, two bf16 of a row per
// 32-bit column.  The whole warp runs the issuing loop and only the lane with
// `lead` set issues: the loop then has no divergent branch, which cost more
// than the waits themselves.
__device__ __forceinline__ void mma_ss(uint32_t d, uint64_t a, uint64_t b, uint32_t idesc, bool accumulate,
                                       uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], %1, %2, %3, p;\n\t}" ::"r"(d),
      "l"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(lead)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint64_t b, uint32_t idesc, bool accumulate,
                                       uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.b32 p, %4, 0;\n\t"
      "setp.ne.b32 q, %5, 0;\n\t"
      "@q tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(d),
      "r"(a), "l"(b), "r"(idesc), "r"(accumulate ? 1u : 0u), "r"(lead)
      : "memory");
}
// Arrives on `bar` once the MMAs that this lane has issued are done.
__device__ __forceinline__ void commit(uint64_t* bar, uint32_t lead) {
  asm volatile(
      "{\n\t.reg .pred q;\n\t"
      "setp.ne.b32 q, %1, 0;\n\t"
      "@q tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];\n\t}" ::"r"(smem_u32(bar)),
      "r"(lead)
      : "memory");
}

// Instruction descriptor of kind::f16: f32 accumulator, bf16 operands, A
// K-major; B K-major, or MN-major when b_mn.
__host__ __device__ constexpr uint32_t idesc_bf16(int m, int n, bool b_mn) {
  return (1u << 4) | (1u << 7) | (1u << 10) | (b_mn ? 1u << 16 : 0u) | (static_cast<uint32_t>(n >> 3) << 17) |
         (static_cast<uint32_t>(m >> 4) << 24);
}

// Shared-memory descriptors of SWIZZLE_128B tiles: rows of 128 bytes (64
// bf16), groups of 8 rows 1024 bytes apart.  K-major: a row is an operand row,
// 16 columns (one MMA step) are 32 bytes further.  MN-major: a row is one
// contraction index, 16 of them are 2048 bytes further, and the next 64
// operand rows are `next` bytes away.
__device__ __forceinline__ uint64_t desc_k(uint32_t addr) { return tc::sdesc_sw128(addr); }
__device__ __forceinline__ uint64_t desc_mn(uint32_t addr, uint32_t next) {
  uint64_t d = static_cast<uint64_t>((addr & 0x3FFFFu) >> 4);
  d |= static_cast<uint64_t>(next >> 4) << 16;
  d |= static_cast<uint64_t>(1024 >> 4) << 32;
  d |= static_cast<uint64_t>(1) << 46;
  d |= static_cast<uint64_t>(2) << 61;
  return d;
}

// 32 lanes x N 32-bit columns of tensor memory; the registers hold the values
// only after tmem_landed().
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, "
      "%16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]), "=f"(v[16]),
        "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]), "=f"(v[24]),
        "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31])
      : "r"(addr));
}
// Waits for this thread's loads; the operands tie later uses to the wait.
__device__ __forceinline__ void tmem_landed(float (&v)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]), "+f"(v[15]),
                 "+f"(v[16]), "+f"(v[17]), "+f"(v[18]), "+f"(v[19]), "+f"(v[20]), "+f"(v[21]), "+f"(v[22]),
                 "+f"(v[23]), "+f"(v[24]), "+f"(v[25]), "+f"(v[26]), "+f"(v[27]), "+f"(v[28]), "+f"(v[29]),
                 "+f"(v[30]), "+f"(v[31])::"memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]), "=f"(v[8]),
        "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15])
      : "r"(addr));
}
__device__ __forceinline__ void tmem_landed(float (&v)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7]),
                 "+f"(v[8]), "+f"(v[9]), "+f"(v[10]), "+f"(v[11]), "+f"(v[12]), "+f"(v[13]), "+f"(v[14]),
                 "+f"(v[15])::"memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, float (&v)[8]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x8.b32 {%0, %1, %2, %3, %4, %5, %6, %7}, [%8];"
               : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7])
               : "r"(addr));
}
__device__ __forceinline__ void tmem_landed(float (&v)[8]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;"
               : "+f"(v[0]), "+f"(v[1]), "+f"(v[2]), "+f"(v[3]), "+f"(v[4]), "+f"(v[5]), "+f"(v[6]), "+f"(v[7])::"memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const float (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "f"(v[0]), "f"(v[1]), "f"(v[2]), "f"(v[3]), "f"(v[4]), "f"(v[5]), "f"(v[6]), "f"(v[7]), "f"(v[8]), "f"(v[9]),
      "f"(v[10]), "f"(v[11]), "f"(v[12]), "f"(v[13]), "f"(v[14]), "f"(v[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};" ::"r"(addr),
      "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]),
      "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
      : "memory");
}

__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&v)[8]) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x8.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8};" ::"r"(addr), "r"(v[0]),
               "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7])
               : "memory");
}

// Two f32 operations in one instruction, on register pairs.
typedef unsigned long long f32x2;
__device__ __forceinline__ f32x2 pair(float x, float y) {
  f32x2 d;
  asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(x), "f"(y));
  return d;
}
__device__ __forceinline__ void unpair(f32x2 d, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(d));
}
__device__ __forceinline__ f32x2 fma2(f32x2 a, f32x2 b, f32x2 c) {
  f32x2 d;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
  return d;
}
__device__ __forceinline__ f32x2 add2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ f32x2 mul2(f32x2 a, f32x2 b) {
  f32x2 d;
  asm("mul.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
  return d;
}

__device__ __forceinline__ uint32_t pack2(float lo, float hi) {
  __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
  return *reinterpret_cast<uint32_t*>(&v);
}

// Bounded wait, false when the block is aborting or after 100,000 tries of up to
// 20 microseconds each (2 s, as elsewhere).  It counts tries instead of reading
// the clock, which keeps the code of the loops around it short.
__device__ __forceinline__ bool wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* dev_error) {
  const uint32_t p = smem_u32(bar);
  if (__builtin_expect(tc::mbar_try_wait(p, parity), 1)) return true;
#pragma unroll 1
  for (int i = 0; i < 100000; i++) {
    if (tc::mbar_try_wait_hint(p, parity, 20000u)) return true;
    if (*abort_flag) return false;
  }
  *abort_flag = 1;
  atomicOr(dev_error, DEV_ERR_TIMEOUT);
  return false;
}
// The same for a whole warp, with one outcome.
__device__ __forceinline__ bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag, int* dev_error) {
  return __all_sync(0xffffffffu, wait(bar, parity, abort_flag, dev_error));
}

// Lets what the arrivals of `bar` stand for (copies or MMAs in flight) finish
// before an aborting block returns; bounded like every wait.
__device__ __forceinline__ void settle(uint64_t* bar, uint32_t parity) {
  const unsigned long long t0 = tc::globaltimer();
  while (!tc::mbar_try_wait(smem_u32(bar), parity) && tc::globaltimer() - t0 < tc::WAIT_TIMEOUT_NS) {
  }
}

// Which of a tile's 64 keys from j0 on exist and are not masked (the whole warp
// calls): load() asks memory for them, so that it can run ahead, bits() answers.
struct Seen {
  bool lo, hi;
  __device__ __forceinline__ void load(const uint8_t* mask, int j0, int len) {
    const int j = j0 + (threadIdx.x & 31);
    lo = j < len && (mask == nullptr || mask[j] != 0);
    hi = j + 32 < len && (mask == nullptr || mask[j + 32] != 0);
  }
  __device__ __forceinline__ uint2 bits() const {
    return make_uint2(__ballot_sync(0xffffffffu, lo), __ballot_sync(0xffffffffu, hi));
  }
};
// Clears the rows of a 64-row tile that `seen` leaves out: `parts` pieces of 128
// bytes a row, 8192 bytes apart.  What is hidden may be NaN, and meets P = 0 in a
// product.
__device__ __forceinline__ void clear_hidden(uint8_t* tile, uint2 seen, int parts) {
  const int lane = threadIdx.x & 31;
#pragma unroll 1
  for (int half = 0; half < 2; half++)
    for (uint32_t gone = ~(half ? seen.y : seen.x); gone; gone &= gone - 1) {
      const int r = half * 32 + __ffs(gone) - 1;
      for (int c = lane; c < parts * 8; c += 32)
        *reinterpret_cast<uint4*>(tile + (c >> 3) * 8192 + r * 128 + (c & 7) * 16) = make_uint4(0, 0, 0, 0);
    }
}

// Tensor map of a bf16 view [n, t, heads, 2 halves, dh] read in boxes of 64
// columns of one half and `rows` rows; columns beyond dh and rows beyond t are
// zero.  The contiguous 2*dh columns of v and dout are read with halves == 1.
int encode_map(CUtensorMap* m, const void* base, int n, int t, int heads, int halves, int cols, long long sb,
               long long sr, long long sh, int rows);
// Whether a view can be read so: 16-byte aligned, strides that a map can hold.
bool map_ok(const void* base, int n, int t, int heads, int cols, long long sb, long long sr, long long sh);

// Whether the tensor-core kernels take a call, and the calls themselves (the
// backward's workspace pointers are set).
bool big_enough(const Args& a);  // for a block's start and end to be worth it
bool tc_fwd_ok(const Args& a);
int tc_fwd(rnn_ctx* ctx, const Args& a);
bool tc_bwd_ok(const Args& a);
int tc_bwd(rnn_ctx* ctx, const Args& a);
int tc_bwd_parts(rnn_ctx* ctx, const Args& a);  // parts (256 floats a key each) that its workspace holds
// The same of the kernel for a few rows over a long cache, which leaves parts
// of 128 columns for join_parts when it splits the keys.
bool dec_ok(const Args& a);
int dec_fwd(rnn_ctx* ctx, const Args& a);
int join_parts(rnn_ctx* ctx, const Args& a);
// The tensor-core kernels in f32.
bool f32_tc_ok(const Args& a, bool backward);
int f32_tc_fwd(rnn_ctx* ctx, const Args& a);
int f32_tc_bwd(rnn_ctx* ctx, const Args& a);
// Joins parts of many rows: 128 columns in bf16, 64 in f32.
int join_rows_bf16(rnn_ctx* ctx, const Args& a);
int join_rows_f32(rnn_ctx* ctx, const Args& a);
int join_rows_f32_wide(rnn_ctx* ctx, const Args& a);  // 128

}  // namespace diff
}  // namespace rnn
