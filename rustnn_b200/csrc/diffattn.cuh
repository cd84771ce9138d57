// Differential attention: arguments, masks, tile loads and warp-level matrix
// products shared by its kernels.
//
// A head's score columns come in two halves (q = [q1 | q2], k = [k1 | k2]);
//   s_m = scale q_m k_m^T,  P_m = softmax(s_m),  o = (P_1 - lam P_2) v.
// Query heads that share a key head are packed: row r of a (sequence, key
// head) is query i = r % tq of head e = r / tq of the group, so a tile of rows
// reads each key and value once for the whole group.
#pragma once

#include <cuda_bf16.h>
#include <math_constants.h>
#include <stdint.h>

#include "common.cuh"

namespace rnn {
namespace diff {

struct Args {
  int n, h, hkv, grp, dh, tq, tk, causal;
  float scale, slog2;  // slog2 = scale * log2(e): scores in base-2 units
  long long qb, qr, qh, kb, kr, kh, vb, vr, vh, ob, orow, oh;  // strides, elements
  const void *q, *k, *v;
  const float* lam;
  void *o, *o2;
  float* lse;
  const int* klen;
  const uint8_t* kmask;
  long long kmb;
  int vec;   // 16-byte loads of q, k, v, dout tiles are aligned
  int pair;  // two neighbouring output columns are one aligned store
  // key split of the forward pass
  int nsplit, split_keys;
  float *part, *stat;  // [split][row][2W], [split][row][4]
  // backward
  long long dqb, dqr, dqh, dkb, dkr, dkh, dvb, dvr, dvh, gb, gr, gh;  // strides of dq, dk, dv, dout
  const void *fo, *fo2;
  const float* flse;
  const void* dout;
  void *dq, *dk, *dv;
  float* dlam;
  float* dsum;   // [n, h, 2, tq]: D_1, D_2
  float* dlrow;  // [h, n * tq]: sum_j P_2 dP of each row, in f32
  int kparts;    // parts that the queries of a key tile are split into
  float* kpart;  // [part][n * hkv][tk][256]: dv, dk_1, dk_2 of a part, 64 columns each piece
};

// Leading keys of sequence b that some query may see.  With RNN_CAUSAL_START the
// last query sits at key tq - 1, and what lies beyond is like what lies beyond
// klen: never read into a product, where 0 times it might be NaN.
__device__ __forceinline__ int key_len(const Args& a, int b) {
  const int most = a.causal == RNN_CAUSAL_START ? min(a.tk, a.tq) : a.tk;
  return a.klen ? min(max(__ldg(a.klen + b), 0), most) : most;
}
// A map's normaliser and log-sum from its reference m and sum l.  A sum is 0 only
// where no key counts (none is visible, or every score is -inf): that map is 0,
// its log-sum +inf.  A sum that is not a number, from NaN or infinite scores,
// makes the row NaN, as the formula has it.
__device__ __forceinline__ float inverse(float l) { return l == 0.0f ? 0.0f : 1.0f / l; }
__device__ __forceinline__ float log_sum(float m, float l) { return l == 0.0f ? CUDART_INF_F : m + log2f(l); }

// Number of leading keys that query i of a sequence of `len` keys may see.
__device__ __forceinline__ int row_limit(const Args& a, int i, int len) {
  if (a.causal == RNN_CAUSAL_START) return min(len, i + 1);
  if (a.causal == RNN_CAUSAL_END) return max(0, min(len, i + 1 + len - a.tq));
  return len;
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ uint32_t smem_addr(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void cp16(void* dst, const void* src, bool ok) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(smem_addr(dst)), "l"(src), "r"(ok ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_wait() {
  asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}

template <class T>
__device__ __forceinline__ float to_f(T x);
template <>
__device__ __forceinline__ float to_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ float to_f<__nv_bfloat16>(__nv_bfloat16 x) {
  return __bfloat162float(x);
}
template <class T>
__device__ __forceinline__ T from_f(float x);
template <>
__device__ __forceinline__ float from_f<float>(float x) {
  return x;
}
template <>
__device__ __forceinline__ __nv_bfloat16 from_f<__nv_bfloat16>(float x) {
  return __float2bfloat16_rn(x);
}

// Two neighbouring columns of an output row; `ok0` / `ok1` say which exist.
template <class T>
__device__ __forceinline__ void store2(T* p, float x, float y, bool ok0, bool ok1, bool pair) {
  if (pair && ok1) {
    if constexpr (sizeof(T) == 4) {
      *reinterpret_cast<float2*>(p) = make_float2(x, y);
    } else {
      *reinterpret_cast<__nv_bfloat162*>(p) = __floats2bfloat162_rn(x, y);
    }
    return;
  }
  if (ok0) p[0] = from_f<T>(x);
  if (ok1) p[1] = from_f<T>(y);
}

// ---------------------------------------------------------------- fragments
//
// Warp matrix products of 16 rows x 8 columns.  bf16: one m16n8k16 MMA.  f32:
// each operand is split as hi + lo, hi rounded to TF32 and lo the rest, which TF32
// holds but for an f32's last bit, and three m16n8k8 MMAs form lo hi, hi lo and
// hi hi (lo lo is below 2^-24).  An MMA cuts off, not rounds, what its accumulator
// has no room for, so the small parts have an accumulator of their own and join in
// f32: 16 x 48 x 48, 4 heads of 64: dq off by 5.6e-7, 13e-7 in one chain of all
// parts, 3.2e-7 in plain f32; forward and backward 22 and 79 us, 21 and 79 in one
// chain; each step's product by itself, 2.7e-7 and 23 and 93 us.
// In both, `from_acc` turns accumulator blocks into the A operand of the next
// product without moving data between lanes: for f32 the contraction index is
// renumbered (lane t holds keys 2t and 2t+1), which `ldB_kn` matches.

template <class T>
struct Frag;

template <>
struct Frag<__nv_bfloat16> {
  using T = __nv_bfloat16;
  static constexpr int KS = 16;
  struct A {
    uint32_t x[4];
  };
  struct B {
    uint32_t x[2];
  };
  // rows row0 .. row0+15, columns k0 .. k0+15 of a row-major tile
  static __device__ __forceinline__ A ldA(const T* s, int pitch, int row0, int k0, int lane) {
    A a;
    const uint32_t p = smem_addr(s + (row0 + (lane & 15)) * pitch + k0 + (lane >> 4) * 8);
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                 : "=r"(a.x[0]), "=r"(a.x[1]), "=r"(a.x[2]), "=r"(a.x[3])
                 : "r"(p));
    return a;
  }
  // B operands of N blocks of 8 columns (N even) at n0 from a tile stored [n][k]
  template <int N>
  static __device__ __forceinline__ void ldB_nk(B (&b)[N], const T* s, int pitch, int n0, int k0, int lane) {
    const int mi = lane >> 3;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t p = smem_addr(s + (n0 + 8 * i + (mi >> 1) * 8 + (lane & 7)) * pitch + k0 + (mi & 1) * 8);
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
                   : "=r"(b[i].x[0]), "=r"(b[i].x[1]), "=r"(b[i + 1].x[0]), "=r"(b[i + 1].x[1])
                   : "r"(p));
    }
  }
  // the same from a tile stored [k][n]
  template <int N>
  static __device__ __forceinline__ void ldB_kn(B (&b)[N], const T* s, int pitch, int k0, int n0, int lane) {
    const int mi = lane >> 3;
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint32_t p = smem_addr(s + (k0 + (mi & 1) * 8 + (lane & 7)) * pitch + n0 + 8 * i + (mi >> 1) * 8);
      asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
                   : "=r"(b[i].x[0]), "=r"(b[i].x[1]), "=r"(b[i + 1].x[0]), "=r"(b[i + 1].x[1])
                   : "r"(p));
    }
  }
  static __device__ __forceinline__ uint32_t pack(float lo, float hi) {
    __nv_bfloat162 v = __floats2bfloat162_rn(lo, hi);
    return *reinterpret_cast<uint32_t*>(&v);
  }
  // A operand of contraction step ks from the accumulator blocks c
  template <int NB>
  static __device__ __forceinline__ A from_acc(const float (&c)[NB][4], int ks) {
    return A{{pack(c[2 * ks][0], c[2 * ks][1]), pack(c[2 * ks][2], c[2 * ks][3]),
              pack(c[2 * ks + 1][0], c[2 * ks + 1][1]), pack(c[2 * ks + 1][2], c[2 * ks + 1][3])}};
  }
  static __device__ __forceinline__ void mma(float (&d)[4], const A& a, const B& b) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a.x[0]), "r"(a.x[1]), "r"(a.x[2]), "r"(a.x[3]), "r"(b.x[0]), "r"(b.x[1]));
  }
  // d += a b for N blocks of columns; in f32 m collects the small parts, for join
  template <int N>
  static __device__ __forceinline__ void mma(float (*d)[4], float (*)[4], const A& a, const B (&b)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) mma(d[i], a, b[i]);
  }
  template <int N>
  static __device__ __forceinline__ void join(float (&)[N][4], const float (&)[N][4]) {}
};

template <>
struct Frag<float> {
  using T = float;
  static constexpr int KS = 8;
  struct A {
    uint32_t hi[4], lo[4];
  };
  struct B {
    uint32_t hi[2], lo[2];
  };
  static __device__ __forceinline__ void split(float x, uint32_t& hi, uint32_t& lo) {
    hi = (__float_as_uint(x) + 0x1000u) & 0xFFFFE000u;
    lo = __float_as_uint(x - __uint_as_float(hi));
  }
  static __device__ __forceinline__ A ldA(const T* s, int pitch, int row0, int k0, int lane) {
    A a;
    const T* p = s + (row0 + (lane >> 2)) * pitch + k0 + (lane & 3);
    split(p[0], a.hi[0], a.lo[0]);
    split(p[8 * pitch], a.hi[1], a.lo[1]);
    split(p[4], a.hi[2], a.lo[2]);
    split(p[8 * pitch + 4], a.hi[3], a.lo[3]);
    return a;
  }
  template <int N>
  static __device__ __forceinline__ void ldB_nk(B (&b)[N], const T* s, int pitch, int n0, int k0, int lane) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const T* p = s + (n0 + 8 * i + (lane >> 2)) * pitch + k0 + (lane & 3);
      split(p[0], b[i].hi[0], b[i].lo[0]);
      split(p[4], b[i].hi[1], b[i].lo[1]);
    }
  }
  template <int N>
  static __device__ __forceinline__ void ldB_kn(B (&b)[N], const T* s, int pitch, int k0, int n0, int lane) {
    const T* p = s + (k0 + 2 * (lane & 3)) * pitch + n0 + (lane >> 2);
#pragma unroll
    for (int i = 0; i < N; i++) {
      split(p[8 * i], b[i].hi[0], b[i].lo[0]);
      split(p[pitch + 8 * i], b[i].hi[1], b[i].lo[1]);
    }
  }
  template <int NB>
  static __device__ __forceinline__ A from_acc(const float (&c)[NB][4], int ks) {
    A a;
    split(c[ks][0], a.hi[0], a.lo[0]);
    split(c[ks][2], a.hi[1], a.lo[1]);
    split(c[ks][1], a.hi[2], a.lo[2]);
    split(c[ks][3], a.hi[3], a.lo[3]);
    return a;
  }
  static __device__ __forceinline__ void mma1(float (&d)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
    asm volatile("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  }
  // d += hi hi, m += lo hi + hi lo.
  template <int N>
  static __device__ __forceinline__ void mma(float (*d)[4], float (*m)[4], const A& a, const B (&b)[N]) {
#pragma unroll
    for (int i = 0; i < N; i++) mma1(m[i], a.lo, b[i].hi);
#pragma unroll
    for (int i = 0; i < N; i++) mma1(d[i], a.hi, b[i].hi);
#pragma unroll
    for (int i = 0; i < N; i++) mma1(m[i], a.hi, b[i].lo);
  }
  template <int N>
  static __device__ __forceinline__ void join(float (&d)[N][4], const float (&m)[N][4]) {
#pragma unroll
    for (int i = 0; i < N; i++)
#pragma unroll
      for (int e = 0; e < 4; e++) d[i][e] += m[i][e];
  }
};

// Tile geometry of one (type, padded half width).  PITCH keeps ldmatrix rows
// (bf16) and the scalar fragment loads (f32) free of bank conflicts.
template <class T, int DH>
struct Geo {
  static constexpr int W = 2 * DH;
  static constexpr int E = 16 / sizeof(T);  // elements of a 16-byte chunk
  static constexpr int PITCH = W + E;
  static constexpr int KS = Frag<T>::KS;
  // keys (or queries) of one register step; 16 where the f32 fragments of a
  // 32-wide step would not fit the register file
  static constexpr int SUB = sizeof(T) == 4 && DH == 64 ? 16 : 32;
  // column blocks whose products run side by side: few MMAs in a row wait for
  // one another, as far as registers go
  static constexpr int SIDE = sizeof(T) == 4 && DH < 64 ? 4 : 2;
  static constexpr int HALF_SIDE = SIDE < DH / 8 ? SIDE : DH / 8;  // of one half
};

// Loads ROWS rows of 2*dh columns into a PITCH-wide tile.  row(r) gives the
// source row or null (zero-filled; `any` is then the address a copy of no
// bytes names).  SPLIT tiles (q, k) put the halves at
// columns 0 and DH; the others (v, dout) are contiguous.  Columns without a
// source are zero.  With `vec` the copies are asynchronous (cp.async).
template <class T, int DH, int ROWS, int THREADS, bool SPLIT, class Row>
__device__ __forceinline__ void load_tile(T* dst, const void* any, int dh, bool vec, Row row) {
  using G = Geo<T, DH>;
  if (vec) {
    constexpr int CH = G::W / G::E;
    for (int i = threadIdx.x; i < ROWS * CH; i += THREADS) {
      const int r = i / CH, c = (i % CH) * G::E;
      int src = c;
      bool ok = c < 2 * dh;
      if (SPLIT) {
        const int half = c >= DH ? 1 : 0, w = c - half * DH;
        src = half * dh + w;
        ok = w < dh;
      }
      const T* p = row(r);
      ok = ok && p != nullptr;
      cp16(dst + r * G::PITCH + c, ok ? static_cast<const void*>(p + src) : any, ok);
    }
  } else {
    for (int i = threadIdx.x; i < ROWS * G::W; i += THREADS) {
      const int r = i / G::W, c = i % G::W;
      int src = c;
      bool ok = c < 2 * dh;
      if (SPLIT) {
        const int half = c >= DH ? 1 : 0, w = c - half * DH;
        src = half * dh + w;
        ok = w < dh;
      }
      const T* p = row(r);
      dst[r * G::PITCH + c] = ok && p != nullptr ? p[src] : from_f<T>(0.0f);
    }
  }
}

// D_m = do . P_m v comes from the saved o and o2, whose rounding to bf16 leaves it
// off by some d_m = sum_j dS_j, which is 0 for the true D.  That reaches dq as
// d_m sum_j P_j k_j: nothing beside a row's dS where many keys take part (d is
// about 2^-9 of the norm of dS), but up to all there is where one key holds the row
// or the values have much in common.  So the bf16 kernels sum dS as they go, in
// f32, hand D + d on, and where d passes 2^-6 of a row's norm of dS go over the
// block's keys once more with D + d.  (Squares out of f32's range say nothing.)
// Normal inputs hardly ever do (d stays below 2^-7 of the norm over 500 to 8192
// keys); keys and values whose mean is half their spread do over 8192, where dq was
// off by up to 9 %.  1 x 8192 x 8192, 8 heads of 64, tcgen05, both kernels: 1134 us
// without the sums, 1176 with them, 1615 where all blocks go over their keys again.
__device__ __forceinline__ bool too_far(float d, float norm2) {
  return d * d > norm2 * (1.0f / 4096) || norm2 > 1e30f || (norm2 < 1e-30f && d != 0.0f);
}

__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

}  // namespace diff
}  // namespace rnn
