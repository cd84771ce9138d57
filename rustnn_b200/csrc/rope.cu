// Rotary positions over several axes, forward and backward.
//
// Token r carries A integer coordinates; axis a owns pairs[a] consecutive
// pairs of every head's columns, and pair p turns by
//   angle = pos[r, axis(p)] * inv_freq[p]:
//   y_i = x_i cos - x_j sin,  y_j = x_i sin + x_j cos
// with (i, j) = (p, p + total) or, interleaved, (2p, 2p + 1).  The backward
// pass turns the gradient by -angle.  Columns from 2 * total on are copied.
//
// Bound by HBM: every element is read and written once; the angles of a token
// are worked out once per block in shared memory and shared by all its heads,
// so no table is read.  The product pos * inv_freq (31 bits by 24) is kept whole in
// two f64 numbers and reduced to a fraction of a turn there before sincospif, so
// the error does not grow with position or frequency; the rotation itself is f32,
// rounded once to the tensor's type.  Measured with a cold L2: 32768 x 32 x 64 bf16,
// 49 us, 5.5 TB/s of a copy's 6.55 (48 without what the product's rounding leaves);
// 30011 x 12 x 48 f32 interleaved, 28 us, 4.9 TB/s.
#include <cuda_bf16.h>

#include <algorithm>

#include "common.cuh"

namespace rnn {
namespace {

constexpr int ROPE_THREADS = 256;
constexpr int ROPE_MAX_AXES = 4;
constexpr int ROPE_SMEM_PAIRS = 4096;  // (row, pair) angles a block holds: 32 KB

struct RopeArgs {
  const void* x;
  void* y;
  long long xrow, xhead, yrow, yhead;  // strides in elements
  int rows, heads, dh, total;          // total = rotated pairs per head
  const int* pos;                      // [rows, axes]
  int axes;
  int last[ROPE_MAX_AXES];  // last[a] = pairs of the axes 0 .. a
  const float* freq;        // [total]
  float sign;               // +1 forward, -1 backward
  int rpb;                  // rows per block
  int units, rest;          // vectors per head: rotated, copied
};

template <class T, int V>
struct alignas(sizeof(T) * V) Vec {
  T v[V];
};

__device__ __forceinline__ float to_f(float x) { return x; }
__device__ __forceinline__ float to_f(__nv_bfloat16 x) { return __bfloat162float(x); }
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

// cos and sin of pos * freq; |fraction of a turn| <= 1/2 after the reduction.
__device__ __forceinline__ float2 turn(int pos, float freq) {
  constexpr double INV2PI_HI = 0.15915494309189535;       // 1 / (2 pi) rounded to f64
  constexpr double INV2PI_LO = -9.839338337591243e-18;   // and what the rounding left
  const double t = static_cast<double>(pos) * static_cast<double>(freq);
  const double rest = fma(static_cast<double>(pos), static_cast<double>(freq), -t);  // what t's rounding left
  const double k = rint(t * INV2PI_HI);
  const double f = fma(t, INV2PI_HI, -k) + fma(t, INV2PI_LO, rest * INV2PI_HI);
  float s, c;
  sincospif(static_cast<float>(2.0 * f), &s, &c);
  return make_float2(c, s);
}

// One vector of V elements per step: half-split pairs take two (columns p and
// p + total), interleaved ones hold V / 2 whole pairs.
template <class T, int V, bool INTER>
__global__ void __launch_bounds__(ROPE_THREADS) rope_kernel(RopeArgs a) {
  extern __shared__ float2 cs[];
  const int r0 = blockIdx.x * a.rpb;
  const int nr = min(a.rpb, a.rows - r0);
  for (int i = threadIdx.x; i < nr * a.total; i += ROPE_THREADS) {
    const int r = i / a.total, p = i - r * a.total;
    int ax = 0;
#pragma unroll
    for (int k = 0; k < ROPE_MAX_AXES - 1; k++) ax += (k < a.axes - 1 && p >= a.last[k]) ? 1 : 0;
    float2 t = turn(__ldg(a.pos + static_cast<long long>(r0 + r) * a.axes + ax), __ldg(a.freq + p));
    t.y *= a.sign;
    cs[i] = t;
  }
  __syncthreads();
  const T* x = static_cast<const T*>(a.x);
  T* y = static_cast<T*>(a.y);
  const int per = a.units + a.rest, per_row = per * a.heads, count = nr * per_row;
  using VT = Vec<T, V>;
  // Interleaved pairs: four vectors a thread at a time, their loads in flight
  // together (30011 x 12 x 48 f32: 39.6 -> 25.8 us).  Half-split pairs have two
  // loads a step already, and four steps' worth costs warps (32768 x 32 x 64
  // bf16: 74.7 against 45.6 us).
  constexpr int U = INTER ? 4 : 1;
  constexpr bool PAIR = INTER && V == 1;  // a pair is two single elements
  for (int i0 = threadIdx.x; i0 < count; i0 += U * ROPE_THREADS) {
    VT v[U], w[U];
    long long to[U];
    int at[U];  // where the vector's angles start, or -1 for a copy
#pragma unroll
    for (int k = 0; k < U; k++) {
      const int i = i0 + k * ROPE_THREADS;
      if (i >= count) break;
      const int r = i / per_row, hu = i - r * per_row;
      const int hd = hu / per, u = hu - hd * per;
      const bool copy = u >= a.units;
      const int c = copy ? 2 * a.total + (u - a.units) * V : PAIR ? 2 * u : u * V;
      const T* src = x + (r0 + r) * a.xrow + hd * a.xhead + c;
      to[k] = (r0 + r) * a.yrow + hd * a.yhead + c;
      at[k] = copy ? -1 : r * a.total + (INTER && V > 1 ? u * (V / 2) : u * V);
      v[k] = *reinterpret_cast<const VT*>(src);
      if (!copy && (!INTER || PAIR)) w[k] = *reinterpret_cast<const VT*>(src + (INTER ? 1 : a.total));
    }
#pragma unroll
    for (int k = 0; k < U; k++) {
      if (i0 + k * ROPE_THREADS >= count) break;
      T* dst = y + to[k];
      const float2* t = cs + at[k];
      if (at[k] >= 0) {
        if constexpr (INTER && V > 1) {
#pragma unroll
          for (int e = 0; e < V / 2; e++) {
            const float2 z = t[e];
            const float p = to_f(v[k].v[2 * e]), q = to_f(v[k].v[2 * e + 1]);
            v[k].v[2 * e] = from_f<T>(p * z.x - q * z.y);
            v[k].v[2 * e + 1] = from_f<T>(p * z.y + q * z.x);
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; e++) {
            const float2 z = t[e];
            const float p = to_f(v[k].v[e]), q = to_f(w[k].v[e]);
            v[k].v[e] = from_f<T>(p * z.x - q * z.y);
            w[k].v[e] = from_f<T>(p * z.y + q * z.x);
          }
          *reinterpret_cast<VT*>(dst + (INTER ? 1 : a.total)) = w[k];
        }
      }
      *reinterpret_cast<VT*>(dst) = v[k];
    }
  }
}

template <class T, int V, bool INTER>
int rope_launch(rnn_ctx* ctx, RopeArgs a) {
  a.units = INTER && V > 1 ? 2 * a.total / V : a.total / V;
  a.rest = (a.dh - 2 * a.total) / V;
  // Rows per block: about eight vectors per thread, so that a token's angles
  // are shared by a long stretch of loads, but fewer rows when that would
  // leave SMs idle (a few decoded tokens), and no more than the angles fit.
  const long long per_row = static_cast<long long>(a.units + a.rest) * a.heads;
  long long rpb = std::max<long long>(1, 8ll * ROPE_THREADS / std::max<long long>(1, per_row));
  rpb = std::min<long long>(rpb, (a.rows + 4ll * ctx->num_sms - 1) / (4ll * ctx->num_sms));
  rpb = std::min<long long>(rpb, std::max(1, ROPE_SMEM_PAIRS / std::max(1, a.total)));
  a.rpb = static_cast<int>(std::max<long long>(1, rpb));
  const int grid = (a.rows - 1) / a.rpb + 1;
  rope_kernel<T, V, INTER>
      <<<grid, ROPE_THREADS, static_cast<size_t>(a.rpb) * a.total * sizeof(float2), ctx->stream>>>(a);
  RNN_CHECK_LAUNCH();
  return RNN_OK;
}

// The widest vector (16 bytes at most) that pointers, strides and the column
// counts allow.
template <class T>
int rope_dispatch(rnn_ctx* ctx, const RopeArgs& a, bool inter) {
  auto fits = [&](long long v) {
    const long long bytes = v * static_cast<long long>(sizeof(T));
    if (reinterpret_cast<uintptr_t>(a.x) % bytes || reinterpret_cast<uintptr_t>(a.y) % bytes) return false;
    if (a.xrow % v || a.xhead % v || a.yrow % v || a.yhead % v) return false;
    if (inter) return (2 * a.total) % v == 0 && (a.dh - 2 * a.total) % v == 0;
    return a.total % v == 0 && (a.dh - 2 * a.total) % v == 0;
  };
  constexpr int W = 16 / sizeof(T);
  if (inter) {
    if (fits(W)) return rope_launch<T, W, true>(ctx, a);
    if (fits(W / 2)) return rope_launch<T, W / 2, true>(ctx, a);
    if (W / 2 > 2 && fits(2)) return rope_launch<T, 2, true>(ctx, a);
    return rope_launch<T, 1, true>(ctx, a);
  }
  if (fits(W)) return rope_launch<T, W, false>(ctx, a);
  if (fits(W / 2)) return rope_launch<T, W / 2, false>(ctx, a);
  if (W / 2 > 2 && fits(2)) return rope_launch<T, 2, false>(ctx, a);
  return rope_launch<T, 1, false>(ctx, a);
}

}  // namespace
}  // namespace rnn

using namespace rnn;

extern "C" int rnn_rope_dev(rnn_ctx* ctx, int dtype, const void* x, long long xrow, long long xhead, int rows, int heads,
                            int dh, const int32_t* pos, int axes, const int* pairs, const float* inv_freq,
                            int interleaved, int backward, void* y, long long yrow, long long yhead) {
  RNN_REQUIRE(ctx != nullptr, "null context");
  RNN_REQUIRE(dtype == RNN_F32 || dtype == RNN_BF16, "rope: unknown dtype %d", dtype);
  RNN_REQUIRE(rows >= 0 && heads >= 1 && dh >= 1 && dh <= 8192 && (long long)heads * dh < (1ll << 30),
              "rope: bad shape rows=%d heads=%d dh=%d", rows, heads, dh);
  RNN_REQUIRE(axes >= 1 && axes <= ROPE_MAX_AXES && pairs != nullptr, "rope: 1 to %d axes, got %d", ROPE_MAX_AXES, axes);
  RopeArgs a{};
  long long total = 0;
  for (int i = 0; i < axes; i++) {
    RNN_REQUIRE(pairs[i] >= 0 && pairs[i] <= dh, "rope: axis %d has %d pairs", i, pairs[i]);
    total += pairs[i];
    a.last[i] = (int)total;
  }
  RNN_REQUIRE(2 * total <= dh, "rope: %lld pairs do not fit %d columns", total, dh);
  if (rows == 0) return RNN_OK;
  RNN_REQUIRE(x != nullptr && y != nullptr && pos != nullptr && (total == 0 || inv_freq != nullptr), "rope: null pointer");
  RNN_REQUIRE(xrow >= 0 && xhead >= 0, "rope: negative input stride");
  // no two (row, head) of the output may share an element
  const bool rows_outer = (heads == 1 || yhead >= dh) && (rows == 1 || yrow >= (heads - 1) * yhead + dh);
  const bool heads_outer = (rows == 1 || yrow >= dh) && (heads == 1 || yhead >= (long long)(rows - 1) * yrow + dh);
  RNN_REQUIRE(yrow >= 0 && yhead >= 0 && (rows_outer || heads_outer), "rope: output rows or heads overlap");
  const size_t esz = dtype == RNN_F32 ? 4 : 2;
  RNN_REQUIRE(reinterpret_cast<uintptr_t>(x) % esz == 0 && reinterpret_cast<uintptr_t>(y) % esz == 0 &&
                  reinterpret_cast<uintptr_t>(pos) % 4 == 0 && reinterpret_cast<uintptr_t>(inv_freq) % 4 == 0,
              "rope: misaligned pointer");
  RNN_RANGE(x, ((rows - 1) * xrow + (heads - 1) * xhead + dh) * esz);
  RNN_RANGE(y, ((rows - 1) * yrow + (heads - 1) * yhead + dh) * esz);
  RNN_RANGE(pos, (size_t)rows * axes * 4);
  RNN_RANGE(inv_freq, (size_t)total * 4);
  a.x = x;
  a.y = y;
  // the stride of an axis of one element is never used: 0 keeps it out of the alignment rule
  a.xrow = rows == 1 ? 0 : xrow;
  a.xhead = heads == 1 ? 0 : xhead;
  a.yrow = rows == 1 ? 0 : yrow;
  a.yhead = heads == 1 ? 0 : yhead;
  a.rows = rows;
  a.heads = heads;
  a.dh = dh;
  a.total = (int)total;
  a.pos = pos;
  a.axes = axes;
  a.freq = inv_freq;
  a.sign = backward ? -1.0f : 1.0f;
  return dtype == RNN_F32 ? rope_dispatch<float>(ctx, a, interleaved != 0)
                          : rope_dispatch<__nv_bfloat16>(ctx, a, interleaved != 0);
}
