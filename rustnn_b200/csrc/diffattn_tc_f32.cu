// Differential attention in f32 on tcgen05: every stride and mask, forward and
// backward.
//
// An f32 operand is split into three bf16 planes, x = h + m + l with h, m, l the
// rounded value, the rounded rest and its rest (24 bits), and a product is six
// bf16 MMAs: l h, h l, m m, m h, h m, h h (what is left out is below 2^-24).
// The small ones come first and every key tile's product starts from zero and
// joins the f32 accumulators in registers, so that the accumulation in tensor
// memory rounds few large sums.
//
// Operands go through registers to be split, so they are read with plain loads
// (any stride, masked keys as zeros) and written as 128-byte-swizzled tiles:
// rows of 64 columns, the two halves of q and k side by side, or (more than 32
// columns) in tiles of their own.  A block owns 128
// packed rows (queries of a key head's group, or keys) and has 8 arithmetic
// warps, two threads a row with 32 columns each, 7 loading warps and one that
// issues MMAs.  Measured: 32 x 256 x 256, 4 heads of 32: 34 us forward and 91
// backward; a step of 64 columns takes about 2 us, of which its 72 (forward), 96
// and 120 MMAs are 1.5; a block's start and end take 9, and 256 blocks are two
// rounds of 148.
#include <algorithm>
#include <type_traits>

#include "diffattn_tc.cuh"

namespace rnn {
namespace diff {
namespace {

constexpr int ROWS = 128, COLS = 64;  // of a block; of a step
constexpr int THREADS = 512;
constexpr int MATH_WARPS = 8, LOAD_WARPS = 7, WARP_MMA = 15, LOADERS = LOAD_WARPS * 32;
constexpr uint32_t ROW_PLANE = ROWS * 128, COL_PLANE = COLS * 128;  // bytes
constexpr uint32_t ROW_TILE = 3 * ROW_PLANE, COL_TILE = 3 * COL_PLANE;
constexpr int FWD_STAGES = 3, BWD_STAGES = 2;

// Tensor memory columns.  Forward: S_1 S_2 | planes of P_1, P_2 | P_1 v, P_2 v.
// Queries' backward: S_1 S_2 dP | planes of dS_1, dS_2 | dq.  Keys' backward:
// four places for three planes each, of which the first three take S_1, S_2 and
// dP first, from column 16 on, so that a thread's planes overwrite its own
// scores alone: P_1 - lam P_2 takes S_2's place, dS_1 dP's, dS_2 the fourth |
// dv, dk.
constexpr uint32_t MAP = 96, PART = 48;  // three planes of 64 bf16 values; of a thread's 32
// where the 16 values of step ks of a plane start
__device__ __forceinline__ uint32_t plane_at(int plane, int ks) { return PART * (ks >> 1) + 16 * plane + 8 * (ks & 1); }
constexpr uint32_t FWD_P = 128, FWD_O = FWD_P + 2 * MAP;
constexpr uint32_t Q_P = 192, Q_O = Q_P + 2 * MAP;
constexpr uint32_t KV_O = 4 * MAP, KV_S = 16;

struct Shared {
  uint64_t rows_full, d_full, full[FWD_STAGES], empty[FWD_STAGES], s_full, s_free, dp_full, p_full, ds_full, o_full, pair[4], drain;
  uint32_t tmem;
  int abort_flag;
  float2 give[2][2][ROWS], d[ROWS];
  uint32_t seen[FWD_STAGES][2];  // keys of a tile that exist and are not masked
  alignas(16) float stat[BWD_STAGES][5][COLS];  // -lse_1, -lse_2, -D_1, -D_2, limit of a tile's queries
  int least[BWD_STAGES][2];                     // least limit of 32 of them
};
constexpr size_t FWD_SMEM = 1024 + ROW_TILE + FWD_STAGES * 2 * COL_TILE + sizeof(Shared);
constexpr size_t FWD_WIDE_SMEM = 1024 + 2 * ROW_TILE + 3 * COL_TILE + sizeof(Shared);
constexpr size_t GRAD_SMEM = 1024 + ROW_TILE + BWD_STAGES * 3 * COL_TILE + sizeof(Shared);
constexpr size_t DV_SMEM = 1024 + 2 * ROW_TILE + 4 * COL_TILE + sizeof(Shared);
static_assert(GRAD_SMEM <= 232448, "fits an SM");
constexpr size_t BWD_SMEM = 1024 + 2 * ROW_TILE + BWD_STAGES * 2 * COL_TILE + sizeof(Shared);

struct Params {
  Args a;
  int* dev_error;  // the context's error word
  int st16;        // 16-byte stores of the outputs are aligned
  int st16_2;      // and of o2
  int ld16;        // 16-byte loads of dout, o and o2 are aligned
};

// Two values as three planes of bf16 pairs.
__device__ __forceinline__ void split3(float x, float y, uint32_t& h, uint32_t& m, uint32_t& l) {
  const f32x2 minus = pair(-1.0f, -1.0f);
  h = pack2(x, y);
  f32x2 r = fma2(pair(__uint_as_float(h << 16), __uint_as_float(h & 0xffff0000u)), minus, pair(x, y));
  unpair(r, x, y);
  m = pack2(x, y);
  r = fma2(pair(__uint_as_float(m << 16), __uint_as_float(m & 0xffff0000u)), minus, r);
  unpair(r, x, y);
  l = pack2(x, y);
}

// Eight columns (chunk c) of a row of 2*dh values, zeros beyond; p is the row or
// null.  SPLIT rows (q, k) put the halves at columns 0 and 32.  VEC: 16-byte
// loads are aligned and dh is a multiple of 4.
template <bool SPLIT, bool VEC>
__device__ __forceinline__ void load8(float (&x)[8], const float* p, int c, int dh) {
  const int w = SPLIT ? (c & 3) * 8 : c * 8, in = p == nullptr ? 0 : (SPLIT ? dh : 2 * dh) - w;
  p += w + (SPLIT ? (c >> 2) * dh : 0);
  if (VEC) {
    float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
    if (in >= 4) u = __ldg(reinterpret_cast<const float4*>(p));
    if (in >= 8) v = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = k < in ? __ldg(p + k) : 0.0f;
  }
}
// Their planes, as chunk c of row r of a tile of R rows.
template <int R>
__device__ __forceinline__ void store8(uint8_t* dst, const float (&x)[8], int r, int c) {
  uint32_t z[3][4];
#pragma unroll
  for (int k = 0; k < 4; k++) split3(x[2 * k], x[2 * k + 1], z[0][k], z[1][k], z[2][k]);
#pragma unroll
  for (int q = 0; q < 3; q++)
    *reinterpret_cast<uint4*>(dst + q * (R * 128) + r * 128 + ((c ^ (r & 7)) << 4)) =
        make_uint4(z[q][0], z[q][1], z[q][2], z[q][3]);
}
// The block's own 128 rows, by the arithmetic warps (thread t of 256), which
// have nothing else to do then: a thread takes chunk t % 8 of four rows.
constexpr int OWN = ROWS * 8 / (MATH_WARPS * 32);
__device__ __forceinline__ int own_row(int t, int u) { return (t >> 3) + u * (ROWS / OWN); }

// Rows of two tensors, the first scaled; x(u) and y(u) give the places of the
// thread's row u.  Aligned loads are all in flight at once; the others take one
// row after the other, which keeps the code that runs once per block short.
template <bool TWO, class X, class Y>
__device__ __forceinline__ void load_own(uint8_t* dst, const Args& a, int t, float scale, X x, Y y) {
  auto put = [&](float (&v)[8], uint8_t* to, int u, float f) {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] *= f;
    store8<ROWS>(to, v, own_row(t, u), t & 7);
  };
  if (a.vec) {
    float v[OWN][8], w[OWN][8];
#pragma unroll
    for (int u = 0; u < OWN; u++) load8<true, true>(v[u], x(u), t & 7, a.dh);
#pragma unroll
    for (int u = 0; TWO && u < OWN; u++) load8<false, true>(w[u], y(u), t & 7, a.dh);
#pragma unroll
    for (int u = 0; u < OWN; u++) put(v[u], dst, u, scale);
#pragma unroll
    for (int u = 0; TWO && u < OWN; u++) put(w[u], dst + ROW_TILE, u, 1.0f);
  } else {
#pragma unroll 1
    for (int u = 0; u < OWN; u++) {
      float v[8];
      load8<true, false>(v, x(u), t & 7, a.dh);
      put(v, dst, u, scale);
      if (TWO) {
        load8<false, false>(v, y(u), t & 7, a.dh);
        put(v, dst + ROW_TILE, u, 1.0f);
      }
    }
  }
}
// A packed row's place, or null: head e of the group and query i, from `base` on.
__device__ __forceinline__ const float* packed(const float* base, const Args& a, int r, int rows, long long sr,
                                               long long sh) {
  const int e = r / a.tq;
  return r < rows ? base + e * sh + (r - e * a.tq) * sr : nullptr;
}

// Two tiles of a step (k and v, or q and dout), by the loading warps.  ready()
// waits until their place is free, false if it never is; aligned loads go before
// it, so that only the stores follow.
template <class First, class Second, class Ready>
__device__ __forceinline__ bool load_step(uint8_t* dst, const Args& a, int t, First first, Second second, Ready ready) {
  constexpr int ITEMS = COLS * 8, N = (2 * ITEMS + LOADERS - 1) / LOADERS;
  if (a.vec) {
    float x[N][8];
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int i = t + u * LOADERS, r = (i & (ITEMS - 1)) >> 3;
      if (i < ITEMS) {
        load8<true, true>(x[u], first(r), i & 7, a.dh);
      } else if (i < 2 * ITEMS) {
        load8<false, true>(x[u], second(r), i & 7, a.dh);
      }
    }
    if (!ready()) return false;
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int i = t + u * LOADERS, r = (i & (ITEMS - 1)) >> 3;
      if (i < 2 * ITEMS) store8<COLS>(dst + (i < ITEMS ? 0 : COL_TILE), x[u], r, i & 7);
    }
  } else {
    if (!ready()) return false;
#pragma unroll 1
    for (int i = t; i < 2 * ITEMS; i += LOADERS) {
      const int r = (i & (ITEMS - 1)) >> 3;
      float x[8];
      if (i < ITEMS) {
        load8<true, false>(x, first(r), i & 7, a.dh);
      } else {
        load8<false, false>(x, second(r), i & 7, a.dh);
      }
      store8<COLS>(dst + (i < ITEMS ? 0 : COL_TILE), x, r, i & 7);
    }
  }
  return true;
}

// Halves of more than 32 columns take tiles of their own, 64 columns each:
// chunk c of a tile's row at p, `in` of whose columns exist.
template <bool VEC>
__device__ __forceinline__ void load8_wide(float (&x)[8], const float* p, int c, int in) {
  in = p == nullptr ? 0 : in - c * 8;
  p += c * 8;
  if (VEC) {
    float4 u = make_float4(0.0f, 0.0f, 0.0f, 0.0f), v = u;
    if (in >= 4) u = __ldg(reinterpret_cast<const float4*>(p));
    if (in >= 8) v = __ldg(reinterpret_cast<const float4*>(p) + 1);
    x[0] = u.x, x[1] = u.y, x[2] = u.z, x[3] = u.w;
    x[4] = v.x, x[5] = v.y, x[6] = v.z, x[7] = v.w;
  } else {
#pragma unroll
    for (int k = 0; k < 8; k++) x[k] = k < in ? __ldg(p + k) : 0.0f;
  }
}
// One tile of the block's own rows; row(u) is where the thread's row u starts.
template <class Row>
__device__ __forceinline__ void own_wide(uint8_t* dst, const Args& a, int t, int in, float scale, Row row) {
  auto put = [&](float (&v)[8], int u) {
#pragma unroll
    for (int k = 0; k < 8; k++) v[k] *= scale;
    store8<ROWS>(dst, v, own_row(t, u), t & 7);
  };
  if (a.vec) {
    float v[OWN][8];
#pragma unroll
    for (int u = 0; u < OWN; u++) load8_wide<true>(v[u], row(u), t & 7, in);
#pragma unroll
    for (int u = 0; u < OWN; u++) put(v[u], u);
  } else {
#pragma unroll 1
    for (int u = 0; u < OWN; u++) {
      float v[8];
      load8_wide<false>(v, row(u), t & 7, in);
      put(v, u);
    }
  }
}
// TILES tiles of a step, as load_step: src(i, r) is where row r of tile i
// starts, in(i) how many of its columns exist.
template <int TILES, class Src, class In, class Ready>
__device__ __forceinline__ bool step_wide(uint8_t* dst, const Args& a, int t, Src src, In in, Ready ready) {
  constexpr int ITEMS = COLS * 8, N = (TILES * ITEMS + LOADERS - 1) / LOADERS;
  if (a.vec) {
    float x[N][8];
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int i = t + u * LOADERS, tile = i / ITEMS, r = (i & (ITEMS - 1)) >> 3;
      if (i < TILES * ITEMS) load8_wide<true>(x[u], src(tile, r), i & 7, in(tile));
    }
    if (!ready()) return false;
#pragma unroll
    for (int u = 0; u < N; u++) {
      const int i = t + u * LOADERS, tile = i / ITEMS, r = (i & (ITEMS - 1)) >> 3;
      if (i < TILES * ITEMS) store8<COLS>(dst + tile * COL_TILE, x[u], r, i & 7);
    }
  } else {
    if (!ready()) return false;
#pragma unroll 1
    for (int i = t; i < TILES * ITEMS; i += LOADERS) {
      const int tile = i / ITEMS, r = (i & (ITEMS - 1)) >> 3;
      float x[8];
      load8_wide<false>(x, src(tile, r), i & 7, in(tile));
      store8<COLS>(dst + tile * COL_TILE, x, r, i & 7);
    }
  }
  return true;
}

// The planes of a thread's 32 values of a map: its 48 columns of the map's 96.
__device__ __forceinline__ void store_planes(uint32_t dst, const float (&s)[32]) {
#pragma unroll
  for (int g = 0; g < 2; g++) {
    uint32_t z[3][8];
#pragma unroll
    for (int k = 0; k < 8; k++) split3(s[g * 16 + 2 * k], s[g * 16 + 2 * k + 1], z[0][k], z[1][k], z[2][k]);
#pragma unroll
    for (int q = 0; q < 3; q++) tmem_st(dst + q * 16 + g * 8, z[q]);
  }
}

// acc <- al acc + 32 columns of tensor memory.
__device__ __forceinline__ void add_tmem(uint32_t src, float (&acc)[32], float al) {
  const f32x2 f = pair(al, al);
#pragma unroll
  for (int g = 0; g < 2; g++) {
    float x[16];
    tmem_ld(src + g * 16, x);
    tmem_landed(x);
#pragma unroll
    for (int k = 0; k < 16; k += 2) {
      float &u = acc[g * 16 + k], &v = acc[g * 16 + k + 1];
      unpair(fma2(pair(u, v), f, pair(x[k], x[k + 1])), u, v);
    }
  }
}
// s <- 2^(s - u); returns the sum.
__device__ __forceinline__ float exp_sum(float (&s)[32], float u) {
  const f32x2 uu = pair(-u, -u);
  f32x2 t[2] = {0ull, 0ull};
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float &x = s[2 * i], &y = s[2 * i + 1];
    unpair(add2(pair(x, y), uu), x, y);
    x = ex2(x);
    y = ex2(y);
    t[i & 1] = add2(t[i & 1], pair(x, y));
  }
  float x, y;
  unpair(add2(t[0], t[1]), x, y);
  return x + y;
}
__device__ __forceinline__ float max_of(const float (&s)[32]) {
  float m[2] = {s[0], s[1]};
#pragma unroll
  for (int c = 2; c < 32; c++) m[c & 1] = fmaxf(m[c & 1], s[c]);
  return fmaxf(m[0], m[1]);
}

// The six products of two operands in planes, the small ones first.
template <int KMAX, class Step>
__device__ __forceinline__ void products(int ksteps, Step step) {
  constexpr int PA[6] = {2, 0, 1, 1, 0, 0}, PB[6] = {0, 2, 1, 0, 1, 0};
#pragma unroll
  for (int p = 0; p < 6; p++)
#pragma unroll
    for (int ks = 0; ks < KMAX; ks++)
      if (ks < ksteps) step(PA[p], PB[p], ks, p > 0 || ks > 0);
}

// A warp's 32 rows x 32 columns, a row a thread, to rows in memory: through
// shared memory, so that eight threads store 128 bytes of a row.  `to` is where
// the thread's row goes, or null; `in` of its columns exist.
__device__ __forceinline__ void store_rows(float* patch, const float (&x)[32], int in, bool st16, float* to) {
  const int lane = threadIdx.x & 31, c = lane & 7;
#pragma unroll
  for (int k = 0; k < 8; k++)
    *reinterpret_cast<float4*>(patch + lane * 32 + ((k ^ (lane & 7)) << 2)) =
        make_float4(x[4 * k], x[4 * k + 1], x[4 * k + 2], x[4 * k + 3]);
  __syncwarp();
  float* p[8];
  float4 v[8];
#pragma unroll
  for (int k = 0; k < 8; k++) {
    const int r = k * 4 + (lane >> 3);
    p[k] = reinterpret_cast<float*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(to), r));
    v[k] = *reinterpret_cast<const float4*>(patch + r * 32 + ((c ^ (r & 7)) << 2));
  }
  in -= c * 4;
  if (st16) {
#pragma unroll
    for (int k = 0; k < 8; k++)
      if (p[k] != nullptr && in >= 4) *reinterpret_cast<float4*>(p[k] + c * 4) = v[k];
  }
  if (!st16 || (in > 0 && in < 4)) {
#pragma unroll
    for (int k = 0; k < 8; k++) {
      const float z[4] = {v[k].x, v[k].y, v[k].z, v[k].w};
#pragma unroll
      for (int e = 0; e < 4; e++)
        if (p[k] != nullptr && e < in) p[k][c * 4 + e] = z[e];
    }
  }
  __syncwarp();
}

struct Block {
  Shared& sh;
  int* dev_error;
  __device__ __forceinline__ bool done(uint64_t* bar, uint32_t parity) {
    return warp_wait(bar, parity, &sh.abort_flag, dev_error);
  }
  // What the two threads of a row tell each other; `turn` counts the exchanges.
  __device__ __forceinline__ bool exchange(int& turn, int w, int part, int row, float2 mine, float2& other) {
    sh.give[turn & 1][part][row] = mine;
    __syncwarp();
    if ((threadIdx.x & 31) == 0) mbar_arrive(&sh.pair[w]);
    if (!done(&sh.pair[w], turn & 1)) return false;
    other = sh.give[turn & 1][part ^ 1][row];
    turn++;
    return true;
  }
};

__device__ __forceinline__ void setup(Shared& sh, int warp) {
  if (threadIdx.x == 0) {
    mbar_init(&sh.rows_full, MATH_WARPS);
    mbar_init(&sh.d_full, MATH_WARPS);
    for (int i = 0; i < FWD_STAGES; i++) {
      mbar_init(&sh.full[i], LOAD_WARPS);
      mbar_init(&sh.empty[i], 1);
    }
    mbar_init(&sh.s_full, 1);
    mbar_init(&sh.s_free, MATH_WARPS);
    mbar_init(&sh.dp_full, 1);
    mbar_init(&sh.p_full, MATH_WARPS);
    mbar_init(&sh.ds_full, MATH_WARPS);
    mbar_init(&sh.o_full, 1);
    for (int i = 0; i < 4; i++) mbar_init(&sh.pair[i], 2);
    mbar_init(&sh.drain, 1);
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
}
__device__ __forceinline__ void signal(uint64_t* bar) {
  __syncwarp();
  if ((threadIdx.x & 31) == 0) mbar_arrive(bar);
}

// Loads tiles of keys [kbeg, kend) for the kernels that own query rows.
template <bool WIDE>
__device__ __forceinline__ void load_keys(Block& blk, uint8_t* stages, int nstage, const Args& a, int b, int kvh,
                                          int kbeg, int kend, int nt, int t0, int col0) {
  const float* kp = static_cast<const float*>(a.k) + b * a.kb + kvh * a.kh;
  const float* vp = static_cast<const float*>(a.v) + b * a.vb + kvh * a.vh;
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;
  for (int t = 0; t < nt; t++) {
    const int st = t % nstage, j0 = kbeg + t * COLS;
    auto on = [&](int r) { return j0 + r < kend && (!mask || mask[j0 + r]); };
    const uint32_t bits = __ballot_sync(0xffffffffu, t0 < COLS && on(t0));
    auto ready = [&] { return t < nstage || blk.done(&blk.sh.empty[st], (t / nstage - 1) & 1); };
    bool ok;
    if constexpr (WIDE) {  // both halves of k, 64 columns of v
      ok = step_wide<3>(stages + st * (3 * COL_TILE), a, t0,
                        [&](int i, int r) -> const float* {
                          if (!on(r)) return nullptr;
                          return i < 2 ? kp + (j0 + r) * a.kr + i * a.dh : vp + (j0 + r) * a.vr + col0;
                        },
                        [&](int i) { return i < 2 ? a.dh : 2 * a.dh - col0; }, ready);
    } else {
      ok = load_step(stages + st * (2 * COL_TILE), a, t0, [&](int r) { return on(r) ? kp + (j0 + r) * a.kr : nullptr; },
                     [&](int r) { return on(r) ? vp + (j0 + r) * a.vr : nullptr; }, ready);
    }
    if (!ok) break;
    if (t0 < COLS && (t0 & 31) == 0) blk.sh.seen[st][t0 >> 5] = bits;
    fence_async_smem();
    signal(&blk.sh.full[st]);
  }
}

// WIDE: halves of 33 to 64 columns.  q and k take two tiles each, and a block
// computes 64 of the value columns (blockIdx.z), the scores of both twice: there
// is no room for more, in shared memory or in registers.
template <bool WIDE>
__global__ void __launch_bounds__(THREADS, 1) f32_fwd_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  constexpr int STG = WIDE ? 1 : FWD_STAGES;
  constexpr uint32_t STAGE = (WIDE ? 3 : 2) * COL_TILE, V_AT = WIDE ? 2 * COL_TILE : COL_TILE;
  constexpr uint32_t Q_HALF = WIDE ? ROW_TILE : 64, K_HALF = WIDE ? COL_TILE : 64;  // bytes from one half to the other
  constexpr int PART_W = WIDE ? 128 : 64;
  uint8_t* stages = base + (WIDE ? 2 : 1) * ROW_TILE;
  Shared& sh = *reinterpret_cast<Shared*>(stages + STG * STAGE);
  const int col0 = WIDE ? blockIdx.z * 64 : 0;  // first value column
  Block blk{sh, p.dev_error};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.grp * a.tq, nbh = a.n * a.hkv, ntile = (rows + ROWS - 1) / ROWS;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;  // longest causal rows first
  const int bh = static_cast<int>(blockIdx.x) % nbh, b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int row0 = tile * ROWS, len = key_len(a, b);
  const int last = min(rows, row0 + ROWS) - 1;
  // a block that spans a head's end holds that head's last query
  const int imax = last / a.tq != row0 / a.tq ? a.tq - 1 : last % a.tq;
  const int kbeg = static_cast<int>(blockIdx.y) * a.split_keys;
  const int kend = min(row_limit(a, imax, len), kbeg + a.split_keys);
  const int nt = max(kend - kbeg + COLS - 1, 0) / COLS;
  setup(sh, warp);
  const uint32_t tmem = sh.tmem;

  if (warp < MATH_WARPS) {
    // registers: 512 threads x 128 at launch = 256 x 168 + 256 x 88
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    if (nt > 0) {
      const float* q = static_cast<const float*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
      auto at_q = [&](int u) { return packed(q, a, row0 + own_row(tid, u), rows, a.qr, a.qh); };
      // in units that make scores exponents of 2
      if (WIDE) {
#pragma unroll 1
        for (int m = 0; m < 2; m++)
          own_wide(base + m * ROW_TILE, a, tid, a.dh, a.slog2, [&](int u) {
            const float* x = at_q(u);
            return x ? x + m * a.dh : x;
          });
      } else {
        load_own<false>(base, a, tid, a.slog2, at_q, at_q);
      }
      fence_async_smem();
      signal(&sh.rows_full);
    }
    const int part = warp >> 2, w = warp & 3, row = w * 32 + lane, r = row0 + row;
    const uint32_t at = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int e = min(r, rows - 1) / a.tq, i = r - e * a.tq, head = kvh * a.grp + e;
    const int lim = r < rows ? min(kend, row_limit(a, i, len)) : 0;
    const int full = __reduce_min_sync(0xffffffffu, lim);
    float x[32], y[32], m1 = -CUDART_INF_F, m2 = -CUDART_INF_F, l1 = 0.0f, l2 = 0.0f;
    float al1 = 0.0f, al2 = 0.0f;  // what the sums before the last tile get
#pragma unroll
    for (int c = 0; c < 32; c++) x[c] = y[c] = 0.0f;
    int turn = 0;
    bool ok = true;
    for (int t = 0; t < nt; t++) {
      // the tile's visible keys come from the loading warps, its scores from the MMAs
      if (!(ok = blk.done(&sh.full[t % STG], (t / STG) & 1) && blk.done(&sh.s_full, t & 1))) break;
      tc_fence_after();
      float s1[32], s2[32];
      tmem_ld(at + part * 32, s1);
      tmem_ld(at + 64 + part * 32, s2);
      tmem_landed(s1);
      tmem_landed(s2);
      const int j0 = kbeg + t * COLS + part * 32;
      const uint32_t seen = sh.seen[t % STG][part];
      tc_fence_before();
      signal(&sh.s_free);
      const bool edge = j0 + 32 > full || seen != 0xffffffffu;
      if (edge) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (j0 + c >= lim || !(seen >> c & 1)) s1[c] = s2[c] = -CUDART_INF_F;
      }
      float2 top = make_float2(max_of(s1), max_of(s2)), other;
      if (!(ok = blk.exchange(turn, w, part, row, top, other))) break;
      top.x = fmaxf(m1, fmaxf(top.x, other.x));
      top.y = fmaxf(m2, fmaxf(top.y, other.y));
      // a row without a visible key so far keeps its maximum at -inf
      const float u1 = top.x == -CUDART_INF_F ? 0.0f : top.x, u2 = top.y == -CUDART_INF_F ? 0.0f : top.y;
      const float f1 = ex2(m1 - u1), f2 = ex2(m2 - u2);
      m1 = top.x;
      m2 = top.y;
      l1 = l1 * f1 + exp_sum(s1, u1);
      l2 = l2 * f2 + exp_sum(s2, u2);
      if (t > 0) {
        if (!(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        add_tmem(at + FWD_O + part * 32, x, al1);
        add_tmem(at + FWD_O + 64 + part * 32, y, al2);
      }
      al1 = f1;
      al2 = f2;
      store_planes(at + FWD_P + part * PART, s1);
      store_planes(at + FWD_P + MAP + part * PART, s2);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.p_full);
    }
    if (ok && nt > 0 && (ok = blk.done(&sh.o_full, (nt - 1) & 1))) {
      tc_fence_after();
      add_tmem(at + FWD_O + part * 32, x, al1);
      add_tmem(at + FWD_O + 64 + part * 32, y, al2);
    }
    float2 other;
    if (ok && blk.exchange(turn, w, part, row, make_float2(l1, l2), other)) {
      // the same order of the two sums in both threads
      const float L1 = part ? other.x + l1 : l1 + other.x, L2 = part ? other.y + l2 : l2 + other.y;
      float* patch = reinterpret_cast<float*>(base) + warp * 1024;  // q is no longer read
      if (a.nsplit > 1) {
        const long long to = (static_cast<long long>(blockIdx.y) * nbh + bh) * rows + r;
        float* q = r < rows ? a.part + to * (2 * PART_W) + col0 + part * 32 : nullptr;
        store_rows(patch, x, 32, true, q);
        store_rows(patch, y, 32, true, q ? q + PART_W : nullptr);
        if (part == 0 && col0 == 0 && r < rows) *reinterpret_cast<float4*>(a.stat + to * 4) = make_float4(m1, L1, m2, L2);
      } else {
        // a map without a key has no part in the products but what 0 * inf or 0 * NaN left
        const bool one = L1 != 0.0f, two = L2 != 0.0f;
        const float i1 = inverse(L1), i2 = inverse(L2), lam = two ? __ldg(a.lam + head) : 0.0f;
#pragma unroll
        for (int c = 0; c < 32; c++) {
          y[c] = two ? y[c] * i2 : 0.0f;
          x[c] = (one ? x[c] * i1 : 0.0f) - lam * y[c];
        }
        const int in = 2 * a.dh - col0 - part * 32;
        store_rows(patch, x, in, p.st16,
                   r < rows ? static_cast<float*>(a.o) + b * a.ob + head * a.oh + i * a.orow + col0 + part * 32 : nullptr);
        if (a.o2)
          store_rows(patch, y, in, p.st16_2,
                     r < rows ? static_cast<float*>(a.o2) +
                                    ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) + col0 + part * 32
                              : nullptr);
        if (a.lse && part == 0 && col0 == 0 && r < rows) {
          float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
          s[0] = log_sum(m1, L1);
          s[a.tq] = log_sum(m2, L2);
        }
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < WARP_MMA) {
      const int t0 = tid - MATH_WARPS * 32;
      if (nt > 0) load_keys<WIDE>(blk, stages, STG, a, b, kvh, kbeg, kend, nt, t0, col0);
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, COLS, false), id_o = idesc_bf16(ROWS, 64, true);
      const uint64_t dq = desc_k(smem_u32(base)), dk = desc_k(smem_u32(stages));
      const uint64_t dv = desc_mn(smem_u32(stages) + V_AT, 0);
      const int ksteps = (a.dh + 15) / 16;
      bool ok = blk.done(&sh.rows_full, 0);
      auto scores = [&](int t) {
        const int st = t % STG;
        if (!blk.done(&sh.full[st], (t / STG) & 1) || (t > 0 && !blk.done(&sh.s_free, (t - 1) & 1))) return false;
        tc_fence_after();
        const uint64_t k = dk + st * (STAGE / 16);
#pragma unroll
        for (int m = 0; m < 2; m++)
          products<WIDE ? 4 : 2>(ksteps, [&](int pa, int pb, int ks, bool acc) {
            mma_ss(tmem + m * 64, dq + (pa * ROW_PLANE + m * Q_HALF + ks * 32) / 16,
                   k + (pb * COL_PLANE + m * K_HALF + ks * 32) / 16, id_s, acc, lead);
          });
        commit(&sh.s_full, lead);
        return true;
      };
      auto values = [&](int t) {
        const int st = t % STG;
        if (!blk.done(&sh.p_full, t & 1)) return false;
        tc_fence_after();
        const uint64_t v = dv + st * (STAGE / 16);
#pragma unroll
        for (int m = 0; m < 2; m++)
          products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
            mma_ts(tmem + FWD_O + m * 64, tmem + FWD_P + m * MAP + plane_at(pa, ks),
                   v + (pb * COL_PLANE + ks * 2048) / 16, id_o, acc, lead);
          });
        commit(&sh.empty[st], lead);
        commit(&sh.o_full, lead);
        return true;
      };
      ok = ok && scores(0);
      for (int t = 0; ok && t < nt; t++) {
        // the next scores run under this tile's exponentials, if a stage holds their tile
        if (STG > 1 && t + 1 < nt && !(ok = scores(t + 1))) break;
        if (!(ok = values(t))) break;
        if (STG == 1 && t + 1 < nt) ok = scores(t + 1);
      }
      if (!ok) {  // no MMA may write tensor memory after it is released
        commit(&sh.drain, lead);
        settle(&sh.drain, 0);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// A row's 32 values of the map's exponent to the map: s <- 2^(s - u).
__device__ __forceinline__ void exp_row(float (&s)[32], float u) {
  const f32x2 uu = pair(-u, -u);
#pragma unroll
  for (int i = 0; i < 16; i++) {
    float &x = s[2 * i], &y = s[2 * i + 1];
    unpair(add2(pair(x, y), uu), x, y);
    x = ex2(x);
    y = ex2(y);
  }
}
// sum of x y over a row's 32 values
__device__ __forceinline__ float dot_row(const float (&x)[32], const float (&y)[32]) {
  f32x2 t[2] = {0ull, 0ull};
#pragma unroll
  for (int i = 0; i < 16; i++) t[i & 1] = fma2(pair(x[2 * i], x[2 * i + 1]), pair(y[2 * i], y[2 * i + 1]), t[i & 1]);
  float u, v;
  unpair(add2(t[0], t[1]), u, v);
  return u + v;
}
// s <- s (dp - d)
__device__ __forceinline__ void times_rest(float (&s)[32], const float (&dp)[32], float d) {
  const f32x2 dd = pair(-d, -d);
#pragma unroll
  for (int i = 0; i < 16; i++)
    unpair(mul2(pair(s[2 * i], s[2 * i + 1]), add2(pair(dp[2 * i], dp[2 * i + 1]), dd)), s[2 * i], s[2 * i + 1]);
}

// dq of 128 packed rows, D_1 and D_2 of each (for the keys' kernel), and the row
// sums of P_2 dP over those of P_2.
__global__ void __launch_bounds__(THREADS, 1) f32_bwd_q_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* stages = base + 2 * ROW_TILE;
  Shared& sh = *reinterpret_cast<Shared*>(stages + BWD_STAGES * 2 * COL_TILE);
  Block blk{sh, p.dev_error};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.grp * a.tq, nbh = a.n * a.hkv, ntile = (rows + ROWS - 1) / ROWS;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;
  const int bh = static_cast<int>(blockIdx.x) % nbh, b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int row0 = tile * ROWS, len = key_len(a, b);
  const int last = min(rows, row0 + ROWS) - 1;
  const int imax = last / a.tq != row0 / a.tq ? a.tq - 1 : last % a.tq;
  const int kend = row_limit(a, imax, len);
  const int nt = (kend + COLS - 1) / COLS;
  setup(sh, warp);
  const uint32_t tmem = sh.tmem;

  if (warp < MATH_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    if (nt > 0) {
      const long long h0 = static_cast<long long>(kvh) * a.grp;
      const float* q = static_cast<const float*>(a.q) + b * a.qb + h0 * a.qh;
      const float* g = static_cast<const float*>(a.dout) + b * a.gb + h0 * a.gh;
      load_own<true>(base, a, tid, a.slog2, [&](int u) { return packed(q, a, row0 + own_row(tid, u), rows, a.qr, a.qh); },
                     [&](int u) { return packed(g, a, row0 + own_row(tid, u), rows, a.gr, a.gh); });
      fence_async_smem();
      signal(&sh.rows_full);
      // D_1 = do . (o + lam o2) and D_2 = do . o2; rows that see one tile of keys
      // sum P dP instead (dS of a lone key comes out as 0).
      if (nt > 1) {
        const float* o = static_cast<const float*>(a.fo) + b * a.ob + h0 * a.oh;
        const float* o2 = static_cast<const float*>(a.fo2) + (static_cast<long long>(b) * a.tq * a.h + h0) * (2 * a.dh);
        auto load = [&](float (&x)[8], const float* q, auto vec) { load8<false, decltype(vec)::value>(x, q, tid & 7, a.dh); };
        auto sums = [&](int u, auto vec) {
          const int r = row0 + own_row(tid, u), e = r < rows ? r / a.tq : -1, i = r - e * a.tq;
          float x[8], y[8], z[8], d = 0.0f, d2 = 0.0f;
          load(x, e < 0 ? nullptr : g + e * a.gh + i * a.gr, vec);
          load(y, e < 0 ? nullptr : o + e * a.oh + i * a.orow, vec);
          load(z, e < 0 ? nullptr : o2 + (static_cast<long long>(i) * a.h + e) * (2 * a.dh), vec);
#pragma unroll
          for (int k = 0; k < 8; k++) {
            d += x[k] * y[k];
            d2 += x[k] * z[k];
          }
#pragma unroll
          for (int k = 1; k < 8; k <<= 1) {
            d += __shfl_xor_sync(0xffffffffu, d, k);
            d2 += __shfl_xor_sync(0xffffffffu, d2, k);
          }
          if ((tid & 7) == 0 && e >= 0) sh.d[r - row0] = make_float2(d + __ldg(a.lam + kvh * a.grp + e) * d2, d2);
        };
        if (p.ld16) {
#pragma unroll
          for (int u = 0; u < OWN; u++) sums(u, std::true_type());
        } else {
#pragma unroll 1
          for (int u = 0; u < OWN; u++) sums(u, std::false_type());
        }
        signal(&sh.d_full);
      }
    }
    const int part = warp >> 2, w = warp & 3, row = w * 32 + lane, r = row0 + row;
    const uint32_t at = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int e = min(r, rows - 1) / a.tq, i = r - e * a.tq, head = kvh * a.grp + e;
    const int lim = r < rows ? min(kend, row_limit(a, i, len)) : 0;
    const int full = __reduce_min_sync(0xffffffffu, lim);
    float ls1 = CUDART_INF_F, ls2 = CUDART_INF_F, d1 = 0.0f, d2 = 0.0f, dl = 0.0f, pl = 0.0f;
    int turn = 0;
    bool ok = true;
    if (r < rows) {
      const float* s = a.flse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
      ls1 = s[0];
      ls2 = s[a.tq];
    }
    if (nt > 1) {
      ok = blk.done(&sh.d_full, 0);
      if (ok && r < rows) {
        d1 = sh.d[row].x;
        d2 = sh.d[row].y;
      }
    }
    float dq[32];
#pragma unroll
    for (int c = 0; c < 32; c++) dq[c] = 0.0f;
    for (int t = 0; ok && t < nt; t++) {
      const int st = t % BWD_STAGES;
      if (!(ok = blk.done(&sh.full[st], (t / BWD_STAGES) & 1) && blk.done(&sh.s_full, t & 1))) break;
      tc_fence_after();
      float s1[32], s2[32], dp[32];
      tmem_ld(at + part * 32, s1);
      tmem_ld(at + 64 + part * 32, s2);
      tmem_ld(at + 128 + part * 32, dp);
      tmem_landed(s1);
      tmem_landed(s2);
      tmem_landed(dp);
      const int j0 = t * COLS + part * 32;
      const uint32_t seen = sh.seen[st][part];
      tc_fence_before();
      signal(&sh.s_free);
      if (j0 + 32 > full || seen != 0xffffffffu) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (j0 + c >= lim || !(seen >> c & 1)) s1[c] = s2[c] = -CUDART_INF_F;
      }
      exp_row(s1, ls1);
      pl += exp_sum(s2, ls2);
      const float dlt = dot_row(s2, dp);
      dl += dlt;
      if (nt == 1) {
        float2 other;
        d1 = dot_row(s1, dp);
        if (!(ok = blk.exchange(turn, w, part, row, make_float2(d1, dlt), other))) break;
        d1 += other.x;
        d2 = dlt + other.y;
      }
      times_rest(s1, dp, d1);
      times_rest(s2, dp, d2);
      if (t > 0) {
        if (!(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        add_tmem(at + Q_O + part * 32, dq, 1.0f);
      }
      store_planes(at + Q_P + part * PART, s1);
      store_planes(at + Q_P + MAP + part * PART, s2);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.p_full);
    }
    if (ok && nt > 0 && (ok = blk.done(&sh.o_full, (nt - 1) & 1))) {
      tc_fence_after();
      add_tmem(at + Q_O + part * 32, dq, 1.0f);
    }
    float2 other;
    if (ok && blk.exchange(turn, w, part, row, make_float2(dl, pl), other)) {
      if (part == 0 && r < rows) {
        // over the map's own sum: what the log-sum's rounding does to a whole row cancels
        const float whole = pl + other.y;
        float* s = a.dsum + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
        s[0] = d1;
        s[a.tq] = d2;
        a.dlrow[static_cast<long long>(head) * a.n * a.tq + static_cast<long long>(b) * a.tq + i] =
            whole == 0.0f ? 0.0f : (dl + other.x) / whole;
      }
      const float f = part ? -a.scale * __ldg(a.lam + head) : a.scale;
#pragma unroll
      for (int c = 0; c < 32; c++) dq[c] *= f;
      store_rows(reinterpret_cast<float*>(base) + warp * 1024, dq, a.dh, p.st16,
                 r < rows ? static_cast<float*>(a.dq) + b * a.dqb + head * a.dqh + i * a.dqr + part * a.dh : nullptr);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < WARP_MMA) {
      if (nt > 0) load_keys<false>(blk, stages, BWD_STAGES, a, b, kvh, 0, kend, nt, tid - MATH_WARPS * 32, 0);
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, COLS, false), id_o = idesc_bf16(ROWS, 32, true);
      const uint64_t dq = desc_k(smem_u32(base)), dg = desc_k(smem_u32(base) + ROW_TILE);
      const uint64_t dk = desc_k(smem_u32(stages)), dv = desc_k(smem_u32(stages) + COL_TILE);
      const uint64_t dkn = desc_mn(smem_u32(stages), 0);
      const int ksteps = (a.dh + 15) / 16, vsteps = (2 * a.dh + 15) / 16;
      bool ok = blk.done(&sh.rows_full, 0);
      for (int t = 0; ok && t <= nt; t++) {
        if (t < nt) {
          const int st = t % BWD_STAGES;
          if (!(ok = blk.done(&sh.full[st], (t / BWD_STAGES) & 1) && (t == 0 || blk.done(&sh.s_free, (t - 1) & 1)))) break;
          tc_fence_after();
          const uint64_t k = dk + st * (2 * COL_TILE / 16), v = dv + st * (2 * COL_TILE / 16);
#pragma unroll
          for (int m = 0; m < 2; m++)
            products<2>(ksteps, [&](int pa, int pb, int ks, bool acc) {
              mma_ss(tmem + m * 64, dq + (pa * ROW_PLANE + m * 64 + ks * 32) / 16,
                     k + (pb * COL_PLANE + m * 64 + ks * 32) / 16, id_s, acc, lead);
            });
          products<4>(vsteps, [&](int pa, int pb, int ks, bool acc) {
            mma_ss(tmem + 128, dg + (pa * ROW_PLANE + ks * 32) / 16, v + (pb * COL_PLANE + ks * 32) / 16, id_s, acc, lead);
          });
          commit(&sh.s_full, lead);
        }
        if (t > 0) {
          const int st = (t - 1) % BWD_STAGES;
          if (!(ok = blk.done(&sh.p_full, (t - 1) & 1))) break;
          tc_fence_after();
          const uint64_t k = dkn + st * (2 * COL_TILE / 16);
#pragma unroll
          for (int m = 0; m < 2; m++)
            products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
              mma_ts(tmem + Q_O + m * 32, tmem + Q_P + m * MAP + plane_at(pa, ks),
                     k + (pb * COL_PLANE + m * 64 + ks * 2048) / 16, id_o, acc, lead);
            });
          commit(&sh.empty[st], lead);
          commit(&sh.o_full, lead);
        }
      }
      if (!ok) {
        commit(&sh.drain, lead);
        settle(&sh.drain, 0);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// dk and dv of 128 keys, over the queries of the group's heads: the transposed
// maps come from k q^T and v do^T, so that keys stay in the rows.
__global__ void __launch_bounds__(THREADS, 1) f32_bwd_kv_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* stages = base + 2 * ROW_TILE;
  Shared& sh = *reinterpret_cast<Shared*>(stages + BWD_STAGES * 2 * COL_TILE);
  Block blk{sh, p.dev_error};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nbh = a.n * a.hkv, nkt = (a.tk + ROWS - 1) / ROWS;
  const bool work = static_cast<int>(blockIdx.x) < nkt * nbh;  // else a block for dlam only
  const int kt = work ? static_cast<int>(blockIdx.x) / nbh : 0;  // the earliest keys, which most queries see, first
  const int bh = static_cast<int>(blockIdx.x) % nbh, b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int key0 = kt * ROWS, len = key_len(a, b);
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;
  // queries before `qbeg` see none of these keys
  int qbeg = 0;
  if (!work || key0 >= len) {
    qbeg = a.tq;
  } else if (a.causal == RNN_CAUSAL_START) {
    qbeg = min(a.tq, key0);
  } else if (a.causal == RNN_CAUSAL_END) {
    qbeg = min(a.tq, max(0, key0 - (len - a.tq)));
  }
  const int per = (a.tq - qbeg + COLS - 1) / COLS, nt = per * a.grp;
  setup(sh, warp);
  const uint32_t tmem = sh.tmem;

  if (warp < MATH_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    if (nt > 0) {
      auto row = [&](const void* q, long long sb, long long sr, long long sh_, int r) -> const float* {
        const int j = key0 + r;
        return j < len && (!mask || mask[j]) ? static_cast<const float*>(q) + b * sb + kvh * sh_ + j * sr : nullptr;
      };
      load_own<true>(base, a, tid, a.slog2, [&](int u) { return row(a.k, a.kb, a.kr, a.kh, own_row(tid, u)); },
                     [&](int u) { return row(a.v, a.vb, a.vr, a.vh, own_row(tid, u)); });
      fence_async_smem();
      signal(&sh.rows_full);
    }
    const int part = warp >> 2, w = warp & 3, row = w * 32 + lane, key = key0 + row;
    const uint32_t at = tmem + (static_cast<uint32_t>(w * 32) << 16);
    // what a query has to see for this key to count
    const int need = key < len && (!mask || mask[key]) ? key : 0x7fffffff;
    const int most = __reduce_max_sync(0xffffffffu, need);
    float dv[32], dk[32];
#pragma unroll
    for (int c = 0; c < 32; c++) dv[c] = dk[c] = 0.0f;
    bool ok = true;
    for (int t = 0; t < nt; t++) {
      const int st = t % BWD_STAGES;
      if (!(ok = blk.done(&sh.full[st], (t / BWD_STAGES) & 1) && blk.done(&sh.s_full, t & 1))) break;
      tc_fence_after();
      float s1[32], s2[32];
      tmem_ld(at + KV_S + part * 32, s1);
      tmem_ld(at + MAP + KV_S + part * 32, s2);
      tmem_landed(s1);
      tmem_landed(s2);
      const float* stat = &sh.stat[st][0][part * 32];
      const float lam = __ldg(a.lam + kvh * a.grp + t / per);
      const f32x2 ll = pair(-lam, -lam);  // s2 is -lam P_2
      if (most >= sh.least[st][part]) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (need >= __float_as_int(stat[4 * COLS + c])) s1[c] = s2[c] = -CUDART_INF_F;
      }
      float z[32];  // P_1 - lam P_2
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const f32x2 l1 = *reinterpret_cast<const f32x2*>(stat + c), l2 = *reinterpret_cast<const f32x2*>(stat + COLS + c);
        float x, y, u, v;
        unpair(add2(pair(s1[c], s1[c + 1]), l1), x, y);
        unpair(add2(pair(s2[c], s2[c + 1]), l2), u, v);
        const f32x2 p1 = pair(ex2(x), ex2(y)), p2 = mul2(pair(ex2(u), ex2(v)), ll);
        unpair(p1, s1[c], s1[c + 1]);
        unpair(p2, s2[c], s2[c + 1]);
        unpair(add2(p1, p2), z[c], z[c + 1]);
      }
      if (t > 0) {
        if (!(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        add_tmem(at + KV_O + part * 32, dv, 1.0f);
        add_tmem(at + KV_O + 64 + part * 32, dk, 1.0f);
      }
      store_planes(at + MAP + part * PART, z);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.p_full);
      if (!(ok = blk.done(&sh.dp_full, t & 1))) break;
      tc_fence_after();
      tmem_ld(at + 2 * MAP + KV_S + part * 32, z);
      tmem_landed(z);
      // s1 = dS_1, s2 = dS_2
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        const f32x2 d1 = *reinterpret_cast<const f32x2*>(stat + 2 * COLS + c);
        const f32x2 d2 = *reinterpret_cast<const f32x2*>(stat + 3 * COLS + c);
        const f32x2 dp = pair(z[c], z[c + 1]);
        unpair(mul2(pair(s1[c], s1[c + 1]), add2(dp, d1)), s1[c], s1[c + 1]);
        unpair(mul2(pair(s2[c], s2[c + 1]), add2(dp, d2)), s2[c], s2[c + 1]);
      }
      store_planes(at + 2 * MAP + part * PART, s1);
      store_planes(at + 3 * MAP + part * PART, s2);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.ds_full);
    }
    if (ok && nt > 0 && (ok = blk.done(&sh.o_full, (nt - 1) & 1))) {
      tc_fence_after();
      add_tmem(at + KV_O + part * 32, dv, 1.0f);
      add_tmem(at + KV_O + 64 + part * 32, dk, 1.0f);
    }
    if (ok && work) {
      float* patch = reinterpret_cast<float*>(base) + warp * 1024;
      const bool hidden = need == 0x7fffffff;  // 0, whatever a query's NaN made of 0 times it
#pragma unroll
      for (int c = 0; c < 32; c++) dv[c] = hidden ? 0.0f : dv[c];
      store_rows(patch, dv, 2 * a.dh - part * 32, p.st16,
                 key < a.tk ? static_cast<float*>(a.dv) + b * a.dvb + kvh * a.dvh + key * a.dvr + part * 32 : nullptr);
#pragma unroll
      for (int c = 0; c < 32; c++) dk[c] = hidden ? 0.0f : dk[c] * a.scale;
      store_rows(patch, dk, a.dh, p.st16,
                 key < a.tk ? static_cast<float*>(a.dk) + b * a.dkb + kvh * a.dkh + key * a.dkr + part * a.dh : nullptr);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < WARP_MMA) {
      const int t0 = tid - MATH_WARPS * 32;
      const float* qp = static_cast<const float*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
      const float* gp = static_cast<const float*>(a.dout) + b * a.gb + static_cast<long long>(kvh) * a.grp * a.gh;
      for (int t = 0; t < nt; t++) {
        const int st = t % BWD_STAGES, e = t / per, i0 = qbeg + (t - e * per) * COLS;
        const int i = i0 + t0;
        const bool in = t0 < COLS && i < a.tq;
        const long long from = (static_cast<long long>(b) * a.h + kvh * a.grp + e) * 2 * a.tq + i;
        const float l1 = in ? a.flse[from] : CUDART_INF_F, l2 = in ? a.flse[from + a.tq] : CUDART_INF_F;
        const float d1 = in ? a.dsum[from] : 0.0f, d2 = in ? a.dsum[from + a.tq] : 0.0f;
        const int lim = in ? row_limit(a, i, len) : 0;
        if (!load_step(stages + st * (2 * COL_TILE), a, t0,
                       [&](int r) { return i0 + r < a.tq ? qp + e * a.qh + (i0 + r) * a.qr : nullptr; },
                       [&](int r) { return i0 + r < a.tq ? gp + e * a.gh + (i0 + r) * a.gr : nullptr; },
                       [&] { return t < BWD_STAGES || blk.done(&sh.empty[st], (t / BWD_STAGES - 1) & 1); }))
          break;
        if (t0 < COLS) {
          sh.stat[st][0][t0] = -l1;
          sh.stat[st][1][t0] = -l2;
          sh.stat[st][2][t0] = -d1;
          sh.stat[st][3][t0] = -d2;
          sh.stat[st][4][t0] = __int_as_float(lim);
          const int least = __reduce_min_sync(0xffffffffu, lim);
          if ((t0 & 31) == 0) sh.least[st][t0 >> 5] = least;
        }
        fence_async_smem();
        signal(&sh.full[st]);
      }
      // dlam: block `head` sums that head's rows in a fixed order
      if (warp == MATH_WARPS && static_cast<int>(blockIdx.x) < a.h && a.tq > 0) {
        const long long cnt = static_cast<long long>(a.n) * a.tq;
        const float* x = a.dlrow + blockIdx.x * cnt;
        double sum = 0.0;
#pragma unroll 8
        for (long long i = lane; i < cnt; i += 32) sum += x[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) a.dlam[blockIdx.x] -= static_cast<float>(sum);
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, COLS, false), id_v = idesc_bf16(ROWS, 64, true);
      const uint32_t id_k = idesc_bf16(ROWS, 32, true);
      const uint64_t dk = desc_k(smem_u32(base)), dv = desc_k(smem_u32(base) + ROW_TILE);
      const uint64_t dq = desc_k(smem_u32(stages)), dg = desc_k(smem_u32(stages) + COL_TILE);
      const uint64_t dqn = desc_mn(smem_u32(stages), 0), dgn = desc_mn(smem_u32(stages) + COL_TILE, 0);
      const int ksteps = (a.dh + 15) / 16, vsteps = (2 * a.dh + 15) / 16;
      bool ok = blk.done(&sh.rows_full, 0);
      auto scores = [&](int t) {
        const int st = t % BWD_STAGES;
        if (!blk.done(&sh.full[st], (t / BWD_STAGES) & 1)) return false;
        tc_fence_after();
        const uint32_t off = st * (2 * COL_TILE / 16);
#pragma unroll
        for (int m = 0; m < 2; m++)
          products<2>(ksteps, [&](int pa, int pb, int ks, bool acc) {
            mma_ss(tmem + m * MAP + KV_S, dk + (pa * ROW_PLANE + m * 64 + ks * 32) / 16,
                   dq + off + (pb * COL_PLANE + m * 64 + ks * 32) / 16, id_s, acc, lead);
          });
        commit(&sh.s_full, lead);
        return true;
      };
      ok = ok && scores(0);
      for (int t = 0; ok && t < nt; t++) {
        const uint32_t off = (t % BWD_STAGES) * (2 * COL_TILE / 16);
        // dP overwrites dS_1 of the step before
        if (t > 0 && !(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        products<4>(vsteps, [&](int pa, int pb, int ks, bool acc) {
          mma_ss(tmem + 2 * MAP + KV_S, dv + (pa * ROW_PLANE + ks * 32) / 16, dg + off + (pb * COL_PLANE + ks * 32) / 16,
                 id_s, acc, lead);
        });
        commit(&sh.dp_full, lead);
        if (!(ok = blk.done(&sh.p_full, t & 1))) break;
        tc_fence_after();
        products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
          mma_ts(tmem + KV_O, tmem + MAP + plane_at(pa, ks), dgn + off + (pb * COL_PLANE + ks * 2048) / 16, id_v, acc, lead);
        });
        // The next scores take the places of the last ones, which are in
        // registers, and of the planes that dv reads: MMAs of one accumulator
        // shape (128 x 64) execute in the order of issue.
        if (t + 1 < nt && !(ok = scores(t + 1))) break;
        if (!(ok = blk.done(&sh.ds_full, t & 1))) break;
        tc_fence_after();
#pragma unroll
        for (int m = 0; m < 2; m++)
          products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
            mma_ts(tmem + KV_O + 64 + m * 32, tmem + (2 + m) * MAP + plane_at(pa, ks),
                   dqn + off + (pb * COL_PLANE + m * 64 + ks * 2048) / 16, id_k, acc, lead);
          });
        commit(&sh.empty[t % BWD_STAGES], lead);
        commit(&sh.o_full, lead);
      }
      if (!ok) {
        commit(&sh.drain, lead);
        settle(&sh.drain, 0);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// Halves of more than 32 columns: the rows of a block with all they meet do not
// fit an SM, so each block takes one map (blockIdx.y): dq_m of 128 packed query
// rows, or dk_m of 128 keys,
//   S_m = X x^T,  dP = Y y^T,  dS_m = P_m (dP - D_m),  dX = dS_m x,
// with X, x = q_m, k_m and Y, y = do, v for queries and the other way round for
// keys.  dP is formed twice that way, and dv has a kernel of its own.  Y, the
// larger of the rows, stays in tensor memory (columns 288 to 480).  Measured: 4 x 1024
// x 1024, 4 heads of 64: 190 us forward and 357 backward, 300 and 1076 on the
// kernels of mma.sync.
constexpr uint32_t G_DP = 64, G_P = 128, G_O = G_P + MAP, G_Y = G_O + 64, Y_PLANE = 64;

template <bool KEYS>
__global__ void __launch_bounds__(THREADS, 1) f32_grad_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  constexpr uint32_t STAGE = 3 * COL_TILE;
  uint8_t* stage = base + ROW_TILE;
  Shared& sh = *reinterpret_cast<Shared*>(stage + BWD_STAGES * STAGE);
  Block blk{sh, p.dev_error};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31, m = blockIdx.y;
  const int rows = KEYS ? a.tk : a.grp * a.tq, nbh = a.n * a.hkv, ntile = (rows + ROWS - 1) / ROWS;
  const bool work = static_cast<int>(blockIdx.x) < ntile * nbh;  // else a block for dlam only
  // what takes longest first: late queries, early keys
  const int order = work ? static_cast<int>(blockIdx.x) / nbh : 0, tile = KEYS ? order : ntile - 1 - order;
  const int bh = static_cast<int>(blockIdx.x) % nbh, b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int row0 = tile * ROWS, len = key_len(a, b);
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;
  const long long h0 = static_cast<long long>(kvh) * a.grp;
  const float* qp = static_cast<const float*>(a.q) + b * a.qb + h0 * a.qh;
  const float* gp = static_cast<const float*>(a.dout) + b * a.gb + h0 * a.gh;
  const float* kp = static_cast<const float*>(a.k) + b * a.kb + kvh * a.kh;
  const float* vp = static_cast<const float*>(a.v) + b * a.vb + kvh * a.vh;
  int kend = 0, qbeg = 0, per = 0, nt;
  if (KEYS) {
    // queries before `qbeg` see none of these keys
    if (!work || row0 >= len) {
      qbeg = a.tq;
    } else if (a.causal == RNN_CAUSAL_START) {
      qbeg = min(a.tq, row0);
    } else if (a.causal == RNN_CAUSAL_END) {
      qbeg = min(a.tq, max(0, row0 - (len - a.tq)));
    }
    per = (a.tq - qbeg + COLS - 1) / COLS;
    nt = per * a.grp;
  } else {
    const int last = min(rows, row0 + ROWS) - 1;
    const int imax = last / a.tq != row0 / a.tq ? a.tq - 1 : last % a.tq;
    kend = row_limit(a, imax, len);
    nt = (kend + COLS - 1) / COLS;
  }
  setup(sh, warp);
  const uint32_t tmem = sh.tmem;

  if (warp < MATH_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    // the place of packed query row r in a tensor of the queries
    auto query = [&](const float* x, long long sr, long long sh_, int r) { return packed(x, a, r, rows, sr, sh_); };
    auto key_row = [&](const float* x, long long sr, int j) {
      return j < len && (!mask || mask[j]) ? x + j * sr : static_cast<const float*>(nullptr);
    };
    if (nt > 0) {
      own_wide(base, a, tid, a.dh, a.slog2, [&](int u) {
        const int r = row0 + own_row(tid, u);
        const float* x = KEYS ? key_row(kp, a.kr, r) : query(qp, a.qr, a.qh, r);
        return x ? x + m * a.dh : x;
      });
      // a thread's 64 columns of its row of Y
      const int c0 = (warp >> 2) * 64, r = row0 + (warp & 3) * 32 + lane, in = 2 * a.dh - c0;
      const float* y = KEYS ? key_row(vp, a.vr, r) : query(gp, a.gr, a.gh, r);
      const uint32_t to = tmem + (static_cast<uint32_t>((warp & 3) * 32) << 16) + G_Y + (warp >> 2) * 32;
#pragma unroll 1
      for (int g = 0; g < 4; g++) {
        float x[16];
        if (a.vec) {
#pragma unroll
          for (int c = 0; c < 16; c += 4) {
            float4 v = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
            if (y && g * 16 + c < in) v = __ldg(reinterpret_cast<const float4*>(y + c0 + g * 16 + c));
            x[c] = v.x, x[c + 1] = v.y, x[c + 2] = v.z, x[c + 3] = v.w;
          }
        } else {
#pragma unroll
          for (int c = 0; c < 16; c++) x[c] = y && g * 16 + c < in ? __ldg(y + c0 + g * 16 + c) : 0.0f;
        }
        uint32_t z[3][8];
#pragma unroll
        for (int k = 0; k < 8; k++) split3(x[2 * k], x[2 * k + 1], z[0][k], z[1][k], z[2][k]);
#pragma unroll
        for (int q = 0; q < 3; q++) tmem_st(to + q * Y_PLANE + g * 8, z[q]);
      }
      tmem_wait_st();
      tc_fence_before();
      fence_async_smem();
      signal(&sh.rows_full);
      // D_m, from do . o and do . o2; rows that see one tile of keys sum P dP
      if (!KEYS && nt > 1) {
        const float* o = static_cast<const float*>(a.fo) + b * a.ob + h0 * a.oh;
        const float* o2 = static_cast<const float*>(a.fo2) + (static_cast<long long>(b) * a.tq * a.h + h0) * (2 * a.dh);
        auto sums = [&](int u, auto vec) {
          constexpr bool VEC = decltype(vec)::value;
          const int r = row0 + own_row(tid, u), c = tid & 7, e = min(r, rows - 1) / a.tq;
          const float lam = m ? 1.0f : __ldg(a.lam + h0 + e);
          const float *pg = query(gp, a.gr, a.gh, r), *po = query(o, a.orow, a.oh, r);
          const float* py = query(o2, static_cast<long long>(a.h) * 2 * a.dh, 2 * a.dh, r);
          float d = 0.0f;
#pragma unroll
          for (int i = 0; i < 2; i++) {
            const int in = 2 * a.dh - i * 64;
            float x[8], y[8], z[8];
            load8_wide<VEC>(x, pg ? pg + i * 64 : pg, c, in);
            load8_wide<VEC>(y, m || !po ? nullptr : po + i * 64, c, in);
            load8_wide<VEC>(z, py ? py + i * 64 : py, c, in);
#pragma unroll
            for (int k = 0; k < 8; k++) d += x[k] * (y[k] + lam * z[k]);
          }
#pragma unroll
          for (int k = 1; k < 8; k <<= 1) d += __shfl_xor_sync(0xffffffffu, d, k);
          if (c == 0) sh.d[r - row0].x = d;
        };
        if (p.ld16) {
#pragma unroll 2
          for (int u = 0; u < OWN; u++) sums(u, std::true_type());
        } else {
#pragma unroll 1
          for (int u = 0; u < OWN; u++) sums(u, std::false_type());
        }
        signal(&sh.d_full);
      }
    }
    const int part = warp >> 2, w = warp & 3, row = w * 32 + lane, r = row0 + row;
    const uint32_t at = tmem + (static_cast<uint32_t>(w * 32) << 16);
    // query rows
    const int e = KEYS ? 0 : min(r, rows - 1) / a.tq, i = r - e * a.tq, head = static_cast<int>(h0) + e;
    const int lim = !KEYS && r < rows ? min(kend, row_limit(a, i, len)) : 0;
    const int full = __reduce_min_sync(0xffffffffu, lim);
    float ls = CUDART_INF_F, d = 0.0f, dl = 0.0f, pl = 0.0f;
    if (!KEYS && r < rows) ls = a.flse[((static_cast<long long>(b) * a.h + head) * 2 + m) * a.tq + i];
    // keys: what a query has to see for this key to count
    const int need = KEYS && r < len && (!mask || mask[r]) ? r : 0x7fffffff;
    const int most = __reduce_max_sync(0xffffffffu, need);
    int turn = 0;
    bool ok = true;
    if (!KEYS && nt > 1) {
      ok = blk.done(&sh.d_full, 0);
      if (ok && r < rows) d = sh.d[row].x;
    }
    float acc[32];
#pragma unroll
    for (int c = 0; c < 32; c++) acc[c] = 0.0f;
    for (int t = 0; ok && t < nt; t++) {
      const int st = t % BWD_STAGES;
      if (!(ok = blk.done(&sh.full[st], (t / BWD_STAGES) & 1) && blk.done(&sh.s_full, t & 1))) break;
      tc_fence_after();
      float s[32], dp[32];
      tmem_ld(at + part * 32, s);
      tmem_landed(s);
      tc_fence_before();
      signal(&sh.s_free);
      const float* stat = &sh.stat[st][0][part * 32];
      if (KEYS) {
        if (most >= sh.least[st][part]) {
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (need >= __float_as_int(stat[4 * COLS + c])) s[c] = -CUDART_INF_F;
        }
        const float f = m ? -__ldg(a.lam + h0 + t / per) : 1.0f;
        const f32x2 ff = pair(f, f);
#pragma unroll
        for (int c = 0; c < 32; c += 2) {
          float u, v;
          unpair(add2(pair(s[c], s[c + 1]), *reinterpret_cast<const f32x2*>(stat + c)), u, v);
          unpair(mul2(pair(ex2(u), ex2(v)), ff), s[c], s[c + 1]);
        }
      } else {
        const int j0 = t * COLS + part * 32;
        const uint32_t seen = sh.seen[st][part];
        if (j0 + 32 > full || seen != 0xffffffffu) {
#pragma unroll
          for (int c = 0; c < 32; c++)
            if (j0 + c >= lim || !(seen >> c & 1)) s[c] = -CUDART_INF_F;
        }
        pl += exp_sum(s, ls);
      }
      if (!(ok = blk.done(&sh.dp_full, t & 1))) break;
      tc_fence_after();
      tmem_ld(at + G_DP + part * 32, dp);
      tmem_landed(dp);
      if (KEYS) {
#pragma unroll
        for (int c = 0; c < 32; c += 2)
          unpair(mul2(pair(s[c], s[c + 1]),
                      add2(pair(dp[c], dp[c + 1]), *reinterpret_cast<const f32x2*>(stat + 2 * COLS + c))),
                 s[c], s[c + 1]);
      } else {
        const float now = dot_row(s, dp);
        dl += now;
        if (nt == 1) {
          float2 other;
          if (!(ok = blk.exchange(turn, w, part, row, make_float2(now, 0.0f), other))) break;
          d = now + other.x;
        }
        times_rest(s, dp, d);
      }
      if (t > 0) {
        if (!(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        add_tmem(at + G_O + part * 32, acc, 1.0f);
      }
      store_planes(at + G_P + part * PART, s);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.p_full);
    }
    if (ok && nt > 0 && (ok = blk.done(&sh.o_full, (nt - 1) & 1))) {
      tc_fence_after();
      add_tmem(at + G_O + part * 32, acc, 1.0f);
    }
    float* patch = reinterpret_cast<float*>(base) + warp * 1024;  // the rows are no longer read
    const int in = a.dh - part * 32;
    if (KEYS) {
#pragma unroll
      for (int c = 0; c < 32; c++) acc[c] = need == 0x7fffffff ? 0.0f : acc[c] * a.scale;  // a hidden key's is 0
      if (ok && work)
        store_rows(patch, acc, in, p.st16,
                   r < rows ? static_cast<float*>(a.dk) + b * a.dkb + kvh * a.dkh + r * a.dkr + m * a.dh + part * 32
                            : nullptr);
    } else {
      float2 other;
      if (ok && blk.exchange(turn, w, part, row, make_float2(dl, pl), other)) {
        if (part == 0 && r < rows) {
          // over the map's own sum: what the log-sum's rounding does to a whole row cancels
          const float whole = pl + other.y;
          a.dsum[((static_cast<long long>(b) * a.h + head) * 2 + m) * a.tq + i] = d;
          if (m)
            a.dlrow[static_cast<long long>(head) * a.n * a.tq + static_cast<long long>(b) * a.tq + i] =
                whole == 0.0f ? 0.0f : (dl + other.x) / whole;
        }
        const float f = m ? -a.scale * __ldg(a.lam + head) : a.scale;
#pragma unroll
        for (int c = 0; c < 32; c++) acc[c] *= f;
        store_rows(patch, acc, in, p.st16,
                   r < rows ? static_cast<float*>(a.dq) + b * a.dqb + head * a.dqh + i * a.dqr + m * a.dh + part * 32
                            : nullptr);
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < WARP_MMA) {
      const int t0 = tid - MATH_WARPS * 32;
      for (int t = 0; t < nt; t++) {
        const int st = t % BWD_STAGES;
        auto ready = [&] { return t < BWD_STAGES || blk.done(&sh.empty[st], (t / BWD_STAGES - 1) & 1); };
        auto in = [&](int i) { return i == 0 ? a.dh : 2 * a.dh - (i - 1) * 64; };
        if (KEYS) {
          const int e = t / per, i0 = qbeg + (t - e * per) * COLS, i = i0 + t0;
          const bool on = t0 < COLS && i < a.tq;
          const long long from = ((static_cast<long long>(b) * a.h + h0 + e) * 2 + m) * a.tq + i;
          const float l = on ? a.flse[from] : CUDART_INF_F, d = on ? a.dsum[from] : 0.0f;
          const int lim = on ? row_limit(a, i, len) : 0;
          if (!step_wide<3>(stage + st * STAGE, a, t0,
                            [&](int k, int r) -> const float* {
                              if (i0 + r >= a.tq) return nullptr;
                              return k == 0 ? qp + e * a.qh + (i0 + r) * a.qr + m * a.dh
                                            : gp + e * a.gh + (i0 + r) * a.gr + (k - 1) * 64;
                            },
                            in, ready))
            break;
          if (t0 < COLS) {
            sh.stat[st][0][t0] = -l;
            sh.stat[st][2][t0] = -d;
            sh.stat[st][4][t0] = __int_as_float(lim);
            const int least = __reduce_min_sync(0xffffffffu, lim);
            if ((t0 & 31) == 0) sh.least[st][t0 >> 5] = least;
          }
        } else {
          const int j0 = t * COLS;
          auto on = [&](int r) { return j0 + r < kend && (!mask || mask[j0 + r]); };
          const uint32_t bits = __ballot_sync(0xffffffffu, t0 < COLS && on(t0));
          if (!step_wide<3>(stage + st * STAGE, a, t0,
                            [&](int k, int r) -> const float* {
                              if (!on(r)) return nullptr;
                              return k == 0 ? kp + (j0 + r) * a.kr + m * a.dh : vp + (j0 + r) * a.vr + (k - 1) * 64;
                            },
                            in, ready))
            break;
          if (t0 < COLS && (t0 & 31) == 0) sh.seen[st][t0 >> 5] = bits;
        }
        fence_async_smem();
        signal(&sh.full[st]);
      }
      // dlam: block `head` sums that head's rows in a fixed order
      if (KEYS && m == 0 && warp == MATH_WARPS && static_cast<int>(blockIdx.x) < a.h && a.tq > 0) {
        const long long cnt = static_cast<long long>(a.n) * a.tq;
        const float* x = a.dlrow + blockIdx.x * cnt;
        double sum = 0.0;
#pragma unroll 8
        for (long long i = lane; i < cnt; i += 32) sum += x[i];
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) a.dlam[blockIdx.x] -= static_cast<float>(sum);
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, COLS, false), id_o = idesc_bf16(ROWS, 64, true);
      const uint64_t dx = desc_k(smem_u32(base));
      const uint64_t cx = desc_k(smem_u32(stage)), cy = desc_k(smem_u32(stage) + COL_TILE);
      const uint64_t cn = desc_mn(smem_u32(stage), 0);
      const int ksteps = (a.dh + 15) / 16, vsteps = (2 * a.dh + 15) / 16;
      bool ok = blk.done(&sh.rows_full, 0);
      auto scores = [&](int t) {
        const int st = t % BWD_STAGES;
        if (!blk.done(&sh.full[st], (t / BWD_STAGES) & 1) || (t > 0 && !blk.done(&sh.s_free, (t - 1) & 1))) return false;
        tc_fence_after();
        products<4>(ksteps, [&](int pa, int pb, int ks, bool acc) {
          mma_ss(tmem, dx + (pa * ROW_PLANE + ks * 32) / 16, cx + st * (STAGE / 16) + (pb * COL_PLANE + ks * 32) / 16, id_s,
                 acc, lead);
        });
        commit(&sh.s_full, lead);
        return true;
      };
      ok = ok && scores(0);
      for (int t = 0; ok && t < nt; t++) {
        const int st = t % BWD_STAGES;
        const uint32_t off = st * (STAGE / 16);
        products<8>(vsteps, [&](int pa, int pb, int ks, bool acc) {
          mma_ts(tmem + G_DP, tmem + G_Y + pa * Y_PLANE + ks * 8,
                 cy + off + ((ks >> 2) * COL_TILE + pb * COL_PLANE + (ks & 3) * 32) / 16, id_s, acc, lead);
        });
        commit(&sh.dp_full, lead);
        if (t + 1 < nt && !(ok = scores(t + 1))) break;  // under this step's arithmetic
        if (!(ok = blk.done(&sh.p_full, t & 1))) break;
        tc_fence_after();
        products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
          mma_ts(tmem + G_O, tmem + G_P + plane_at(pa, ks), cn + off + (pb * COL_PLANE + ks * 2048) / 16, id_o, acc,
                 lead);
        });
        commit(&sh.empty[st], lead);
        commit(&sh.o_full, lead);
      }
      if (!ok) {
        commit(&sh.drain, lead);
        settle(&sh.drain, 0);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// dv of 128 keys for halves of more than 32 columns: (P_1 - lam P_2)^T do.
__global__ void __launch_bounds__(THREADS, 1) f32_dv_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  uint8_t* stage = base + 2 * ROW_TILE;
  Shared& sh = *reinterpret_cast<Shared*>(stage + 4 * COL_TILE);
  Block blk{sh, p.dev_error};
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nbh = a.n * a.hkv, key0 = static_cast<int>(blockIdx.x) / nbh * ROWS;
  const int bh = static_cast<int>(blockIdx.x) % nbh, b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int len = key_len(a, b);
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;
  int qbeg = 0;
  if (key0 >= len) {
    qbeg = a.tq;
  } else if (a.causal == RNN_CAUSAL_START) {
    qbeg = min(a.tq, key0);
  } else if (a.causal == RNN_CAUSAL_END) {
    qbeg = min(a.tq, max(0, key0 - (len - a.tq)));
  }
  const int per = (a.tq - qbeg + COLS - 1) / COLS, nt = per * a.grp;
  setup(sh, warp);
  const uint32_t tmem = sh.tmem;

  if (warp < MATH_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 168;");
    if (nt > 0) {
      const float* kp = static_cast<const float*>(a.k) + b * a.kb + kvh * a.kh;
#pragma unroll 1
      for (int m = 0; m < 2; m++)
        own_wide(base + m * ROW_TILE, a, tid, a.dh, a.slog2, [&](int u) {
          const int j = key0 + own_row(tid, u);
          return j < len && (!mask || mask[j]) ? kp + j * a.kr + m * a.dh : static_cast<const float*>(nullptr);
        });
      fence_async_smem();
      signal(&sh.rows_full);
    }
    const int part = warp >> 2, w = warp & 3, row = w * 32 + lane, key = key0 + row;
    const uint32_t at = tmem + (static_cast<uint32_t>(w * 32) << 16);
    const int need = key < len && (!mask || mask[key]) ? key : 0x7fffffff;
    const int most = __reduce_max_sync(0xffffffffu, need);
    float v0[32], v1[32];
#pragma unroll
    for (int c = 0; c < 32; c++) v0[c] = v1[c] = 0.0f;
    bool ok = true;
    for (int t = 0; t < nt; t++) {
      if (!(ok = blk.done(&sh.full[0], t & 1) && blk.done(&sh.s_full, t & 1))) break;
      tc_fence_after();
      float s1[32], s2[32];
      tmem_ld(at + part * 32, s1);
      tmem_ld(at + 64 + part * 32, s2);
      tmem_landed(s1);
      tmem_landed(s2);
      const float* stat = &sh.stat[0][0][part * 32];
      if (most >= sh.least[0][part]) {
#pragma unroll
        for (int c = 0; c < 32; c++)
          if (need >= __float_as_int(stat[4 * COLS + c])) s1[c] = s2[c] = -CUDART_INF_F;
      }
      const float lam = __ldg(a.lam + kvh * a.grp + t / per);
      const f32x2 ll = pair(-lam, -lam);
#pragma unroll
      for (int c = 0; c < 32; c += 2) {
        float x, y, u, v;
        unpair(add2(pair(s1[c], s1[c + 1]), *reinterpret_cast<const f32x2*>(stat + c)), x, y);
        unpair(add2(pair(s2[c], s2[c + 1]), *reinterpret_cast<const f32x2*>(stat + COLS + c)), u, v);
        unpair(fma2(pair(ex2(u), ex2(v)), ll, pair(ex2(x), ex2(y))), s1[c], s1[c + 1]);
      }
      if (t > 0) {
        if (!(ok = blk.done(&sh.o_full, (t - 1) & 1))) break;
        tc_fence_after();
        add_tmem(at + G_O + part * 32, v0, 1.0f);
        add_tmem(at + G_O + 64 + part * 32, v1, 1.0f);
      }
      store_planes(at + G_P + part * PART, s1);
      tmem_wait_st();
      tc_fence_before();
      signal(&sh.p_full);
    }
    if (ok && nt > 0 && (ok = blk.done(&sh.o_full, (nt - 1) & 1))) {
      tc_fence_after();
      add_tmem(at + G_O + part * 32, v0, 1.0f);
      add_tmem(at + G_O + 64 + part * 32, v1, 1.0f);
    }
    if (ok) {
      float* patch = reinterpret_cast<float*>(base) + warp * 1024;
      float* to = key < a.tk ? static_cast<float*>(a.dv) + b * a.dvb + kvh * a.dvh + key * a.dvr + part * 32 : nullptr;
#pragma unroll
      for (int c = 0; c < 32; c++) {  // a hidden key's is 0, whatever a query's NaN made of 0 times it
        v0[c] = need == 0x7fffffff ? 0.0f : v0[c];
        v1[c] = need == 0x7fffffff ? 0.0f : v1[c];
      }
      store_rows(patch, v0, 2 * a.dh - part * 32, p.st16, to);
      store_rows(patch, v1, 2 * a.dh - 64 - part * 32, p.st16, to ? to + 64 : nullptr);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 88;");
    if (warp < WARP_MMA) {
      const int t0 = tid - MATH_WARPS * 32;
      const float* qp = static_cast<const float*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
      const float* gp = static_cast<const float*>(a.dout) + b * a.gb + static_cast<long long>(kvh) * a.grp * a.gh;
      for (int t = 0; t < nt; t++) {
        const int e = t / per, i0 = qbeg + (t - e * per) * COLS, i = i0 + t0;
        const bool on = t0 < COLS && i < a.tq;
        const long long from = (static_cast<long long>(b) * a.h + kvh * a.grp + e) * 2 * a.tq + i;
        const float l1 = on ? a.flse[from] : CUDART_INF_F, l2 = on ? a.flse[from + a.tq] : CUDART_INF_F;
        const int lim = on ? row_limit(a, i, len) : 0;
        if (!step_wide<2>(stage, a, t0,
                          [&](int k, int r) { return i0 + r < a.tq ? qp + e * a.qh + (i0 + r) * a.qr + k * a.dh : nullptr; },
                          [&](int) { return a.dh; }, [&] { return t == 0 || blk.done(&sh.empty[0], (t - 1) & 1); }))
          break;
        step_wide<2>(stage + 2 * COL_TILE, a, t0,
                     [&](int k, int r) { return i0 + r < a.tq ? gp + e * a.gh + (i0 + r) * a.gr + k * 64 : nullptr; },
                     [&](int k) { return 2 * a.dh - k * 64; }, [] { return true; });
        if (t0 < COLS) {
          sh.stat[0][0][t0] = -l1;
          sh.stat[0][1][t0] = -l2;
          sh.stat[0][4][t0] = __int_as_float(lim);
          const int least = __reduce_min_sync(0xffffffffu, lim);
          if ((t0 & 31) == 0) sh.least[0][t0 >> 5] = least;
        }
        fence_async_smem();
        signal(&sh.full[0]);
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, COLS, false), id_o = idesc_bf16(ROWS, 64, true);
      const uint64_t dk = desc_k(smem_u32(base)), cq = desc_k(smem_u32(stage));
      const uint64_t cg = desc_mn(smem_u32(stage) + 2 * COL_TILE, 0);
      const int ksteps = (a.dh + 15) / 16;
      bool ok = blk.done(&sh.rows_full, 0);
      for (int t = 0; ok && t < nt; t++) {
        if (!(ok = blk.done(&sh.full[0], t & 1))) break;
        tc_fence_after();
#pragma unroll
        for (int m = 0; m < 2; m++)
          products<4>(ksteps, [&](int pa, int pb, int ks, bool acc) {
            mma_ss(tmem + m * 64, dk + (m * ROW_TILE + pa * ROW_PLANE + ks * 32) / 16,
                   cq + (m * COL_TILE + pb * COL_PLANE + ks * 32) / 16, id_s, acc, lead);
          });
        commit(&sh.s_full, lead);
        if (!(ok = blk.done(&sh.p_full, t & 1))) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; c++)
          products<COLS / 16>(COLS / 16, [&](int pa, int pb, int ks, bool acc) {
            mma_ts(tmem + G_O + c * 64, tmem + G_P + plane_at(pa, ks),
                   cg + (c * COL_TILE + pb * COL_PLANE + ks * 2048) / 16, id_o, acc, lead);
          });
        commit(&sh.empty[0], lead);
        commit(&sh.o_full, lead);
      }
      if (!ok) {
        commit(&sh.drain, lead);
        settle(&sh.drain, 0);
      }
      __syncwarp();
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

}  // namespace

// A block starts and ends in about 9 us beside 2 us a tile, more than the
// kernels of mma.sync, which keep what is small (forward and backward of 128 x 64
// x 64, 4 heads of 32: 28 and 70 us against 38 and 83 here).  Here are faster: 64
// x 128 x 128: 25 and 62 against 47 and 116; 32 x 256 x 256: 34 and 91 against 82
// and 206; 64 x 64 x 256: 35 and 91 against 43 and 103; 1 x 64 x 5000: 25 and 283
// against 26 and 524.  Halves of more than 32 columns the same (4 x 64 x 64: no
// difference; 64 x 100 x 100 of 48: 66 and 168 against 80 and 315), but forward,
// where the scores are formed twice, only if rows fill a block or keys are many
// (128 x 64 x 128, 4 heads of 64: 120 against 88, backward 276 against 353).
bool f32_tc_ok(const Args& a, bool backward) {
  const long long rows = static_cast<long long>(a.grp) * a.tq;
  if (rows < 64 || rows * a.tk < 64 * 128) return false;
  return backward || a.dh <= 32 || rows >= 96 || a.tk >= 256;
}

int f32_tc_fwd(rnn_ctx* ctx, const Args& a) {
  Params p;
  p.a = a;
  p.dev_error = ctx->dev_error;
  auto m4 = [](long long s) { return s % 4 == 0; };
  p.st16 = reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && m4(a.ob) && m4(a.orow) && m4(a.oh);
  p.st16_2 = reinterpret_cast<uintptr_t>(a.o2) % 16 == 0 && a.dh % 2 == 0;
  const long long rows = static_cast<long long>(a.grp) * a.tq, nbh = static_cast<long long>(a.n) * a.hkv;
  const long long blocks = (rows + ROWS - 1) / ROWS * nbh;
  RNN_REQUIRE(blocks < (1ll << 31), "diffattn: too many rows");
  const bool wide = a.dh > 32;
  const int tiles = (a.tk + COLS - 1) / COLS;
  const long long parts = std::max(1ll, std::min<long long>(ctx->num_sms / (wide ? 2 * blocks : blocks), tiles / 4));
  p.a.split_keys = static_cast<int>((tiles + parts - 1) / parts) * COLS;
  p.a.nsplit = (a.tk + p.a.split_keys - 1) / p.a.split_keys;
  if (p.a.nsplit > 1) {
    const size_t all = static_cast<size_t>(p.a.nsplit) * nbh * rows;
    const size_t width = wide ? 256 : 128;
    RNN_TRY(ensure_ws(ctx, all * (width + 4) * sizeof(float)));
    p.a.part = static_cast<float*>(ctx->ws);
    p.a.stat = p.a.part + all * width;
  }
  static std::atomic<unsigned long long> optin[2];
  const auto kernel = wide ? f32_fwd_kernel<true> : f32_fwd_kernel<false>;
  const size_t smem = wide ? FWD_WIDE_SMEM : FWD_SMEM;
  RNN_TRY(tc::ensure_smem_optin(kernel, optin[wide], ctx->device, static_cast<int>(smem)));
  kernel<<<dim3(static_cast<unsigned>(blocks), p.a.nsplit, wide ? 2 : 1), THREADS, smem, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  if (p.a.nsplit == 1) return RNN_OK;
  return wide ? join_rows_f32_wide(ctx, p.a) : join_rows_f32(ctx, p.a);
}

int f32_tc_bwd(rnn_ctx* ctx, const Args& a) {
  Params p;
  p.a = a;
  p.dev_error = ctx->dev_error;
  auto a16 = [](const void* q) { return reinterpret_cast<uintptr_t>(q) % 16 == 0; };
  auto m4 = [](std::initializer_list<long long> s) {
    for (long long x : s)
      if (x % 4) return false;
    return true;
  };
  p.st16 = a.dh % 4 == 0 && a16(a.dq) && a16(a.dk) && a16(a.dv) &&
           m4({a.dqb, a.dqr, a.dqh, a.dkb, a.dkr, a.dkh, a.dvb, a.dvr, a.dvh});
  p.ld16 = a.vec && a16(a.fo) && a16(a.fo2) && m4({a.ob, a.orow, a.oh});
  const long long rows = static_cast<long long>(a.grp) * a.tq, nbh = static_cast<long long>(a.n) * a.hkv;
  const long long qblocks = (rows + ROWS - 1) / ROWS * nbh;
  const long long kblocks = std::max<long long>((a.tk + ROWS - 1ll) / ROWS * nbh, a.h);
  RNN_REQUIRE(qblocks < (1ll << 31) && kblocks < (1ll << 31), "diffattn: too many rows");
  if (a.dh > 32) {
    static std::atomic<unsigned long long> optin_r{0}, optin_c{0}, optin_v{0};
    RNN_TRY(tc::ensure_smem_optin(f32_grad_kernel<false>, optin_r, ctx->device, static_cast<int>(GRAD_SMEM)));
    RNN_TRY(tc::ensure_smem_optin(f32_grad_kernel<true>, optin_c, ctx->device, static_cast<int>(GRAD_SMEM)));
    RNN_TRY(tc::ensure_smem_optin(f32_dv_kernel, optin_v, ctx->device, static_cast<int>(DV_SMEM)));
    f32_grad_kernel<false><<<dim3(static_cast<unsigned>(qblocks), 2), THREADS, GRAD_SMEM, ctx->stream>>>(p);
    RNN_CHECK_LAUNCH();
    f32_grad_kernel<true><<<dim3(static_cast<unsigned>(kblocks), 2), THREADS, GRAD_SMEM, ctx->stream>>>(p);
    RNN_CHECK_LAUNCH();
    f32_dv_kernel<<<static_cast<unsigned>((a.tk + ROWS - 1ll) / ROWS * nbh), THREADS, DV_SMEM, ctx->stream>>>(p);
    RNN_CHECK_LAUNCH();
    return RNN_OK;
  }
  static std::atomic<unsigned long long> optin_q{0}, optin_k{0};
  RNN_TRY(tc::ensure_smem_optin(f32_bwd_q_kernel, optin_q, ctx->device, static_cast<int>(BWD_SMEM)));
  RNN_TRY(tc::ensure_smem_optin(f32_bwd_kv_kernel, optin_k, ctx->device, static_cast<int>(BWD_SMEM)));
  f32_bwd_q_kernel<<<static_cast<unsigned>(qblocks), THREADS, BWD_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  f32_bwd_kv_kernel<<<static_cast<unsigned>(kblocks), THREADS, BWD_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  return RNN_OK;
}

}  // namespace diff
}  // namespace rnn
