// Differential attention backward on tcgen05: bf16, halves of 8 .. 64 columns
// (multiples of 8).  Two kernels, as in diffattn.cu: one owns 128 queries of a
// head (dq, D_1, D_2), one owns 128 keys of a key head
// (dk, dv).  Both form scores and dP = do v^T anew, 64 columns at a time, and
// both are bound by the exponentials and the tensor cores about alike.
//
// 16 warps turn scores into dS, 16 columns of a row at a time: with the saved
// log-sums no thread needs another's values, so a row is shared by four of
// them.  Warp 16 copies tiles (and in the keys' kernel brings the queries'
// log-sums and D).  Two warps issue MMAs, 17 the products with dS and dP, 18 the
// scores: an issuing warp stalls while the tensor cores are busy, and one warp
// alone left them idle at each of its waits.  Measured: 1 x 8192 x 8192, 8 heads
// of 64: 1176 us for both, 0.59 PF/s of the formula's products (about 2000 clocks
// a tile in the queries' kernel, 2220 in the keys').  Warp 19 clears what is masked or
// lies beyond a sequence's length (queries' kernel) or sums dlam (keys' kernel).
#include <algorithm>
#include <cmath>

#include "diffattn_tc.cuh"

namespace rnn {
namespace diff {
namespace {

constexpr int THREADS = 640, SOFT = 16, WARP_COPY = 16, WARP_MMA = 17, WARP_SCORE = 18, WARP_AUX = 19;
constexpr int ROWS = 128, COLS = 64;               // a block's rows, a tile's columns
constexpr uint32_t BIG = ROWS * 128, SMALL = COLS * 128;  // 64-column parts of a 128- and a 64-row tile, bytes

struct alignas(64) Params {
  CUtensorMap q, k, v, g;  // g: dout
  Args a;
  int* dev_error;
  int st16;  // 16-byte stores of the gradients are aligned
};

__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 512;" ::: "memory"); }

// 16 values times f to bf16 at p, the first n of them (a multiple of 8).
__device__ __forceinline__ void store16(__nv_bfloat16* p, const float (&v)[16], float f, bool on, int n, bool st16) {
  uint32_t w[8];
#pragma unroll
  for (int k = 0; k < 8; k++) w[k] = on ? pack2(v[2 * k] * f, v[2 * k + 1] * f) : 0u;
  if (st16) {
    if (n > 0) *reinterpret_cast<uint4*>(p) = make_uint4(w[0], w[1], w[2], w[3]);
    if (n > 8) *reinterpret_cast<uint4*>(p + 8) = make_uint4(w[4], w[5], w[6], w[7]);
  } else {
#pragma unroll
    for (int k = 0; k < 16; k++)
      if (k < n) p[k] = __ushort_as_bfloat16(static_cast<unsigned short>(w[k >> 1] >> (16 * (k & 1))));
  }
}

// ------------------------------------------------------------------ queries
//
// Two teams of 8 warps take the tiles alternately.  Tensor memory: dq_1 | dq_2
// at [0, 128); S_1 | S_2 | dP of even tiles at [128, 320), of odd ones at
// [320, 512).  dS takes the place of dP (16 keys of both maps: the 16 columns
// that their dP had), so that the scores of a team's next tile are formed as
// soon as this one's are in registers; only its dP waits for the products with
// dS, behind the exponentials.

constexpr int Q_STAGES = 4;
constexpr uint32_t Q_STAGE = 4 * SMALL;  // k halves, v parts
struct QShared {
  uint64_t q_full, kv_full[Q_STAGES], kv_empty[Q_STAGES], landed[Q_STAGES], s_full[2], s_free[2], d_full[2], p_full[2];
  uint64_t o_full[2], decided, drain[2];
  uint32_t tmem;
  int abort_flag;
  int again;             // whether the tiles are gone over once more
  uint2 seen[Q_STAGES];  // masked calls: which keys of a tile count
  float4 part[4][ROWS];
};
constexpr size_t Q_SMEM = 1024 + 4 * BIG + Q_STAGES * Q_STAGE + sizeof(QShared);

template <bool MASK>
__global__ void __launch_bounds__(THREADS, 1) tc_bwd_q_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const uint32_t sq = smem_u32(base), sg = sq + 2 * BIG, skv = sg + 2 * BIG;
  QShared& sh = *reinterpret_cast<QShared*>(base + 4 * BIG + Q_STAGES * Q_STAGE);
  volatile int* abort_flag = &sh.abort_flag;
  int* dev_error = p.dev_error;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ntile = (a.tq + ROWS - 1) / ROWS, nbh = a.n * a.h;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;  // longest causal rows first
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.h, head = bh - b * a.h, kvh = head / a.grp;
  const int i0 = tile * ROWS;
  const int len = key_len(a, b);
  const int kend = row_limit(a, min(i0 + ROWS, a.tq) - 1, len);
  const int nt = (kend + COLS - 1) / COLS;
  // tiles from clear0 on have hidden keys and values to be cleared, as in the forward pass
  const uint8_t* mask = MASK ? a.kmask + b * a.kmb : nullptr;
  const int clear0 = MASK ? 0 : nt > 0 && nt * COLS > len && len < a.tk ? nt - 1 : nt;
  // Step t is tile t, or t - nt the second time over the tiles.  Phase of a step's arrival for the clearing
  // warp: the stage's uses so far, which without a mask are the last tile's alone.
  auto clears = [&](int t) {
    return MASK ? static_cast<uint32_t>(t / Q_STAGES) & 1u : t >= nt && nt % Q_STAGES == 0 ? 1u : 0u;
  };
  auto cleared = [&](int t) { return (t < nt ? t : t - nt) >= clear0; };
  const int wide = 2 * a.dh > 64 ? 2 : 1, ksteps = (a.dh + 15) / 16, dsteps = a.dh / 8;

  if (tid == 0) {
    mbar_init(&sh.q_full, 1);
    for (int i = 0; i < Q_STAGES; i++) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
      mbar_init(&sh.landed[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.s_full[i], 1);
      mbar_init(&sh.s_free[i], 8);
      mbar_init(&sh.d_full[i], 1);
      mbar_init(&sh.p_full[i], 8);
    }
    mbar_init(&sh.o_full[0], 1);
    mbar_init(&sh.o_full[1], 1);
    mbar_init(&sh.decided, SOFT);
    mbar_init(&sh.drain[0], 1);
    mbar_init(&sh.drain[1], 1);
    sh.abort_flag = sh.again = 0;
    fence_barrier_init();
  }
  if (warp == WARP_MMA) {
    tmem_alloc(&sh.tmem, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = sh.tmem;
  // Whether to go over the tiles `pass` times and once more (a row of at most two tiles has its D from P dP).
  auto goes_on = [&](int pass) {
    if (pass == 0) return nt > 0;
    return pass == 1 && nt > 2 && wait(&sh.decided, 0, abort_flag, dev_error) &&
           *static_cast<volatile int*>(&sh.again) != 0;
  };

  // registers: 640 threads x 96 at launch = 512 x 104 + 128 x 64
  if (warp < SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int team = warp >> 3, half = (warp >> 2) & 1, w = warp & 3, row = w * 32 + lane, i = i0 + row;
    const int k4 = team * 2 + half;  // which of the row's four threads
    const uint32_t lanes = static_cast<uint32_t>(w * 32) << 16;
    const uint32_t ts = tmem + lanes + 128 + team * 192 + half * 32;
    const bool in = i < a.tq;
    const int lim = (in ? row_limit(a, i, len) : 0) - half * 32;
    const int full = __reduce_min_sync(0xffffffffu, lim);
    const float lam = __ldg(a.lam + head), c2 = a.slog2;
    const long long stat = (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
    const float ls1 = in ? a.flse[stat] : CUDART_INF_F, ls2 = in ? a.flse[stat + a.tq] : CUDART_INF_F;
    const f32x2 cc = pair(c2, c2), n1 = pair(-ls1, -ls1), n2 = pair(-ls2, -ls2);

    // both maps' entries of 16 columns from the scores
    auto maps = [&](uint32_t t, float (&x)[16], float (&y)[16], int visible, bool edge, uint32_t seen) {
      tmem_ld(t, x);
      tmem_ld(t + 64, y);
      tmem_landed(x);
      tmem_landed(y);
#pragma unroll
      for (int c = 0; c < 16; c += 2) {
        unpair(fma2(pair(x[c], x[c + 1]), cc, n1), x[c], x[c + 1]);
        unpair(fma2(pair(y[c], y[c + 1]), cc, n2), y[c], y[c + 1]);
        x[c] = ex2(x[c]);
        x[c + 1] = ex2(x[c + 1]);
        y[c] = ex2(y[c]);
        y[c + 1] = ex2(y[c + 1]);
      }
      if (__builtin_expect(edge, 0)) {
#pragma unroll
        for (int c = 0; c < 16; c++)
          if (c >= visible || !(seen >> c & 1)) x[c] = y[c] = 0.0f;
      }
    };
    // which of this thread's 32 keys of step t count
    auto counts = [&](int t) { return !MASK ? 0xffffffffu : half ? sh.seen[t % Q_STAGES].y : sh.seen[t % Q_STAGES].x; };

    // D_1 and D_2: from o and o2 (too_far() on what their rounding does), or, where a
    // row sees at most two tiles, from P dP itself.
    float d1 = 0.0f, d2 = 0.0f;
    if (nt > 2) {
      if (in) {
        const int c0 = k4 * (a.dh / 2);
        const __nv_bfloat16* po = static_cast<const __nv_bfloat16*>(a.fo) + b * a.ob + head * a.oh + i * a.orow + c0;
        const __nv_bfloat16* py = static_cast<const __nv_bfloat16*>(a.fo2) +
                                  ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) + c0;
        const __nv_bfloat16* pg = static_cast<const __nv_bfloat16*>(a.dout) + b * a.gb + head * a.gh + i * a.gr + c0;
#pragma unroll 2
        for (int c = 0; c < a.dh / 2; c += 4) {
          const uint2 uo = *reinterpret_cast<const uint2*>(po + c), uy = *reinterpret_cast<const uint2*>(py + c),
                      ug = *reinterpret_cast<const uint2*>(pg + c);
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const uint32_t wo = e ? uo.y : uo.x, wy = e ? uy.y : uy.x, wg = e ? ug.y : ug.x;
#pragma unroll
            for (int f = 0; f < 2; f++) {
              // a bf16 is the high half of the f32 it stands for
              const float o = __uint_as_float(f ? wo & 0xffff0000u : wo << 16);
              const float y = __uint_as_float(f ? wy & 0xffff0000u : wy << 16);
              const float g = __uint_as_float(f ? wg & 0xffff0000u : wg << 16);
              d2 += g * y;
              d1 += g * (o + lam * y);
            }
          }
        }
      }
    } else if (team < nt) {
      warp_wait(&sh.kv_full[team], 0, abort_flag, dev_error);
      warp_wait(&sh.s_full[team], 0, abort_flag, dev_error);
      warp_wait(&sh.d_full[team], 0, abort_flag, dev_error);
      tc_fence_after();
#pragma unroll 1
      for (int c = 0; c < 32; c += 16) {
        float x[16], y[16], dp[16];
        maps(ts + c, x, y, lim - team * COLS - c, true, counts(team) >> c);
        tmem_ld(ts + 128 + c, dp);
        tmem_landed(dp);
#pragma unroll
        for (int e = 0; e < 16; e++) {
          d1 += x[e] * dp[e];
          d2 += y[e] * dp[e];
        }
      }
    }
    // a row's sum of its four threads' shares
    auto row_sum = [&](float4 mine) {
      sh.part[k4][row] = mine;
      soft_sync();
      float4 s = sh.part[0][row];
#pragma unroll
      for (int k = 1; k < 4; k++) {
        const float4 x = sh.part[k][row];
        s.x += x.x, s.y += x.y, s.z += x.z, s.w += x.w;
      }
      soft_sync();
      return s;
    };
    const float4 d = row_sum(make_float4(d1, d2, 0.0f, 0.0f));
    f32x2 e1 = pair(-d.x, -d.x), e2 = pair(-d.y, -d.y);  // -D_1, -D_2
    int pass = 0;
    for (;; pass++) {
      // sums of dS and of its squares
      f32x2 b1 = 0ull, b2 = 0ull, sq1 = 0ull, sq2 = 0ull;
      for (int t = pass * nt + ((team + pass * nt) & 1); t < (pass + 1) * nt; t += 2) {
        const uint32_t par = (t >> 1) & 1;
        const int j = t - pass * nt;
        bool edge = j * COLS + 32 > full;
        uint32_t seen = 0xffffffffu;
        if (MASK) {  // from the clearing warp
          if (!warp_wait(&sh.kv_full[t % Q_STAGES], (t / Q_STAGES) & 1, abort_flag, dev_error)) break;
          seen = counts(t);
          edge |= seen != 0xffffffffu;
        }
        float x[2][16], y[2][16];
        if (!warp_wait(&sh.s_full[team], par, abort_flag, dev_error)) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; c++) maps(ts + c * 16, x[c], y[c], lim - j * COLS - c * 16, edge, seen >> (c * 16));
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.s_free[team]);
        if (!warp_wait(&sh.d_full[team], par, abort_flag, dev_error)) break;
        tc_fence_after();
#pragma unroll
        for (int c = 0; c < 2; c++) {
          uint32_t u[8], v[8];
#pragma unroll
          for (int h = 0; h < 2; h++) {
            float dp[8];
            tmem_ld(ts + 128 + c * 16 + h * 8, dp);
            tmem_landed(dp);
#pragma unroll
            for (int e = 0; e < 4; e++) {
              const int k = h * 4 + e;
              const f32x2 g = pair(dp[2 * e], dp[2 * e + 1]);
              const f32x2 s1 = mul2(pair(x[c][2 * k], x[c][2 * k + 1]), add2(g, e1));
              const f32x2 s2 = mul2(pair(y[c][2 * k], y[c][2 * k + 1]), add2(g, e2));
              unpair(s1, x[c][2 * k], x[c][2 * k + 1]);
              u[k] = pack2(x[c][2 * k], x[c][2 * k + 1]);
              unpair(s2, y[c][2 * k], y[c][2 * k + 1]);
              v[k] = pack2(y[c][2 * k], y[c][2 * k + 1]);
            }
          }
          tmem_st(ts + 128 + c * 16, u);
          tmem_st(ts + 128 + c * 16 + 8, v);
        }
        tmem_wait_st();
        tc_fence_before();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.p_full[team]);
        // under the products with this tile's dS, which others wait for
#pragma unroll
        for (int c = 0; c < 2; c++)
#pragma unroll
          for (int k = 0; k < 16; k += 2) {
            const f32x2 s1 = pair(x[c][k], x[c][k + 1]), s2 = pair(y[c][k], y[c][k + 1]);
            b1 = add2(b1, s1);
            b2 = add2(b2, s2);
            sq1 = fma2(s1, s1, sq1);
            sq2 = fma2(s2, s2, sq2);
          }
      }
      if (pass > 0) break;
      auto both = [](f32x2 z) {
        float l, r;
        unpair(z, l, r);
        return l + r;
      };
      const float4 off = row_sum(make_float4(both(b1), both(b2), both(sq1), both(sq2)));
      // a map that has no key has no D either
      const float D1 = ls1 == CUDART_INF_F ? 0.0f : d.x + off.x, D2 = ls2 == CUDART_INF_F ? 0.0f : d.y + off.y;
      if (in && k4 == 0) {
        a.dsum[stat] = D1;
        a.dsum[stat + a.tq] = D2;
        a.dlrow[static_cast<long long>(head) * a.n * a.tq + static_cast<long long>(b) * a.tq + i] = D2;
      }
      if (nt <= 2) break;
      e1 = pair(-D1, -D1);
      e2 = pair(-D2, -D2);
      const bool far = in && (too_far(off.x, off.z) || too_far(off.y, off.w));
      if (__any_sync(0xffffffffu, far) && lane == 0) *static_cast<volatile int*>(&sh.again) = 1;
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.decided);
      if (!__all_sync(0xffffffffu, goes_on(1))) break;
    }

    bool ok = true;
    if (nt > 0) {
      ok = warp_wait(&sh.o_full[pass], 0, abort_flag, dev_error);
      tc_fence_after();
    }
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.dq) + b * a.dqb + head * a.dqh + i * a.dqr;
    if (ok) {
#pragma unroll
      for (int m = 0; m < 2; m++) {
        float x[16] = {};
        if (nt > 0) {
          tmem_ld(tmem + lanes + m * 64 + k4 * 16, x);
          tmem_landed(x);
        }
        if (in) store16(o + m * a.dh + k4 * 16, x, m ? -a.scale * lam : a.scale, nt > 0, a.dh - k4 * 16, p.st16);
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == WARP_COPY) {
      if (elect_one() && nt > 0) {
        mbar_arrive_expect_tx(&sh.q_full, (2 + wide) * BIG);
        for (int h = 0; h < 2; h++) tma_5d(sq + h * BIG, &p.q, 0, h, head, i0, b, &sh.q_full);
        for (int c = 0; c < wide; c++) tma_5d(sg + c * BIG, &p.g, c * 64, 0, head, i0, b, &sh.q_full);
        int t = 0;
        for (; t < nt || (t < 2 * nt && goes_on(1)); t++) {
          const int st = t % Q_STAGES, j = t < nt ? t : t - nt;
          if (t >= Q_STAGES && !wait(&sh.kv_empty[st], (t / Q_STAGES - 1) & 1, abort_flag, dev_error)) break;
          const uint32_t dst = skv + st * Q_STAGE;
          // a tile to be cleared lands for the clearing warp, which passes it on
          uint64_t* bar = cleared(t) ? &sh.landed[st] : &sh.kv_full[st];
          mbar_arrive_expect_tx(bar, (2 + wide) * SMALL);
          for (int h = 0; h < 2; h++) tma_5d(dst + h * SMALL, &p.k, 0, h, kvh, j * COLS, b, bar);
          for (int c = 0; c < wide; c++) tma_5d(dst + (2 + c) * SMALL, &p.v, c * 64, 0, kvh, j * COLS, b, bar);
        }
        // what was asked for lands before the block may end, aborting or not
        settle(&sh.q_full, 0);
        for (int i = max(0, t - Q_STAGES); i < t; i++)
          if (cleared(i)) settle(&sh.landed[i % Q_STAGES], clears(i));
          else settle(&sh.kv_full[i % Q_STAGES], (i / Q_STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == WARP_AUX) {
      Seen keys;
      for (int pass = 0; clear0 < nt && __all_sync(0xffffffffu, goes_on(pass)); pass++) {
        keys.load(mask, clear0 * COLS, len);
        for (int j = clear0; j < nt; j++) {
          const int t = pass * nt + j, st = t % Q_STAGES;
          const uint2 seen = keys.bits();
          if (j + 1 < nt) keys.load(mask, (j + 1) * COLS, len);
          if (!warp_wait(&sh.landed[st], clears(t), abort_flag, dev_error)) break;
          clear_hidden(base + 4 * BIG + st * Q_STAGE, seen, 2 + wide);
          if (lane == 0) sh.seen[st] = seen;
          fence_async_smem();
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.kv_full[st]);
        }
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, 64, false);
      auto done = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity, abort_flag, dev_error); };
      auto landed = [&](int j, int st) { return done(&sh.kv_full[st], (j / Q_STAGES) & 1); };
      bool ok = done(&sh.q_full, 0);
      int st = 0;
      if (warp == WARP_SCORE) {
        const uint64_t dq = desc_k(sq), dkv = desc_k(skv);
        for (int j = 0; ok && (j < nt || (j < 2 * nt && __all_sync(0xffffffffu, goes_on(1)))); j++) {
          // the team has the scores of step j - 2 in registers
          if (!(ok = landed(j, st) && (j < 2 || done(&sh.s_free[j & 1], ((j >> 1) - 1) & 1)))) break;
          tc_fence_after();
          const uint64_t kv = dkv + st * (Q_STAGE / 16);
          const uint32_t d = tmem + 128 + (j & 1) * 192;
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
              if (ks < ksteps)
                mma_ss(d + h * 64, dq + (h * BIG + ks * 32) / 16, kv + (h * SMALL + ks * 32) / 16, id_s, ks > 0, lead);
          commit(&sh.s_full[j & 1], lead);
          if (++st == Q_STAGES) st = 0;
        }
      } else {
        // One accumulator shape: MMAs of a thread then execute in the order of
        // issue, and the next dP may take the place of dS right after the
        // products with it.
        const uint32_t id_o = idesc_bf16(ROWS, 64, true);
        const uint64_t dg = desc_k(sg), dkv = desc_k(skv), dmn = desc_mn(skv, 0);
        auto slopes = [&](int j, int s1) {
          const uint64_t kv = dkv + s1 * (Q_STAGE / 16);
#pragma unroll
          for (int ks = 0; ks < 8; ks++)
            if (ks < dsteps)
              mma_ss(tmem + 256 + (j & 1) * 192, dg + ((ks >> 2) * BIG + (ks & 3) * 32) / 16,
                     kv + ((2 + (ks >> 2)) * SMALL + (ks & 3) * 32) / 16, id_s, ks > 0, lead);
          commit(&sh.d_full[j & 1], lead);
        };
        for (int pass = 0; ok && __all_sync(0xffffffffu, goes_on(pass)); pass++) {
          const int first = pass * nt, last = first + nt;
          for (int j = first; ok && j < min(first + 2, last); j++)
            if ((ok = landed(j, j % Q_STAGES))) {
              tc_fence_after();
              slopes(j, j % Q_STAGES);
            }
          st = first % Q_STAGES;
          int st2 = (first + 2) % Q_STAGES;
          for (int j = first; ok && j < last; j++) {
            if (!(ok = (j + 2 >= last || landed(j + 2, st2)) && done(&sh.p_full[j & 1], (j >> 1) & 1))) break;
            tc_fence_after();
            const uint64_t k = dmn + st * (Q_STAGE / 16);
            const uint32_t s = tmem + 256 + (j & 1) * 192;
#pragma unroll
            for (int m = 0; m < 2; m++)
#pragma unroll
              for (int ks = 0; ks < 4; ks++)
                mma_ts(tmem + m * 64, s + ks * 16 + m * 8, k + (m * SMALL + ks * 2048) / 16, id_o, j > first || ks > 0,
                       lead);
            // the scores of step j are long done: dS came of them
            commit(&sh.kv_empty[st], lead);
            if (j + 1 == last) commit(&sh.o_full[pass], lead);
            if (j + 2 < last) slopes(j + 2, st2);
            if (++st == Q_STAGES) st = 0;
            if (++st2 == Q_STAGES) st2 = 0;
          }
        }
      }
      if (!ok) {  // no MMA may write tensor memory after it is released
        uint64_t* drain = &sh.drain[warp == WARP_SCORE];
        commit(drain, lead);
        settle(drain, 0);
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// --------------------------------------------------------------------- keys
//
// Rows are keys, columns the queries of a tile; all 16 warps share a tile.
// Tensor memory: dv at [0, 128), dk_1 | dk_2 at [128, 256), S_1 | S_2 at
// [256, 384), dP of even tiles at [384, 448), of odd ones at [448, 512), with dS
// in its place (16 queries of both maps: the 16 columns that their dP had).  The
// combined map, operand of dv, goes through shared memory, two tiles' worth.
// The scores are read into registers at once, so that the next tile's are
// formed while this one's exponentials are taken, and no warp waits for the
// products of the tile before.

constexpr int K_STAGES = 3;
constexpr uint32_t K_STAGE = 4 * SMALL;  // q halves, dout parts
struct KShared {
  uint64_t kv_full, q_full[K_STAGES], q_empty[K_STAGES], s_full, s_free, d_full[2], p_full[2], pv[2];
  uint64_t o_full, drain[2];
  uint32_t tmem;
  int abort_flag;
  alignas(16) float st[K_STAGES][4][COLS];  // -lse_1, -lse_2, -D_1, -D_2 of a tile's queries
};
constexpr size_t K_SMEM = 1024 + 4 * BIG + K_STAGES * K_STAGE + 2 * BIG + sizeof(KShared);

__global__ void __launch_bounds__(THREADS, 1) tc_bwd_kv_kernel(const __grid_constant__ Params p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const uint32_t sk = smem_u32(base), sv = sk + 2 * BIG, sqg = sv + 2 * BIG, sp = sqg + K_STAGES * K_STAGE;
  KShared& sh = *reinterpret_cast<KShared*>(base + 4 * BIG + K_STAGES * K_STAGE + 2 * BIG);
  volatile int* abort_flag = &sh.abort_flag;
  int* dev_error = p.dev_error;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int nbh = a.n * a.hkv, nkt = (a.tk + ROWS - 1) / ROWS;
  const bool work = static_cast<int>(blockIdx.x) < nkt * nbh;  // else a block for dlam only
  const int kt = static_cast<int>(blockIdx.x) / nbh;           // the earliest keys, which most queries see, first
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int key0 = kt * ROWS;
  const int len = key_len(a, b);
  // queries before `qbeg` see none of these keys
  int qbeg = 0;
  if (!work || key0 >= len) {
    qbeg = a.tq;
  } else if (a.causal == RNN_CAUSAL_START) {
    qbeg = min(a.tq, key0);
  } else if (a.causal == RNN_CAUSAL_END) {
    qbeg = min(a.tq, max(0, key0 - (len - a.tq)));
  }
  // tiles of all the group's queries, of which this block takes its part
  const int per = (a.tq - qbeg + COLS - 1) / COLS, all = per * a.grp;
  const int tbeg = static_cast<int>(static_cast<long long>(all) * blockIdx.y / a.kparts);
  const int nt = static_cast<int>(static_cast<long long>(all) * (blockIdx.y + 1) / a.kparts) - tbeg;
  const int wide = 2 * a.dh > 64 ? 2 : 1, ksteps = (a.dh + 15) / 16, dsteps = a.dh / 8;

  if (tid == 0) {
    mbar_init(&sh.kv_full, 1);
    for (int i = 0; i < K_STAGES; i++) {
      mbar_init(&sh.q_full[i], 2);
      mbar_init(&sh.q_empty[i], 1);
    }
    mbar_init(&sh.s_full, 1);
    mbar_init(&sh.s_free, SOFT);
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.d_full[i], 1);
      mbar_init(&sh.p_full[i], SOFT);
      mbar_init(&sh.pv[i], 1);
    }
    mbar_init(&sh.o_full, 1);
    mbar_init(&sh.drain[0], 1);
    mbar_init(&sh.drain[1], 1);
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
  const uint32_t tmem = sh.tmem;

  if (warp < SOFT) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 104;");
    const int k4 = warp >> 2, w = warp & 3, row = w * 32 + lane, key = key0 + row;
    const uint32_t lanes = static_cast<uint32_t>(w * 32) << 16;
    const uint32_t ts = tmem + lanes + 256 + k4 * 16;
    const f32x2 cc = pair(a.slog2, a.slog2);
    uint8_t* pc = base + 4 * BIG + K_STAGES * K_STAGE + row * 128;
    const int ch0 = ((2 * k4) ^ (row & 7)) << 4, ch1 = ((2 * k4 + 1) ^ (row & 7)) << 4;

    int st = 0, e = nt > 0 ? tbeg / per : 0, q0 = nt > 0 ? qbeg + tbeg % per * COLS : 0;
    for (int t = 0; t < nt; t++) {
      const float lam = __ldg(a.lam + kvh * a.grp + e);
      float x[16], y[16], dp[16];
      if (!warp_wait(&sh.q_full[st], (t / K_STAGES) & 1, abort_flag, dev_error)) break;
      if (!warp_wait(&sh.s_full, t & 1, abort_flag, dev_error)) break;
      tc_fence_after();
      tmem_ld(ts, x);
      tmem_ld(ts + 64, y);
      tmem_landed(x);
      tmem_landed(y);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.s_free);
      const float* s = &sh.st[st][0][k4 * 16];
      const f32x2 ll = pair(-lam, -lam);
      // the first query that sees this key
      int first = 0;
      if (a.causal) first = (a.causal == RNN_CAUSAL_START ? key : key - (len - a.tq)) - (q0 + k4 * 16);
      const bool edge = __any_sync(0xffffffffu, first > 0);
      auto exps = [&](int c0) {
#pragma unroll
        for (int c = c0; c < c0 + 8; c += 4) {
          const ulonglong2 n1 = *reinterpret_cast<const ulonglong2*>(s + c);
          const ulonglong2 n2 = *reinterpret_cast<const ulonglong2*>(s + COLS + c);
          unpair(fma2(pair(x[c], x[c + 1]), cc, n1.x), x[c], x[c + 1]);
          unpair(fma2(pair(y[c], y[c + 1]), cc, n2.x), y[c], y[c + 1]);
          unpair(fma2(pair(x[c + 2], x[c + 3]), cc, n1.y), x[c + 2], x[c + 3]);
          unpair(fma2(pair(y[c + 2], y[c + 3]), cc, n2.y), y[c + 2], y[c + 3]);
#pragma unroll
          for (int k = c; k < c + 4; k++) {
            x[k] = ex2(x[k]);
            y[k] = ex2(y[k]);
          }
        }
        if (__builtin_expect(edge, 0)) {
#pragma unroll
          for (int c = c0; c < c0 + 8; c++)
            if (c < first) x[c] = y[c] = 0.0f;
        }
      };
      uint32_t u[8], v[8], z[8];
      ulonglong2 e1, e2;  // -D_1, -D_2 of four queries
      auto grads = [&](int c0) {
#pragma unroll
        for (int c = c0 / 2; c < c0 / 2 + 4; c++) {
          if ((c & 1) == 0) {
            e1 = *reinterpret_cast<const ulonglong2*>(s + 2 * COLS + 2 * c);
            e2 = *reinterpret_cast<const ulonglong2*>(s + 3 * COLS + 2 * c);
          }
          const f32x2 g = pair(dp[2 * c], dp[2 * c + 1]), x2 = pair(x[2 * c], x[2 * c + 1]);
          const f32x2 y2 = mul2(pair(y[2 * c], y[2 * c + 1]), ll);  // -lam P_2
          float r0, r1;
          unpair(mul2(x2, add2(g, c & 1 ? e1.y : e1.x)), r0, r1);
          u[c] = pack2(r0, r1);
          unpair(mul2(y2, add2(g, c & 1 ? e2.y : e2.x)), r0, r1);
          v[c] = pack2(r0, r1);
          unpair(add2(x2, y2), r0, r1);
          z[c] = pack2(r0, r1);
        }
      };
      exps(0);
      exps(8);
      const uint32_t par = (t >> 1) & 1, td = ts + 128 + (t & 1) * 64;
      if (!warp_wait(&sh.d_full[t & 1], par, abort_flag, dev_error)) break;
      tc_fence_after();
      tmem_ld(td, dp);
      tmem_landed(dp);
      grads(0);
      grads(8);
      tmem_st(td, u);
      tmem_st(td + 8, v);
      // the products of two tiles ago have read the combined map's place
      if (t > 1 && !warp_wait(&sh.pv[t & 1], par ^ 1, abort_flag, dev_error)) break;
      uint8_t* pt = pc + (t & 1) * BIG;
      *reinterpret_cast<uint4*>(pt + ch0) = make_uint4(z[0], z[1], z[2], z[3]);
      *reinterpret_cast<uint4*>(pt + ch1) = make_uint4(z[4], z[5], z[6], z[7]);
      fence_async_smem();
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[t & 1]);
      if (++st == K_STAGES) st = 0;
      q0 += COLS;
      if (q0 >= qbeg + per * COLS) {
        q0 = qbeg;
        e++;
      }
    }
    bool ok = true;
    if (nt > 0) {
      ok = warp_wait(&sh.o_full, 0, abort_flag, dev_error);
      tc_fence_after();
    }
    if (ok && work) {
      const bool some = nt > 0 && key < len && (!a.kmask || a.kmask[b * a.kmb + key]);
      __nv_bfloat16* odk = static_cast<__nv_bfloat16*>(a.dk) + b * a.dkb + kvh * a.dkh + key * a.dkr;
      __nv_bfloat16* odv = static_cast<__nv_bfloat16*>(a.dv) + b * a.dvb + kvh * a.dvh + key * a.dvr;
      float* part = a.kparts > 1
                        ? a.kpart + ((static_cast<long long>(blockIdx.y) * nbh + bh) * a.tk + key) * 256 + k4 * 16
                        : nullptr;
#pragma unroll
      for (int m = 0; m < 4; m++) {
        float x[16] = {};
        if (nt > 0) {
          tmem_ld(tmem + lanes + m * 64 + k4 * 16, x);
          tmem_landed(x);
        }
        if (key < a.tk && part) {
#pragma unroll
          for (int c = 0; c < 16; c += 4)
            *reinterpret_cast<float4*>(part + m * 64 + c) =
                some ? make_float4(x[c], x[c + 1], x[c + 2], x[c + 3]) : make_float4(0.0f, 0.0f, 0.0f, 0.0f);
        } else if (key < a.tk) {
          if (m < 2) {
            store16(odv + m * 64 + k4 * 16, x, 1.0f, some, 2 * a.dh - m * 64 - k4 * 16, p.st16);
          } else {
            store16(odk + (m - 2) * a.dh + k4 * 16, x, a.scale, some, a.dh - k4 * 16, p.st16);
          }
        }
        __syncwarp();
      }
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 64;");
    if (warp == WARP_COPY) {
      if (nt > 0) {
        const bool lead = elect_one();
        if (lead) {
          mbar_arrive_expect_tx(&sh.kv_full, (2 + wide) * BIG);
          for (int h = 0; h < 2; h++) tma_5d(sk + h * BIG, &p.k, 0, h, kvh, key0, b, &sh.kv_full);
          for (int c = 0; c < wide; c++) tma_5d(sv + c * BIG, &p.v, c * 64, 0, kvh, key0, b, &sh.kv_full);
        }
        int t = 0;
        for (; t < nt; t++) {
          const int st = t % K_STAGES;
          if (t >= K_STAGES && !warp_wait(&sh.q_empty[st], (t / K_STAGES - 1) & 1, abort_flag, dev_error)) break;
          const uint32_t dst = sqg + st * K_STAGE;
          const int head = kvh * a.grp + (tbeg + t) / per, i0 = qbeg + (tbeg + t) % per * COLS;
          if (lead) {
            mbar_arrive_expect_tx(&sh.q_full[st], (2 + wide) * SMALL);
            for (int h = 0; h < 2; h++) tma_5d(dst + h * SMALL, &p.q, 0, h, head, i0, b, &sh.q_full[st]);
            for (int c = 0; c < wide; c++) tma_5d(dst + (2 + c) * SMALL, &p.g, c * 64, 0, head, i0, b, &sh.q_full[st]);
          }
          __syncwarp();
          const long long at = (static_cast<long long>(b) * a.h + head) * 2 * a.tq;
#pragma unroll
          for (int c = lane; c < COLS; c += 32) {
            const int i = i0 + c;
            const bool in = i < a.tq;
            sh.st[st][0][c] = in ? -a.flse[at + i] : -CUDART_INF_F;
            sh.st[st][1][c] = in ? -a.flse[at + a.tq + i] : -CUDART_INF_F;
            sh.st[st][2][c] = in ? -a.dsum[at + i] : 0.0f;
            sh.st[st][3][c] = in ? -a.dsum[at + a.tq + i] : 0.0f;
          }
          __syncwarp();
          if (lane == 0) mbar_arrive(&sh.q_full[st]);
        }
        // what was asked for lands before the block may end, aborting or not
        settle(&sh.kv_full, 0);
        for (int i = max(0, t - K_STAGES); i < t; i++) settle(&sh.q_full[i % K_STAGES], (i / K_STAGES) & 1);
      }
      __syncwarp();
    } else if (warp == WARP_AUX) {
      // dlam: block `head` sums that head's rows in a fixed order
      if (static_cast<int>(blockIdx.x) < a.h && blockIdx.y == 0 && a.tq > 0) {
        const long long cnt = static_cast<long long>(a.n) * a.tq;
        const float* x = a.dlrow + blockIdx.x * cnt;
        double s[4] = {0.0, 0.0, 0.0, 0.0};
        long long i = lane;
        for (; i + 96 < cnt; i += 128)
#pragma unroll
          for (int k = 0; k < 4; k++) s[k] += x[i + 32 * k];
        for (; i < cnt; i += 32) s[0] += x[i];
        double sum = (s[0] + s[1]) + (s[2] + s[3]);
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
        if (lane == 0) a.dlam[blockIdx.x] -= static_cast<float>(sum);
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(ROWS, 64, false);
      auto done = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity, abort_flag, dev_error); };
      auto landed = [&](int t, int st) { return done(&sh.q_full[st], (t / K_STAGES) & 1); };
      bool ok = done(&sh.kv_full, 0);
      int st = 0;
      if (warp == WARP_SCORE) {
        const uint64_t dk = desc_k(sk), dqg = desc_k(sqg);
        for (int t = 0; ok && t < nt; t++) {
          // the warps have the scores of tile t - 1 in registers
          if (!(ok = landed(t, st) && (t < 1 || done(&sh.s_free, (t - 1) & 1)))) break;
          tc_fence_after();
          const uint64_t q = dqg + st * (K_STAGE / 16);
#pragma unroll
          for (int h = 0; h < 2; h++)
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
              if (ks < ksteps)
                mma_ss(tmem + 256 + h * 64, dk + (h * BIG + ks * 32) / 16, q + (h * SMALL + ks * 32) / 16, id_s, ks > 0,
                       lead);
          commit(&sh.s_full, lead);
          if (++st == K_STAGES) st = 0;
        }
      } else {
        const uint32_t id_k = idesc_bf16(ROWS, 64, true), id_v = idesc_bf16(ROWS, 2 * a.dh, true);
        const uint64_t dv = desc_k(sv), dqg = desc_k(sqg), dp = desc_k(sp);
        const uint64_t mq = desc_mn(sqg, 0), mg = desc_mn(sqg + 2 * SMALL, SMALL);
        auto slopes = [&](int t, int s1) {
          const uint64_t q = dqg + s1 * (K_STAGE / 16);
#pragma unroll
          for (int ks = 0; ks < 8; ks++)
            if (ks < dsteps)
              mma_ss(tmem + 384 + (t & 1) * 64, dv + ((ks >> 2) * BIG + (ks & 3) * 32) / 16,
                     q + ((2 + (ks >> 2)) * SMALL + (ks & 3) * 32) / 16, id_s, ks > 0, lead);
          commit(&sh.d_full[t & 1], lead);
        };
        for (int t = 0; ok && t < min(nt, 2); t++)
          if ((ok = landed(t, t))) {
            tc_fence_after();
            slopes(t, t);
          }
        int st2 = 2;
        for (int t = 0; ok && t < nt; t++) {
          if (!(ok = done(&sh.p_full[t & 1], (t >> 1) & 1))) break;
          tc_fence_after();
          const uint64_t q = mq + st * (K_STAGE / 16), g = mg + st * (K_STAGE / 16);
          const uint64_t pt = dp + (t & 1) * (BIG / 16);
          const uint32_t ds = tmem + 384 + (t & 1) * 64;
#pragma unroll
          for (int m = 0; m < 2; m++)
#pragma unroll
            for (int ks = 0; ks < 4; ks++)
              mma_ts(tmem + 128 + m * 64, ds + ks * 16 + m * 8, q + (m * SMALL + ks * 2048) / 16, id_k, t > 0 || ks > 0,
                     lead);
#pragma unroll
          for (int ks = 0; ks < 4; ks++) mma_ss(tmem, pt + ks * 2, g + ks * (2048 / 16), id_v, t > 0 || ks > 0, lead);
          commit(&sh.pv[t & 1], lead);
          // the scores of tile t are long done: dS came of them
          commit(&sh.q_empty[st], lead);
          if (t + 1 == nt) commit(&sh.o_full, lead);
          if (t + 2 < nt) {
            // in the place of the dS that the products above have read (they are
            // of the same accumulator shape, and so executed before)
            if (!(ok = landed(t + 2, st2))) break;
            tc_fence_after();
            slopes(t + 2, st2);
          }
          if (++st == K_STAGES) st = 0;
          if (++st2 == K_STAGES) st2 = 0;
        }
      }
      if (!ok) {  // no MMA may write tensor memory after it is released
        uint64_t* drain = &sh.drain[warp == WARP_SCORE];
        commit(drain, lead);
        settle(drain, 0);
      }
      __syncwarp();
    }
  }

  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == WARP_MMA) tmem_dealloc(tmem, 512);
}

// Joins the parts of dk and dv in their order: 64 threads a key, four of its 256
// columns each.
__global__ void __launch_bounds__(256) join_keys_kernel(Args a) {
  const long long total = static_cast<long long>(a.n) * a.hkv * a.tk;
  const long long idx = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (idx >= total) return;
  const int c = (threadIdx.x & 63) * 4;
  float4 s = make_float4(0.0f, 0.0f, 0.0f, 0.0f);
#pragma unroll 4
  for (int k = 0; k < a.kparts; k++) {
    const float4 x = *reinterpret_cast<const float4*>(a.kpart + (k * total + idx) * 256 + c);
    s.x += x.x;
    s.y += x.y;
    s.z += x.z;
    s.w += x.w;
  }
  const int key = static_cast<int>(idx % a.tk), bh = static_cast<int>(idx / a.tk);
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  __nv_bfloat16* o;
  if (c < 128) {
    if (c >= 2 * a.dh) return;
    o = static_cast<__nv_bfloat16*>(a.dv) + b * a.dvb + kvh * a.dvh + key * a.dvr + c;
  } else {
    const int m = c >= 192 ? 1 : 0, w = c - 128 - m * 64;
    if (w >= a.dh) return;
    o = static_cast<__nv_bfloat16*>(a.dk) + b * a.dkb + kvh * a.dkh + key * a.dkr + m * a.dh + w;
    s = make_float4(s.x * a.scale, s.y * a.scale, s.z * a.scale, s.w * a.scale);
  }
  o[0] = __float2bfloat16_rn(s.x);
  o[1] = __float2bfloat16_rn(s.y);
  o[2] = __float2bfloat16_rn(s.z);
  o[3] = __float2bfloat16_rn(s.w);
}

bool mult8(std::initializer_list<long long> s) {
  for (long long x : s)
    if (x % 8) return false;
  return true;
}

}  // namespace

// What is short on both sides or little work stays with the kernels of mma.sync,
// whose blocks start and end faster (256 x 48 x 48, 4 heads of 32: 69 us against 86 here; 128 x
// 64 x 64: 49 against 50).  The rest is faster here, few rows over many keys too
// (4 x 4 x 4096, 32 heads on 4: 132 us against 468; 64 x 24 x 256, 8 heads of 32:
// 84 against 88; 32 x 1000 x 16, 8 of 64: 163 against 281).
bool tc_bwd_ok(const Args& a) {
  if (a.dh % 8 || a.dh > 64 || !(a.slog2 > 0.0f) || a.slog2 > 1e30f) return false;
  if (!big_enough(a)) return false;
  if (reinterpret_cast<uintptr_t>(a.fo) % 16 || reinterpret_cast<uintptr_t>(a.fo2) % 16) return false;
  if (!mult8({a.ob, a.orow, a.oh})) return false;
  return map_ok(a.q, a.n, a.tq, a.h, a.dh, a.qb, a.qr, a.qh) && map_ok(a.k, a.n, a.tk, a.hkv, a.dh, a.kb, a.kr, a.kh) &&
         map_ok(a.v, a.n, a.tk, a.hkv, 2 * a.dh, a.vb, a.vr, a.vh) &&
         map_ok(a.dout, a.n, a.tq, a.h, 2 * a.dh, a.gb, a.gr, a.gh);
}

int tc_bwd(rnn_ctx* ctx, const Args& a) {
  Params p;
  p.a = a;
  p.dev_error = ctx->dev_error;
  p.st16 = mult8({a.dqb, a.dqr, a.dqh, a.dkb, a.dkr, a.dkh, a.dvb, a.dvr, a.dvh}) &&
           (reinterpret_cast<uintptr_t>(a.dq) | reinterpret_cast<uintptr_t>(a.dk) | reinterpret_cast<uintptr_t>(a.dv)) %
                   16 == 0;
  const long long qblocks = (a.tq + ROWS - 1ll) / ROWS * a.n * a.h;
  const long long kblocks = std::max<long long>((a.tk + ROWS - 1ll) / ROWS * a.n * a.hkv, a.h);
  RNN_REQUIRE(qblocks < (1ll << 31) && kblocks < (1ll << 31), "diffattn: too many rows");
  static std::atomic<unsigned long long> optin_q[2], optin_k{0};
  const auto q_kernel = a.kmask ? tc_bwd_q_kernel<true> : tc_bwd_q_kernel<false>;
  RNN_TRY(tc::ensure_smem_optin(q_kernel, optin_q[a.kmask != nullptr], ctx->device, static_cast<int>(Q_SMEM)));
  RNN_TRY(tc::ensure_smem_optin(tc_bwd_kv_kernel, optin_k, ctx->device, static_cast<int>(K_SMEM)));
  RNN_TRY(encode_map(&p.q, a.q, a.n, a.tq, a.h, 2, a.dh, a.qb, a.qr, a.qh, ROWS));
  RNN_TRY(encode_map(&p.g, a.dout, a.n, a.tq, a.h, 1, 2 * a.dh, a.gb, a.gr, a.gh, ROWS));
  RNN_TRY(encode_map(&p.k, a.k, a.n, a.tk, a.hkv, 2, a.dh, a.kb, a.kr, a.kh, COLS));
  RNN_TRY(encode_map(&p.v, a.v, a.n, a.tk, a.hkv, 1, 2 * a.dh, a.vb, a.vr, a.vh, COLS));
  q_kernel<<<static_cast<unsigned>(qblocks), THREADS, Q_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  // the keys' kernel owns 128 keys and reads the queries 64 at a time
  RNN_TRY(encode_map(&p.q, a.q, a.n, a.tq, a.h, 2, a.dh, a.qb, a.qr, a.qh, COLS));
  RNN_TRY(encode_map(&p.g, a.dout, a.n, a.tq, a.h, 1, 2 * a.dh, a.gb, a.gr, a.gh, COLS));
  RNN_TRY(encode_map(&p.k, a.k, a.n, a.tk, a.hkv, 2, a.dh, a.kb, a.kr, a.kh, ROWS));
  RNN_TRY(encode_map(&p.v, a.v, a.n, a.tk, a.hkv, 1, 2 * a.dh, a.vb, a.vr, a.vh, ROWS));
  tc_bwd_kv_kernel<<<dim3(static_cast<unsigned>(kblocks), a.kparts), THREADS, K_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  if (a.kparts > 1) {
    const long long keys = static_cast<long long>(a.n) * a.hkv * a.tk;
    join_keys_kernel<<<static_cast<unsigned>((keys + 3) / 4), 256, 0, ctx->stream>>>(p.a);
    RNN_CHECK_LAUNCH();
  }
  return RNN_OK;
}

// When the keys alone leave SMs idle (few sequences and key heads), the queries
// of a key tile are split over blocks.  Time is counted in tiles (about 1.1 us):
// the waves of blocks, each with its share and a start and end worth six tiles,
// and the parts' way through memory.  Measured: 5 x 1003 tokens, 2 key heads of
// 3 queries' heads each (80 key tiles), 75 us whole and 50 in three parts with
// their join; 2 x 1024, 8 heads (128 key tiles), 63 us whole and 85 in two parts.
int tc_bwd_parts(rnn_ctx* ctx, const Args& a) {
  const double blocks = static_cast<double>((a.tk + ROWS - 1) / ROWS) * a.n * a.hkv;
  const double tiles = static_cast<double>((a.tq + COLS - 1) / COLS) * a.grp;
  const double pass = 2048.0 * a.n * a.hkv * a.tk / 6.5e12 / 1.1e-6;  // a part written and read
  int best = 1;
  double least = 0.0;
  for (int parts = 1; parts <= 16 && (parts == 1 || tiles >= 4.0 * parts); parts++) {
    const double waves = std::ceil(blocks * parts / ctx->num_sms);
    const double time = waves * (tiles / parts + 6.0) + (parts > 1 ? 4.0 + parts * pass : 0.0);
    if (parts == 1 || time < least) {
      least = time;
      best = parts;
    }
  }
  return best;
}

}  // namespace diff
}  // namespace rnn
