// Differential attention, forward and backward, on warp-level matrix
// products: every type, width, stride and mask.
//
// Forward.  One pass over the keys with running maxima and sums of both maps.
// Subtracting two separately rounded maps would lose what they have in common,
// so the accumulators hold
//   A = sum_j (P_1 - r P_2) v   and   B = sum_j P_2 v      (unnormalised)
// with r = lam l_1 / l_2 of the keys read so far: the combined map is rounded
// once.  When maxima and sums move by alpha_m = exp(m_old - m_new), A becomes
//   alpha_1 A + (r_old alpha_1 - r_new alpha_2) B,
// so that after the last key o = A / l_1 exactly, and P_2 v = B / l_2.
//
// Backward.  With dP = do v^T and D_m = sum_j P_m dP:
//   dS_1 = P_1 (dP - D_1),  dS_2 = -lam P_2 (dP - D_2),
//   dq_m = scale dS_m k_m,  dk_m = scale dS_m^T q_m,
//   dv = (P_1 - lam P_2)^T do,  dlam = -sum_rows D_2.
// Two kernels recompute the maps from the saved log-sums: one owns query rows
// (dq, and D, of which dlam is the sum), one owns keys (dk, dv).  No
// atomics: results do not depend on scheduling.
//
// Bound by the latency of dependent instructions (8 to 12 warps fit an SM, two
// thirds of their waits are fixed latencies; the tensor pipe is 40 % busy), so
// only what is too small or too odd for the tcgen05 kernels is left to these.
// Measured: f32 forward of 128 x 64 x 64, 4 heads of 32: 30 us with a cold L2.
#include <algorithm>

#include "diffattn_tc.cuh"

namespace rnn {
namespace diff {
namespace {

constexpr int THREADS = 128;

// ------------------------------------------------------------------ forward
//
// Four warps: RW of them share the block's 16 * RW packed rows, the 4 / RW
// warps of a row group take the keys of a tile in turn.  RW = 4 for ordinary
// calls, RW = 1 when a (sequence, key head) has at most 16 rows (new tokens
// against a cache): the call is then a read of the cache, and each key is read
// once.  When the rows alone leave SMs idle the keys are split over blocks and
// a second kernel joins the parts.

template <class T, int DH, int RW>
struct Fwd {
  using G = Geo<T, DH>;
  static constexpr int KW = 4 / RW;
  static constexpr int ROWS = 16 * RW;
  static constexpr int BN = (sizeof(T) == 4 ? 32 : 64) * (KW > 1 ? 2 : 1);  // keys per stage
  static constexpr int SUBK = KW > 1 && BN / KW < G::SUB ? BN / KW : G::SUB;
  static constexpr int Q_ELEMS = ROWS * G::PITCH, KV_ELEMS = BN * G::PITCH;
  static constexpr size_t TILES = (Q_ELEMS + 4 * KV_ELEMS) * sizeof(T);
  static constexpr size_t SMEM = TILES + 2 * BN;  // + one visibility byte per key and stage
  // the join of the key warps reuses the tiles
  static_assert(KW == 1 || static_cast<size_t>(KW) * ROWS * (2 * G::W + 4) * 4 <= TILES, "join fits");
};

template <class T, int DH, int RW>
__global__ void __launch_bounds__(THREADS) fwd_kernel(Args a) {
  using F = Fwd<T, DH, RW>;
  using G = Geo<T, DH>;
  using FR = Frag<T>;
  constexpr int W = G::W, PITCH = G::PITCH, KS = G::KS, SUB = F::SUBK, BN = F::BN;
  constexpr int NS = SUB / 8, NB = W / 8, NSIDE = NS < G::SIDE ? NS : G::SIDE;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sq = reinterpret_cast<T*>(smem);
  T* sk = sq + F::Q_ELEMS;
  T* sv = sk + 2 * F::KV_ELEMS;
  uint8_t* sok = smem + F::TILES;

  const int rows = a.grp * a.tq;  // packed rows of a (sequence, key head)
  const int ntile = (rows + F::ROWS - 1) / F::ROWS;
  const int nbh = a.n * a.hkv;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;  // longest causal rows first
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int rw = warp % RW, kw = warp / RW;
  const int row0 = tile * F::ROWS;
  const int len = key_len(a, b);

  const T* qp = static_cast<const T*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + kvh * a.vh;
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;

  // keys that some row of the block sees, cut to this block's part
  int kend = len;
  if (a.causal) {
    kend = 0;
    const int last = min(rows, row0 + F::ROWS) - 1;
    // a block that spans a head's end holds that head's last query
    const int imax = last / a.tq != row0 / a.tq ? a.tq - 1 : last % a.tq;
    kend = row_limit(a, imax, len);
  }
  int kbeg = 0;
  if (a.nsplit > 1) {
    kbeg = static_cast<int>(blockIdx.y) * a.split_keys;
    kend = min(kend, kbeg + a.split_keys);
  }
  const int ntk = kend > kbeg ? (kend - kbeg + BN - 1) / BN : 0;

  // this lane's two rows
  int lim[2];
  float lam[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = row0 + rw * 16 + (lane >> 2) + 8 * i;
    lim[i] = r < rows ? min(kend, row_limit(a, r % a.tq, len)) : 0;
    lam[i] = r < rows ? __ldg(a.lam + kvh * a.grp + r / a.tq) : 0.0f;
  }
  // keys below this are visible to all rows of the warp unless masked
  const int full = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));

  float A[NB][4], B[NB][4];
#pragma unroll
  for (int i = 0; i < NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) A[i][j] = B[i][j] = 0.0f;
  float m1[2] = {-CUDART_INF_F, -CUDART_INF_F}, m2[2] = {-CUDART_INF_F, -CUDART_INF_F};
  float l1[2] = {0.0f, 0.0f}, l2[2] = {0.0f, 0.0f}, ratio[2] = {lam[0], lam[1]};

  auto load_kv = [&](int t) {
    const int st = t & 1, j0 = kbeg + t * BN;
    auto at = [&](const T* p, long long stride, int r) -> const T* {
      const int j = j0 + r;
      return j < kend && (!mask || mask[j]) ? p + j * stride : nullptr;
    };
    load_tile<T, DH, BN, THREADS, true>(sk + st * F::KV_ELEMS, kp, a.dh, a.vec,
                                        [&](int r) { return at(kp, a.kr, r); });
    load_tile<T, DH, BN, THREADS, false>(sv + st * F::KV_ELEMS, vp, a.dh, a.vec,
                                         [&](int r) { return at(vp, a.vr, r); });
    if (mask)
      for (int r = tid; r < BN; r += THREADS) sok[st * BN + r] = j0 + r < kend && mask[j0 + r];
    cp_commit();
  };
  if (ntk > 0) {
    load_tile<T, DH, F::ROWS, THREADS, true>(sq, qp, a.dh, a.vec, [&](int r) -> const T* {
      const int p = row0 + r;
      if (p >= rows) return nullptr;
      const int e = p / a.tq;
      return qp + e * a.qh + (p - e * a.tq) * a.qr;
    });
    load_kv(0);
  }

  for (int t = 0; t < ntk; t++) {
    if (t + 1 < ntk) {
      load_kv(t + 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    const T* k = sk + (t & 1) * F::KV_ELEMS;
    const T* v = sv + (t & 1) * F::KV_ELEMS;
    const uint8_t* ok = sok + (t & 1) * BN;
    for (int s0 = kw * (BN / F::KW); s0 < (kw + 1) * (BN / F::KW); s0 += SUB) {
      const int j0 = kbeg + t * BN + s0;
      if (j0 >= kend) break;
      float s1[NS][4], s2[NS][4], m1s[NS][4] = {}, m2s[NS][4] = {};
#pragma unroll
      for (int i = 0; i < NS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s1[i][j] = s2[i][j] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < DH / KS; ks++) {
        const typename FR::A q1 = FR::ldA(sq, PITCH, rw * 16, ks * KS, lane);
        const typename FR::A q2 = FR::ldA(sq, PITCH, rw * 16, DH + ks * KS, lane);
#pragma unroll
        for (int nb = 0; nb < NS; nb += NSIDE) {
          typename FR::B f[NSIDE], g[NSIDE];
          FR::ldB_nk(f, k, PITCH, s0 + nb * 8, ks * KS, lane);
          FR::ldB_nk(g, k, PITCH, s0 + nb * 8, DH + ks * KS, lane);
          FR::mma(s1 + nb, m1s + nb, q1, f);
          FR::mma(s2 + nb, m2s + nb, q2, g);
        }
      }
      FR::join(s1, m1s);
      FR::join(s2, m2s);
      const bool edge = mask != nullptr || j0 + SUB > full;
      float mx1[2] = {m1[0], m1[1]}, mx2[2] = {m2[0], m2[1]};
#pragma unroll
      for (int nb = 0; nb < NS; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          float x = s1[nb][e] * a.slog2, y = s2[nb][e] * a.slog2;
          if (edge) {
            const int c = nb * 8 + 2 * (lane & 3) + (e & 1);
            if (j0 + c >= lim[e >> 1] || (mask && !ok[s0 + c])) x = y = -CUDART_INF_F;
          }
          s1[nb][e] = x;
          s2[nb][e] = y;
          mx1[e >> 1] = fmaxf(mx1[e >> 1], x);
          mx2[e >> 1] = fmaxf(mx2[e >> 1], y);
        }
      float al1[2], al2[2], de[2], u1[2], u2[2], t1[2] = {0.0f, 0.0f}, t2[2] = {0.0f, 0.0f};
#pragma unroll
      for (int i = 0; i < 2; i++) {
        mx1[i] = quad_max(mx1[i]);
        mx2[i] = quad_max(mx2[i]);
        // a row without a visible key so far keeps its maximum at -inf
        u1[i] = mx1[i] == -CUDART_INF_F ? 0.0f : mx1[i];
        u2[i] = mx2[i] == -CUDART_INF_F ? 0.0f : mx2[i];
        al1[i] = ex2(m1[i] - u1[i]);
        al2[i] = ex2(m2[i] - u2[i]);
        m1[i] = mx1[i];
        m2[i] = mx2[i];
      }
#pragma unroll
      for (int nb = 0; nb < NS; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          s1[nb][e] = ex2(s1[nb][e] - u1[e >> 1]);
          s2[nb][e] = ex2(s2[nb][e] - u2[e >> 1]);
          t1[e >> 1] += s1[nb][e];
          t2[e >> 1] += s2[nb][e];
        }
#pragma unroll
      for (int i = 0; i < 2; i++) {
        l1[i] = l1[i] * al1[i] + quad_sum(t1[i]);
        l2[i] = l2[i] * al2[i] + quad_sum(t2[i]);
        const float now = l2[i] > 0.0f ? lam[i] * __fdividef(l1[i], l2[i]) : lam[i];
        de[i] = ratio[i] * al1[i] - now * al2[i];
        ratio[i] = now;
      }
#pragma unroll
      for (int nb = 0; nb < NS; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) s1[nb][e] -= ratio[e >> 1] * s2[nb][e];
      typename FR::A pa[SUB / KS], pb[SUB / KS];
#pragma unroll
      for (int ks = 0; ks < SUB / KS; ks++) {
        pa[ks] = FR::from_acc(s1, ks);
        pb[ks] = FR::from_acc(s2, ks);
      }
      // the step's products start at zero and join the accumulators in one
      // f32 addition, so long sums are not left to the MMA's own rounding
#pragma unroll
      for (int nb = 0; nb < NB; nb += G::SIDE) {
        float x[G::SIDE][4] = {}, y[G::SIDE][4] = {}, xs[G::SIDE][4] = {}, ys[G::SIDE][4] = {};
#pragma unroll
        for (int ks = 0; ks < SUB / KS; ks++) {
          typename FR::B f[G::SIDE];
          FR::ldB_kn(f, v, PITCH, s0 + ks * KS, nb * 8, lane);
          FR::mma(x, xs, pa[ks], f);
          FR::mma(y, ys, pb[ks], f);
        }
        FR::join(x, xs);
        FR::join(y, ys);
#pragma unroll
        for (int i = 0; i < G::SIDE; i++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int h = e >> 1;
            A[nb + i][e] = al1[h] * A[nb + i][e] + (de[h] * B[nb + i][e] + x[i][e]);
            B[nb + i][e] = al2[h] * B[nb + i][e] + y[i][e];
          }
      }
    }
    __syncthreads();
  }

  if constexpr (F::KW > 1) {
    // join the key warps through shared memory; warp 0 finishes
    float* sj = reinterpret_cast<float*>(smem);
    constexpr int RJ = 2 * W + 4;
    const int g = lane >> 2, q = lane & 3;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      float* r = sj + (kw * F::ROWS + g + 8 * i) * RJ;
#pragma unroll
      for (int nb = 0; nb < NB; nb++)
#pragma unroll
        for (int e = 0; e < 2; e++) {
          const float o2 = B[nb][2 * i + e];
          r[nb * 8 + 2 * q + e] = A[nb][2 * i + e] + ratio[i] * o2;
          r[W + nb * 8 + 2 * q + e] = o2;
        }
      if (q == 0) {
        r[2 * W] = m1[i];
        r[2 * W + 1] = l1[i];
        r[2 * W + 2] = m2[i];
        r[2 * W + 3] = l2[i];
      }
    }
    __syncthreads();
    // thread (row, column group): all 128 threads share the block's 16 rows
    const int r = tid >> 3, c0 = tid & 7;
    const int p = row0 + r;
    if (p >= rows) return;
    float M1 = -CUDART_INF_F, M2 = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < F::KW; w++) {
      M1 = fmaxf(M1, sj[(w * F::ROWS + r) * RJ + 2 * W]);
      M2 = fmaxf(M2, sj[(w * F::ROWS + r) * RJ + 2 * W + 2]);
    }
    const float U1 = M1 == -CUDART_INF_F ? 0.0f : M1, U2 = M2 == -CUDART_INF_F ? 0.0f : M2;
    float w1[F::KW], w2[F::KW], L1 = 0.0f, L2 = 0.0f;
#pragma unroll
    for (int w = 0; w < F::KW; w++) {
      const float* s = sj + (w * F::ROWS + r) * RJ + 2 * W;
      w1[w] = ex2(s[0] - U1);
      w2[w] = ex2(s[2] - U2);
      L1 += w1[w] * s[1];
      L2 += w2[w] * s[3];
    }
    const int e = p / a.tq, i = p - e * a.tq;
    const int head = kvh * a.grp + e;
    if (a.nsplit > 1) {
      const long long row = (static_cast<long long>(blockIdx.y) * nbh + bh) * rows + p;
      for (int c = c0; c < 2 * W; c += 8) {
        float x = 0.0f;
#pragma unroll
        for (int w = 0; w < F::KW; w++) x += (c < W ? w1[w] : w2[w]) * sj[(w * F::ROWS + r) * RJ + c];
        a.part[row * (2 * W) + c] = x;
      }
      if (c0 == 0) {
        float* s = a.stat + row * 4;
        s[0] = M1;
        s[1] = L1;
        s[2] = M2;
        s[3] = L2;
      }
      return;
    }
    const float i1 = inverse(L1), i2 = inverse(L2);
    const float lm = L2 == 0.0f ? 0.0f : __ldg(a.lam + head);
    T* o = static_cast<T*>(a.o) + b * a.ob + head * a.oh + i * a.orow;
    T* o2 = a.o2 ? static_cast<T*>(a.o2) + ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) : nullptr;
    for (int c = c0; c < 2 * a.dh; c += 8) {
      float x = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < F::KW; w++) {
        x += w1[w] * sj[(w * F::ROWS + r) * RJ + c];
        y += w2[w] * sj[(w * F::ROWS + r) * RJ + W + c];
      }
      o[c] = from_f<T>(x * i1 - lm * (y * i2));
      if (o2) o2[c] = from_f<T>(y * i2);
    }
    if (a.lse && c0 == 0) {
      float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
      s[0] = log_sum(M1, L1);
      s[a.tq] = log_sum(M2, L2);
    }
  } else {
#pragma unroll
    for (int h = 0; h < 2; h++) {
      const int p = row0 + rw * 16 + (lane >> 2) + 8 * h;
      if (p >= rows) continue;
      const int e = p / a.tq, i = p - e * a.tq;
      const int head = kvh * a.grp + e;
      if (a.nsplit > 1) {
        const long long row = (static_cast<long long>(blockIdx.y) * nbh + bh) * rows + p;
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
          float* q = a.part + row * (2 * W) + nb * 8 + 2 * (lane & 3);
          const float x = B[nb][2 * h], y = B[nb][2 * h + 1];
          *reinterpret_cast<float2*>(q) =
              make_float2(A[nb][2 * h] + ratio[h] * x, A[nb][2 * h + 1] + ratio[h] * y);
          *reinterpret_cast<float2*>(q + W) = make_float2(x, y);
        }
        if ((lane & 3) == 0)
          *reinterpret_cast<float4*>(a.stat + row * 4) = make_float4(m1[h], l1[h], m2[h], l2[h]);
        continue;
      }
      const float i2 = inverse(l2[h]);
      // where the first map is 0 A holds nothing, and o = -lam P_2 v
      const float i1 = inverse(l1[h]), f2 = l1[h] == 0.0f && l2[h] != 0.0f ? -lam[h] * i2 : 0.0f;
      T* o = static_cast<T*>(a.o) + b * a.ob + head * a.oh + i * a.orow;
      T* o2 =
          a.o2 ? static_cast<T*>(a.o2) + ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) : nullptr;
#pragma unroll
      for (int nb = 0; nb < NB; nb++) {
        const int c = nb * 8 + 2 * (lane & 3);
        const float x = A[nb][2 * h] * i1 + f2 * B[nb][2 * h], y = A[nb][2 * h + 1] * i1 + f2 * B[nb][2 * h + 1];
        store2(o + c, x, y, c < 2 * a.dh, c + 1 < 2 * a.dh, a.pair);
        if (o2) store2(o2 + c, B[nb][2 * h] * i2, B[nb][2 * h + 1] * i2, c < 2 * a.dh, c + 1 < 2 * a.dh, true);
      }
      if (a.lse && (lane & 3) == 0) {
        float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
        s[0] = log_sum(m1[h], l1[h]);
        s[a.tq] = log_sum(m2[h], l2[h]);
      }
    }
  }
}

// Joins the key parts of a row: one block per packed row.  Its threads weigh the
// parts first; then 2 * W threads take a column each and groups of them a share
// of the parts each, so that the loads of all parts are in flight at once.
constexpr int JOIN_THREADS = 256, JOIN_PARTS = 1184;  // parts at most: eight for each SM

template <class T, int W>
__global__ void __launch_bounds__(JOIN_THREADS) join_kernel(Args a) {
  constexpr int GROUPS = JOIN_THREADS / W > 0 ? JOIN_THREADS / W : 1;
  __shared__ float4 w[JOIN_PARTS];  // w_1, w_2 and what the sums get of each
  __shared__ float2 red[JOIN_THREADS / 32], acc[GROUPS][W];
  const int rows = a.grp * a.tq;
  const long long total = static_cast<long long>(a.n) * a.hkv * rows, idx = blockIdx.x;
  const int tid = threadIdx.x, lane = tid & 31;
  const int p = static_cast<int>(idx % rows), bh = static_cast<int>(idx / rows);
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  float M1 = -CUDART_INF_F, M2 = -CUDART_INF_F;
  for (int s = tid; s < a.nsplit; s += JOIN_THREADS) {
    w[s] = *reinterpret_cast<const float4*>(a.stat + (s * total + idx) * 4);
    M1 = fmaxf(M1, w[s].x);
    M2 = fmaxf(M2, w[s].z);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    M1 = fmaxf(M1, __shfl_xor_sync(0xffffffffu, M1, o));
    M2 = fmaxf(M2, __shfl_xor_sync(0xffffffffu, M2, o));
  }
  if (lane == 0) red[tid >> 5] = make_float2(M1, M2);
  __syncthreads();
#pragma unroll
  for (int i = 0; i < JOIN_THREADS / 32; i++) {
    M1 = fmaxf(M1, red[i].x);
    M2 = fmaxf(M2, red[i].y);
  }
  const float U1 = M1 == -CUDART_INF_F ? 0.0f : M1, U2 = M2 == -CUDART_INF_F ? 0.0f : M2;
  for (int s = tid; s < a.nsplit; s += JOIN_THREADS) {
    const float4 v = w[s];
    const float w1 = ex2(v.x - U1), w2 = ex2(v.z - U2);
    w[s] = make_float4(w1, w2, w1 * v.y, w2 * v.w);
  }
  __syncthreads();
  const int col = tid % W, grp = tid / W;
  float x = 0.0f, y = 0.0f;
#pragma unroll 8
  for (int s = grp; s < a.nsplit; s += GROUPS) {
    const float* q = a.part + (s * total + idx) * (2 * W) + col;
    x += w[s].x * q[0];
    y += w[s].y * q[W];
  }
  acc[grp][col] = make_float2(x, y);
  __syncthreads();
  if (tid >= W) return;
  float L1 = 0.0f, L2 = 0.0f;
  for (int s = 0; s < a.nsplit; s++) {
    L1 += w[s].z;
    L2 += w[s].w;
  }
  x = y = 0.0f;
#pragma unroll
  for (int k = 0; k < GROUPS; k++) {
    x += acc[k][col].x;
    y += acc[k][col].y;
  }
  const int e = p / a.tq, i = p - e * a.tq;
  const int head = kvh * a.grp + e;
  const float i1 = inverse(L1), i2 = inverse(L2), lm = L2 == 0.0f ? 0.0f : __ldg(a.lam + head);
  if (col < 2 * a.dh) {
    static_cast<T*>(a.o)[b * a.ob + head * a.oh + i * a.orow + col] = from_f<T>(x * i1 - lm * (y * i2));
    if (a.o2)
      static_cast<T*>(a.o2)[((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) + col] =
          from_f<T>(y * i2);
  }
  if (a.lse && tid == 0) {
    float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
    s[0] = log_sum(M1, L1);
    s[a.tq] = log_sum(M2, L2);
  }
}

template <class T, int W>
int join_launch(rnn_ctx* ctx, const Args& a) {
  const long long rows = static_cast<long long>(a.n) * a.h * a.tq;
  RNN_REQUIRE(rows < (1ll << 31) && a.nsplit <= JOIN_PARTS, "diffattn: too many rows or parts to join");
  join_kernel<T, W><<<static_cast<unsigned>(rows), JOIN_THREADS, 0, ctx->stream>>>(a);
  RNN_CHECK_LAUNCH();
  return RNN_OK;
}

// Joins the parts that the keys were split into, a warp for each row: the maps'
// sums meet at the larger maximum.  (The rows here are many and the parts few;
// for a token over a long cache, where it is the other way round, the parts are
// shared out over a block.)
constexpr int JOIN_WARPS = 8;
template <class T, int W>
__global__ void __launch_bounds__(JOIN_WARPS * 32) join_rows_kernel(const __grid_constant__ Args a) {
  const long long total = static_cast<long long>(a.n) * a.h * a.tq;
  const long long idx = static_cast<long long>(blockIdx.x) * JOIN_WARPS + (threadIdx.x >> 5);
  const int lane = threadIdx.x & 31;
  if (idx >= total) return;
  float M1 = -CUDART_INF_F, M2 = -CUDART_INF_F;
  for (int s = 0; s < a.nsplit; s++) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(a.stat) + s * total + idx);
    M1 = fmaxf(M1, v.x);
    M2 = fmaxf(M2, v.z);
  }
  const float U1 = M1 == -CUDART_INF_F ? 0.0f : M1, U2 = M2 == -CUDART_INF_F ? 0.0f : M2;
  float L1 = 0.0f, L2 = 0.0f;
  float4 x = make_float4(0.0f, 0.0f, 0.0f, 0.0f), y = x;
  const bool mine = lane * 4 < 2 * a.dh;
#pragma unroll 4
  for (int s = 0; s < a.nsplit; s++) {
    const float4 v = __ldg(reinterpret_cast<const float4*>(a.stat) + s * total + idx);
    const float4* part = reinterpret_cast<const float4*>(a.part + (s * total + idx) * (2 * W)) + lane;
    const float w1 = ex2(v.x - U1), w2 = ex2(v.z - U2);
    L1 += w1 * v.y;
    L2 += w2 * v.w;
    if (mine) {
      const float4 p = part[0], q = part[W / 4];
      x.x += w1 * p.x, x.y += w1 * p.y, x.z += w1 * p.z, x.w += w1 * p.w;
      y.x += w2 * q.x, y.y += w2 * q.y, y.z += w2 * q.z, y.w += w2 * q.w;
    }
  }
  const int rows = a.grp * a.tq;
  const int bh = static_cast<int>(idx / rows), r = static_cast<int>(idx - static_cast<long long>(bh) * rows);
  const int b = bh / a.hkv, e = r / a.tq, i = r - e * a.tq, head = (bh - b * a.hkv) * a.grp + e;
  const float i1 = inverse(L1), i2 = inverse(L2), f = L2 == 0.0f ? 0.0f : __ldg(a.lam + head) * i2;
  if (mine) {
    T* o = static_cast<T*>(a.o) + b * a.ob + head * a.oh + i * a.orow + lane * 4;
    const int in = 2 * a.dh - lane * 4;  // at least 2
    store2(o, x.x * i1 - f * y.x, x.y * i1 - f * y.y, true, true, a.pair);
    store2(o + 2, x.z * i1 - f * y.z, x.w * i1 - f * y.w, in > 2, in > 3, a.pair);
    if (a.o2) {
      T* o2 = static_cast<T*>(a.o2) + ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) + lane * 4;
      store2(o2, y.x * i2, y.y * i2, true, true, true);
      store2(o2 + 2, y.z * i2, y.w * i2, in > 2, in > 3, true);
    }
  }
  if (a.lse && lane < 2) {
    float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
    if (lane == 0) s[0] = log_sum(M1, L1);
    else s[a.tq] = log_sum(M2, L2);
  }
}

template <class T, int W>
int join_rows_launch(rnn_ctx* ctx, const Args& a) {
  const long long rows = static_cast<long long>(a.n) * a.h * a.tq;
  RNN_REQUIRE(rows < (1ll << 31), "diffattn: too many rows to join");
  join_rows_kernel<T, W>
      <<<static_cast<unsigned>((rows + JOIN_WARPS - 1) / JOIN_WARPS), JOIN_WARPS * 32, 0, ctx->stream>>>(a);
  RNN_CHECK_LAUNCH();
  return RNN_OK;
}

// ----------------------------------------------------------------- backward

template <class T, int DH>
struct BwdQ {
  using G = Geo<T, DH>;
  static constexpr int ROWS = 64;
  static constexpr int BN = sizeof(T) == 4 ? 32 : 64;
  static constexpr int Q_ELEMS = ROWS * G::PITCH, KV_ELEMS = BN * G::PITCH;
  static constexpr size_t TILES = (2 * Q_ELEMS + 4 * KV_ELEMS) * sizeof(T);
  static constexpr size_t SMEM = TILES + ROWS * 2 * sizeof(float) + 2 * BN;
};

// dq of 64 packed rows, and D_1 and D_2 of each for the key kernel.
template <class T, int DH>
__global__ void __launch_bounds__(THREADS) bwd_q_kernel(Args a) {
  using F = BwdQ<T, DH>;
  using G = Geo<T, DH>;
  using FR = Frag<T>;
  constexpr int W = G::W, PITCH = G::PITCH, KS = G::KS, SUB = G::SUB, BN = F::BN;
  constexpr int NS = SUB / 8, NB = W / 8, NSIDE = NS < G::SIDE ? NS : G::SIDE;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sq = reinterpret_cast<T*>(smem);
  T* sdo = sq + F::Q_ELEMS;
  T* sk = sdo + F::Q_ELEMS;
  T* sv = sk + 2 * F::KV_ELEMS;
  float* sd = reinterpret_cast<float*>(smem + F::TILES);
  uint8_t* sok = smem + F::TILES + F::ROWS * 2 * sizeof(float);

  const int rows = a.grp * a.tq;
  const int ntile = (rows + F::ROWS - 1) / F::ROWS;
  const int nbh = a.n * a.hkv;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int row0 = tile * F::ROWS;
  const int len = key_len(a, b);

  const T* qp = static_cast<const T*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + kvh * a.vh;
  const T* dop = static_cast<const T*>(a.dout) + b * a.gb + static_cast<long long>(kvh) * a.grp * a.gh;
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;

  int kend = len;
  if (a.causal) {
    const int last = min(rows, row0 + F::ROWS) - 1;
    const int imax = last / a.tq != row0 / a.tq ? a.tq - 1 : last % a.tq;
    kend = row_limit(a, imax, len);
  }
  const int ntk = kend > 0 ? (kend + BN - 1) / BN : 0;

  auto load_kv = [&](int t) {
    const int st = t & 1, j0 = t * BN;
    auto at = [&](const T* p, long long stride, int r) -> const T* {
      const int j = j0 + r;
      return j < kend && (!mask || mask[j]) ? p + j * stride : nullptr;
    };
    load_tile<T, DH, BN, THREADS, true>(sk + st * F::KV_ELEMS, kp, a.dh, a.vec,
                                        [&](int r) { return at(kp, a.kr, r); });
    load_tile<T, DH, BN, THREADS, false>(sv + st * F::KV_ELEMS, vp, a.dh, a.vec,
                                         [&](int r) { return at(vp, a.vr, r); });
    if (mask)
      for (int r = tid; r < BN; r += THREADS) sok[st * BN + r] = j0 + r < kend && mask[j0 + r];
    cp_commit();
  };
  load_tile<T, DH, F::ROWS, THREADS, true>(sq, qp, a.dh, a.vec, [&](int r) -> const T* {
    const int p = row0 + r;
    if (p >= rows) return nullptr;
    const int e = p / a.tq;
    return qp + e * a.qh + (p - e * a.tq) * a.qr;
  });
  load_tile<T, DH, F::ROWS, THREADS, false>(sdo, dop, a.dh, a.vec, [&](int r) -> const T* {
    const int p = row0 + r;
    if (p >= rows) return nullptr;
    const int e = p / a.tq;
    return dop + e * a.gh + (p - e * a.tq) * a.gr;
  });
  cp_commit();
  if (ntk > 0) load_kv(0);

  // D_1 = do . (o + lam o2) and D_2 = do . o2 of the warp's 16 rows.  Rows that see
  // one register step of keys sum P dP there instead (dS of a lone key comes out as
  // 0), and in bf16 rows of up to 128 keys, of which few share each row, sum it in a
  // pass of its own; the others follow too_far().
  const bool one_step = kend <= SUB;
  const bool own_pass = !one_step && sizeof(T) == 2 && kend <= 128;
  if (!one_step && !own_pass) {
    if (ntk > 0) {
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    // eight rows at a time, so that their loads are in flight together
#pragma unroll 1
    for (int r0 = warp * 16; r0 < warp * 16 + 16; r0 += 8) {
      float e1[8], e2[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        const int p = min(row0 + r0 + k, rows - 1);
        const int e = p / a.tq, i = p - e * a.tq;
        const int head = kvh * a.grp + e;
        const T* o = static_cast<const T*>(a.fo) + b * a.ob + head * a.oh + i * a.orow;
        const T* o2 = static_cast<const T*>(a.fo2) + ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh);
        const float lm = __ldg(a.lam + head);
        e1[k] = e2[k] = 0.0f;
#pragma unroll
        for (int c0 = 0; c0 < W; c0 += 32) {
          const int c = c0 + lane;
          const bool on = c < 2 * a.dh;
          const float g = on ? to_f<T>(sdo[(r0 + k) * PITCH + c]) : 0.0f, y = on ? to_f<T>(o2[c]) : 0.0f;
          const float x = on ? to_f<T>(o[c]) : 0.0f;
          e2[k] += g * y;
          e1[k] += g * (x + lm * y);
        }
      }
#pragma unroll
      for (int k = 0; k < 8; k++) {
#pragma unroll
        for (int x = 16; x > 0; x >>= 1) {
          e1[k] += __shfl_xor_sync(0xffffffffu, e1[k], x);
          e2[k] += __shfl_xor_sync(0xffffffffu, e2[k], x);
        }
        if (lane == 0) {
          sd[2 * (r0 + k)] = e1[k];
          sd[2 * (r0 + k) + 1] = e2[k];
        }
      }
    }
    __syncwarp();
  }

  int lim[2];
  float ls1[2], ls2[2], d1[2], d2[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    const int r = warp * 16 + (lane >> 2) + 8 * i, p = row0 + r;
    lim[i] = 0;
    ls1[i] = ls2[i] = CUDART_INF_F;
    d1[i] = d2[i] = 0.0f;
    if (p < rows) {
      const int e = p / a.tq, q = p - e * a.tq;
      const float* s = a.flse + (static_cast<long long>(b) * a.h + kvh * a.grp + e) * 2 * a.tq + q;
      lim[i] = row_limit(a, q, len);
      ls1[i] = s[0];
      ls2[i] = s[a.tq];
      if (!one_step && !own_pass) {
        d1[i] = sd[2 * r];
        d2[i] = sd[2 * r + 1];
      }
    }
  }
  const int full = __reduce_min_sync(0xffffffffu, min(lim[0], lim[1]));

  float dq[NB][4];
#pragma unroll
  for (int i = 0; i < NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) dq[i][j] = 0.0f;

  float b1[2], b2[2], sq1[2], sq2[2];  // sums of dS and of its squares
  for (int pass = own_pass ? -1 : 0;; pass++) {
    const bool sums = pass < 0;  // the pass for D alone
#pragma unroll
    for (int i = 0; i < 2; i++) b1[i] = b2[i] = sq1[i] = sq2[i] = 0.0f;
    for (int t = 0; t < ntk; t++) {
      if (t + 1 < ntk) {
        load_kv(t + 1);
        cp_wait<1>();
      } else {
        cp_wait<0>();
      }
      __syncthreads();
      const T* k = sk + (t & 1) * F::KV_ELEMS;
      const T* v = sv + (t & 1) * F::KV_ELEMS;
      const uint8_t* ok = sok + (t & 1) * BN;
      for (int s0 = 0; s0 < BN; s0 += SUB) {
        const int j0 = t * BN + s0;
        if (j0 >= kend) break;
        float s1[NS][4], s2[NS][4], dp[NS][4], m1[NS][4] = {}, m2[NS][4] = {}, mp[NS][4] = {};
#pragma unroll
        for (int i = 0; i < NS; i++)
#pragma unroll
          for (int j = 0; j < 4; j++) s1[i][j] = s2[i][j] = dp[i][j] = 0.0f;
#pragma unroll
        for (int ks = 0; ks < DH / KS; ks++) {
          const typename FR::A q1 = FR::ldA(sq, PITCH, warp * 16, ks * KS, lane);
          const typename FR::A q2 = FR::ldA(sq, PITCH, warp * 16, DH + ks * KS, lane);
#pragma unroll
          for (int nb = 0; nb < NS; nb += NSIDE) {
            typename FR::B f[NSIDE], g[NSIDE];
            FR::ldB_nk(f, k, PITCH, s0 + nb * 8, ks * KS, lane);
            FR::ldB_nk(g, k, PITCH, s0 + nb * 8, DH + ks * KS, lane);
            FR::mma(s1 + nb, m1 + nb, q1, f);
            FR::mma(s2 + nb, m2 + nb, q2, g);
          }
        }
#pragma unroll
        for (int ks = 0; ks < W / KS; ks++) {
          const typename FR::A g = FR::ldA(sdo, PITCH, warp * 16, ks * KS, lane);
#pragma unroll
          for (int nb = 0; nb < NS; nb += NSIDE) {
            typename FR::B f[NSIDE];
            FR::ldB_nk(f, v, PITCH, s0 + nb * 8, ks * KS, lane);
            FR::mma(dp + nb, mp + nb, g, f);
          }
        }
        FR::join(s1, m1);
        FR::join(s2, m2);
        FR::join(dp, mp);
        const bool edge = mask != nullptr || j0 + SUB > full;
#pragma unroll
        for (int nb = 0; nb < NS; nb++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float x = ex2(s1[nb][e] * a.slog2 - ls1[e >> 1]), y = ex2(s2[nb][e] * a.slog2 - ls2[e >> 1]);
            if (edge) {
              const int c = nb * 8 + 2 * (lane & 3) + (e & 1);
              if (j0 + c >= lim[e >> 1] || (mask && !ok[s0 + c])) x = y = 0.0f;
            }
            s1[nb][e] = x;
            s2[nb][e] = y;
            if (sums) {
              d1[e >> 1] += x * dp[nb][e];
              d2[e >> 1] += y * dp[nb][e];
            }
          }
        if (sums) continue;
        if (one_step) {
#pragma unroll
          for (int i = 0; i < 2; i++) {
            float x = 0.0f, y = 0.0f;
#pragma unroll
            for (int nb = 0; nb < NS; nb++) {
              x += s1[nb][2 * i] * dp[nb][2 * i] + s1[nb][2 * i + 1] * dp[nb][2 * i + 1];
              y += s2[nb][2 * i] * dp[nb][2 * i] + s2[nb][2 * i + 1] * dp[nb][2 * i + 1];
            }
            d1[i] = quad_sum(x);
            d2[i] = quad_sum(y);
          }
        }
#pragma unroll
        for (int nb = 0; nb < NS; nb++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            const int i = e >> 1;
            const float x = s1[nb][e] * (dp[nb][e] - d1[i]), y = s2[nb][e] * (dp[nb][e] - d2[i]);
            s1[nb][e] = x;
            s2[nb][e] = y;
            b1[i] += x;
            b2[i] += y;
            if (sizeof(T) == 2) {
              sq1[i] += x * x;
              sq2[i] += y * y;
            }
          }
#pragma unroll
        for (int m = 0; m < 2; m++) {
          typename FR::A ds[SUB / KS];
#pragma unroll
          for (int ks = 0; ks < SUB / KS; ks++) ds[ks] = m ? FR::from_acc(s2, ks) : FR::from_acc(s1, ks);
#pragma unroll
          for (int nb = m * NB / 2; nb < (m + 1) * NB / 2; nb += G::HALF_SIDE) {
            float x[G::HALF_SIDE][4] = {}, xs[G::HALF_SIDE][4] = {};
#pragma unroll
            for (int ks = 0; ks < SUB / KS; ks++) {
              typename FR::B f[G::HALF_SIDE];
              FR::ldB_kn(f, k, PITCH, s0 + ks * KS, nb * 8, lane);
              FR::mma(x, xs, ds[ks], f);
            }
            FR::join(x, xs);
#pragma unroll
            for (int i = 0; i < G::HALF_SIDE; i++)
#pragma unroll
              for (int e = 0; e < 4; e++) dq[nb + i][e] += x[i][e];
          }
        }
      }
      __syncthreads();
    }
    bool far = false;
#pragma unroll
    for (int i = 0; i < 2; i++) {
      if (sums) {
        d1[i] = quad_sum(d1[i]);
        d2[i] = quad_sum(d2[i]);
        continue;
      }
      b1[i] = quad_sum(b1[i]);
      b2[i] = quad_sum(b2[i]);
      sq1[i] = quad_sum(sq1[i]);  // all lanes take part, so not within the condition
      sq2[i] = quad_sum(sq2[i]);
      far |= too_far(b1[i], sq1[i]) || too_far(b2[i], sq2[i]);
      // a map that has no key has no D either
      d1[i] = ls1[i] == CUDART_INF_F ? 0.0f : d1[i] + b1[i];
      d2[i] = ls2[i] == CUDART_INF_F ? 0.0f : d2[i] + b2[i];
    }
    if (!sums && (sizeof(T) == 4 || one_step || own_pass || pass > 0 || !__syncthreads_or(far))) break;
#pragma unroll
    for (int i = 0; i < NB; i++)
#pragma unroll
      for (int j = 0; j < 4; j++) dq[i][j] = 0.0f;
    if (ntk > 0) load_kv(0);
  }
  cp_wait<0>();

#pragma unroll
  for (int h = 0; h < 2; h++) {
    const int p = row0 + warp * 16 + (lane >> 2) + 8 * h;
    if (p >= rows) continue;
    const int e = p / a.tq, i = p - e * a.tq;
    const int head = kvh * a.grp + e;
    if ((lane & 3) == 0) {
      float* s = a.dsum + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
      s[0] = d1[h];
      s[a.tq] = d2[h];
      a.dlrow[static_cast<long long>(head) * a.n * a.tq + static_cast<long long>(b) * a.tq + i] = d2[h];
    }
    const float f1 = a.scale, f2 = -a.scale * __ldg(a.lam + head);
    T* o = static_cast<T*>(a.dq) + b * a.dqb + head * a.dqh + i * a.dqr;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int half = nb >= NB / 2 ? 1 : 0;
      const int w = nb * 8 - half * DH + 2 * (lane & 3);
      const float f = half ? f2 : f1;
      store2(o + half * a.dh + w, dq[nb][2 * h] * f, dq[nb][2 * h + 1] * f, w < a.dh, w + 1 < a.dh, a.pair);
    }
  }
}

template <class T, int DH>
struct BwdKV {
  using G = Geo<T, DH>;
  static constexpr int KEYS = 64;
  static constexpr int BM = 32;  // queries per stage
  static constexpr int K_ELEMS = KEYS * G::PITCH, Q_ELEMS = BM * G::PITCH;
  static constexpr size_t TILES = (2 * K_ELEMS + 4 * Q_ELEMS) * sizeof(T);
  static constexpr size_t SMEM = TILES + 2 * BM * 5 * sizeof(float);  // + lse_1, lse_2, D_1, D_2, limit per query
};

// dk and dv of 64 keys: loops over the queries of the group's heads.  The
// transposed maps (keys x queries) come from k q^T and v do^T, so that keys
// stay in the accumulators' rows.
template <class T, int DH>
__global__ void __launch_bounds__(THREADS) bwd_kv_kernel(Args a) {
  using F = BwdKV<T, DH>;
  using G = Geo<T, DH>;
  using FR = Frag<T>;
  constexpr int W = G::W, PITCH = G::PITCH, KS = G::KS, SUB = G::SUB, BM = F::BM;
  constexpr int NS = SUB / 8, NB = W / 8, NSIDE = NS < G::SIDE ? NS : G::SIDE;
  extern __shared__ __align__(16) unsigned char smem[];
  T* sk = reinterpret_cast<T*>(smem);
  T* sv = sk + F::K_ELEMS;
  T* sq = sv + F::K_ELEMS;
  T* sdo = sq + 2 * F::Q_ELEMS;
  float* sst = reinterpret_cast<float*>(smem + F::TILES);

  const int nbh = a.n * a.hkv;
  const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;

  // dlam: block `head` sums that head's rows in a fixed order, if there are any
  if (static_cast<int>(blockIdx.x) < a.h && a.tq > 0) {
    const int head = blockIdx.x;
    const long long cnt = static_cast<long long>(a.n) * a.tq;
    const float* x = a.dlrow + head * cnt;
    double s = 0.0;
    for (long long i = tid; i < cnt; i += THREADS) s += x[i];
    double* red = reinterpret_cast<double*>(smem);
    red[tid] = s;
    __syncthreads();
    for (int o = THREADS / 2; o > 0; o >>= 1) {
      if (tid < o) red[tid] += red[tid + o];
      __syncthreads();
    }
    if (tid == 0) a.dlam[head] -= static_cast<float>(red[0]);
    __syncthreads();
  }
  const int nkt = (a.tk + F::KEYS - 1) / F::KEYS;
  if (static_cast<int>(blockIdx.x) >= nkt * nbh) return;  // a block for dlam only
  const int kt = static_cast<int>(blockIdx.x) / nbh;      // the earliest keys, which most queries see, first
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int key0 = kt * F::KEYS;
  const int len = key_len(a, b);

  const T* qp = static_cast<const T*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
  const T* kp = static_cast<const T*>(a.k) + b * a.kb + kvh * a.kh;
  const T* vp = static_cast<const T*>(a.v) + b * a.vb + kvh * a.vh;
  const T* dop = static_cast<const T*>(a.dout) + b * a.gb + static_cast<long long>(kvh) * a.grp * a.gh;
  const uint8_t* mask = a.kmask ? a.kmask + b * a.kmb : nullptr;

  // queries before `qbeg` see none of these keys
  int qbeg = 0;
  if (key0 >= len) {
    qbeg = a.tq;
  } else if (a.causal == RNN_CAUSAL_START) {
    qbeg = min(a.tq, key0);
  } else if (a.causal == RNN_CAUSAL_END) {
    qbeg = min(a.tq, max(0, key0 - (len - a.tq)));
  }
  const int per = (a.tq - qbeg + BM - 1) / BM, nt = per * a.grp;

  auto load_q = [&](int t) {
    const int st = t & 1, e = t / per, i0 = qbeg + (t - e * per) * BM;
    load_tile<T, DH, BM, THREADS, true>(sq + st * F::Q_ELEMS, qp, a.dh, a.vec, [&](int r) -> const T* {
      return i0 + r < a.tq ? qp + e * a.qh + (i0 + r) * a.qr : nullptr;
    });
    load_tile<T, DH, BM, THREADS, false>(sdo + st * F::Q_ELEMS, dop, a.dh, a.vec, [&](int r) -> const T* {
      return i0 + r < a.tq ? dop + e * a.gh + (i0 + r) * a.gr : nullptr;
    });
    if (tid < BM) {
      float* s = sst + st * 5 * BM + tid;
      const int i = i0 + tid;
      const bool in = i < a.tq;
      const long long at = (static_cast<long long>(b) * a.h + kvh * a.grp + e) * 2 * a.tq + i;
      s[0] = in ? a.flse[at] : CUDART_INF_F;
      s[BM] = in ? a.flse[at + a.tq] : CUDART_INF_F;
      s[2 * BM] = in ? a.dsum[at] : 0.0f;
      s[3 * BM] = in ? a.dsum[at + a.tq] : 0.0f;
      s[4 * BM] = __int_as_float(in ? row_limit(a, i, len) : 0);
    }
    cp_commit();
  };

  float dk[NB][4], dv[NB][4];
#pragma unroll
  for (int i = 0; i < NB; i++)
#pragma unroll
    for (int j = 0; j < 4; j++) dk[i][j] = dv[i][j] = 0.0f;

  int key[2];
  bool seen[2];
#pragma unroll
  for (int i = 0; i < 2; i++) {
    key[i] = key0 + warp * 16 + (lane >> 2) + 8 * i;
    seen[i] = key[i] < len && (!mask || mask[key[i]]);
  }
  if (nt > 0) {
    auto at = [&](const T* p, long long stride, int r) -> const T* {
      const int j = key0 + r;
      return j < len && (!mask || mask[j]) ? p + j * stride : nullptr;
    };
    load_tile<T, DH, F::KEYS, THREADS, true>(sk, kp, a.dh, a.vec, [&](int r) { return at(kp, a.kr, r); });
    load_tile<T, DH, F::KEYS, THREADS, false>(sv, vp, a.dh, a.vec, [&](int r) { return at(vp, a.vr, r); });
    load_q(0);
  }
  for (int t = 0; t < nt; t++) {
    if (t + 1 < nt) {
      load_q(t + 1);
      cp_wait<1>();
    } else {
      cp_wait<0>();
    }
    __syncthreads();
    const T* q = sq + (t & 1) * F::Q_ELEMS;
    const T* g = sdo + (t & 1) * F::Q_ELEMS;
    const float* st = sst + (t & 1) * 5 * BM;
    const float lam = __ldg(a.lam + kvh * a.grp + t / per);
    for (int s0 = 0; s0 < BM; s0 += SUB) {
      float s1[NS][4], s2[NS][4], dp[NS][4], m1[NS][4] = {}, m2[NS][4] = {}, mp[NS][4] = {};
#pragma unroll
      for (int i = 0; i < NS; i++)
#pragma unroll
        for (int j = 0; j < 4; j++) s1[i][j] = s2[i][j] = dp[i][j] = 0.0f;
#pragma unroll
      for (int ks = 0; ks < DH / KS; ks++) {
        const typename FR::A k1 = FR::ldA(sk, PITCH, warp * 16, ks * KS, lane);
        const typename FR::A k2 = FR::ldA(sk, PITCH, warp * 16, DH + ks * KS, lane);
#pragma unroll
        for (int nb = 0; nb < NS; nb += NSIDE) {
          typename FR::B f[NSIDE], h[NSIDE];
          FR::ldB_nk(f, q, PITCH, s0 + nb * 8, ks * KS, lane);
          FR::ldB_nk(h, q, PITCH, s0 + nb * 8, DH + ks * KS, lane);
          FR::mma(s1 + nb, m1 + nb, k1, f);
          FR::mma(s2 + nb, m2 + nb, k2, h);
        }
      }
#pragma unroll
      for (int ks = 0; ks < W / KS; ks++) {
        const typename FR::A x = FR::ldA(sv, PITCH, warp * 16, ks * KS, lane);
#pragma unroll
        for (int nb = 0; nb < NS; nb += NSIDE) {
          typename FR::B f[NSIDE];
          FR::ldB_nk(f, g, PITCH, s0 + nb * 8, ks * KS, lane);
          FR::mma(dp + nb, mp + nb, x, f);
        }
      }
      FR::join(s1, m1);
      FR::join(s2, m2);
      FR::join(dp, mp);
      // after this: s1 = dS_1, s2 = dS_2, dp = P_1 - lam P_2 (transposed)
#pragma unroll
      for (int nb = 0; nb < NS; nb++)
#pragma unroll
        for (int e = 0; e < 4; e++) {
          const int c = s0 + nb * 8 + 2 * (lane & 3) + (e & 1);
          const bool on = seen[e >> 1] && key[e >> 1] < __float_as_int(st[4 * BM + c]);
          const float x = on ? ex2(s1[nb][e] * a.slog2 - st[c]) : 0.0f;
          const float y = on ? lam * ex2(s2[nb][e] * a.slog2 - st[BM + c]) : 0.0f;
          s1[nb][e] = x * (dp[nb][e] - st[2 * BM + c]);
          s2[nb][e] = -y * (dp[nb][e] - st[3 * BM + c]);
          dp[nb][e] = x - y;
        }
#pragma unroll
      for (int m = 0; m < 3; m++) {
        typename FR::A f[SUB / KS];
#pragma unroll
        for (int ks = 0; ks < SUB / KS; ks++)
          f[ks] = m == 0 ? FR::from_acc(s1, ks) : m == 1 ? FR::from_acc(s2, ks) : FR::from_acc(dp, ks);
        const T* src = m == 2 ? g : q;
#pragma unroll
        for (int nb = (m == 1 ? NB / 2 : 0); nb < (m == 0 ? NB / 2 : NB); nb += G::HALF_SIDE) {
          float x[G::HALF_SIDE][4] = {}, xs[G::HALF_SIDE][4] = {};
#pragma unroll
          for (int ks = 0; ks < SUB / KS; ks++) {
            typename FR::B w[G::HALF_SIDE];
            FR::ldB_kn(w, src, PITCH, s0 + ks * KS, nb * 8, lane);
            FR::mma(x, xs, f[ks], w);
          }
          FR::join(x, xs);
#pragma unroll
          for (int i = 0; i < G::HALF_SIDE; i++)
#pragma unroll
            for (int e = 0; e < 4; e++) {
              if (m == 2) {
                dv[nb + i][e] += x[i][e];
              } else {
                dk[nb + i][e] += x[i][e];
              }
            }
        }
      }
    }
    __syncthreads();
  }
#pragma unroll
  for (int h = 0; h < 2; h++) {
    if (key[h] >= a.tk) continue;
    if (!seen[h]) {  // 0, whatever a query's NaN made of 0 times it
#pragma unroll
      for (int nb = 0; nb < NB; nb++) dk[nb][2 * h] = dk[nb][2 * h + 1] = dv[nb][2 * h] = dv[nb][2 * h + 1] = 0.0f;
    }
    T* ok = static_cast<T*>(a.dk) + b * a.dkb + kvh * a.dkh + key[h] * a.dkr;
    T* ov = static_cast<T*>(a.dv) + b * a.dvb + kvh * a.dvh + key[h] * a.dvr;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
      const int half = nb >= NB / 2 ? 1 : 0;
      const int c = nb * 8 + 2 * (lane & 3), w = c - half * DH;
      store2(ok + half * a.dh + w, dk[nb][2 * h] * a.scale, dk[nb][2 * h + 1] * a.scale, w < a.dh, w + 1 < a.dh,
             a.pair);
      store2(ov + c, dv[nb][2 * h], dv[nb][2 * h + 1], c < 2 * a.dh, c + 1 < 2 * a.dh, a.pair);
    }
  }
}

// --------------------------------------------------------------------- host

template <class T, int DH, int RW>
int fwd_launch(rnn_ctx* ctx, Args a) {
  using F = Fwd<T, DH, RW>;
  const long long rows = static_cast<long long>(a.grp) * a.tq;
  const long long nbh = static_cast<long long>(a.n) * a.hkv;
  const long long blocks = (rows + F::ROWS - 1) / F::ROWS * nbh;
  RNN_REQUIRE(blocks < (1ll << 31), "diffattn: too many rows");
  static std::atomic<unsigned long long> optin{0};
  RNN_TRY(tc::ensure_smem_optin(fwd_kernel<T, DH, RW>, optin, ctx->device, static_cast<int>(F::SMEM)));
  // Split the keys when the rows alone do not give every SM a block: in parts of
  // at least four tiles, or for a token's few rows of one (one row and 777 keys
  // in f32, two sequences of 4 heads: 10.9 us with parts of a tile, 16.0 of two,
  // 21.6 of four).
  static std::atomic<int> resident{0};  // blocks of this kernel an SM holds (every device here is the same part)
  int per_sm = resident.load(std::memory_order_relaxed);
  if (per_sm == 0) {
    RNN_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&per_sm, fwd_kernel<T, DH, RW>, THREADS, F::SMEM));
    resident.store(per_sm, std::memory_order_relaxed);
  }
  const long long slots = static_cast<long long>(ctx->num_sms) * std::max(1, per_sm);
  const int tiles = (a.tk + F::BN - 1) / F::BN;
  long long ns = std::min<long long>(slots / std::max(1ll, blocks), RW == 1 ? tiles : tiles / 4);
  a.nsplit = static_cast<int>(std::max(1ll, ns));
  a.split_keys = (tiles + a.nsplit - 1) / a.nsplit * F::BN;
  a.nsplit = std::max(1, (a.tk + a.split_keys - 1) / std::max(1, a.split_keys));
  if (a.nsplit > 1) {
    const size_t part = static_cast<size_t>(a.nsplit) * nbh * rows * 2 * F::G::W * sizeof(float);
    const size_t stat = static_cast<size_t>(a.nsplit) * nbh * rows * 4 * sizeof(float);
    RNN_TRY(ensure_ws(ctx, part + stat));
    a.part = static_cast<float*>(ctx->ws);
    a.stat = a.part + part / sizeof(float);
  }
  fwd_kernel<T, DH, RW><<<dim3(static_cast<unsigned>(blocks), a.nsplit), THREADS, F::SMEM, ctx->stream>>>(a);
  RNN_CHECK_LAUNCH();
  return a.nsplit > 1 ? join_launch<T, F::G::W>(ctx, a) : RNN_OK;
}

template <class T, int DH>
int fwd_dh(rnn_ctx* ctx, const Args& a) {
  return static_cast<long long>(a.grp) * a.tq <= 16 ? fwd_launch<T, DH, 1>(ctx, a) : fwd_launch<T, DH, 4>(ctx, a);
}

template <class T>
int fwd_type(rnn_ctx* ctx, const Args& a) {
  if (a.dh <= 16) return fwd_dh<T, 16>(ctx, a);
  if (a.dh <= 32) return fwd_dh<T, 32>(ctx, a);
  return fwd_dh<T, 64>(ctx, a);
}

template <class T, int DH>
int bwd_launch(rnn_ctx* ctx, Args a) {
  using FQ = BwdQ<T, DH>;
  using FK = BwdKV<T, DH>;
  const long long rows = static_cast<long long>(a.grp) * a.tq, nbh = static_cast<long long>(a.n) * a.hkv;
  const long long qblocks = (rows + FQ::ROWS - 1) / FQ::ROWS * nbh;
  const long long kblocks = std::max<long long>((a.tk + FK::KEYS - 1ll) / FK::KEYS * nbh, a.h);
  RNN_REQUIRE(qblocks < (1ll << 31) && kblocks < (1ll << 31), "diffattn: too many rows");
  static std::atomic<unsigned long long> optin_q{0}, optin_kv{0};
  RNN_TRY(tc::ensure_smem_optin(bwd_q_kernel<T, DH>, optin_q, ctx->device, static_cast<int>(FQ::SMEM)));
  RNN_TRY(tc::ensure_smem_optin(bwd_kv_kernel<T, DH>, optin_kv, ctx->device, static_cast<int>(FK::SMEM)));
  if (qblocks > 0) {
    bwd_q_kernel<T, DH><<<static_cast<unsigned>(qblocks), THREADS, FQ::SMEM, ctx->stream>>>(a);
    RNN_CHECK_LAUNCH();
  }
  bwd_kv_kernel<T, DH><<<static_cast<unsigned>(kblocks), THREADS, FK::SMEM, ctx->stream>>>(a);
  RNN_CHECK_LAUNCH();
  return RNN_OK;
}

template <class T>
int bwd_type(rnn_ctx* ctx, const Args& a) {
  if (a.dh <= 16) return bwd_launch<T, 16>(ctx, a);
  if (a.dh <= 32) return bwd_launch<T, 32>(ctx, a);
  return bwd_launch<T, 64>(ctx, a);
}

// Extent in elements of a [n, t, heads, cols] view, 0 when it is empty.
size_t extent(int n, int t, int heads, long long sb, long long sr, long long sh, int cols) {
  if (n == 0 || t == 0 || heads == 0) return 0;
  return static_cast<size_t>((n - 1) * sb + (t - 1) * sr + (heads - 1) * sh + cols);
}

// Whether no two (sequence, row, head) of a written view share an element:
// sorted by stride, each step has to clear what the smaller ones span.
bool disjoint(int n, int t, int heads, long long sb, long long sr, long long sh, int cols) {
  if (n == 0 || t == 0 || heads == 0) return true;
  std::pair<long long, int> d[3] = {{sb, n}, {sr, t}, {sh, heads}};
  std::sort(d, d + 3);
  long long span = cols;
  for (auto& x : d) {
    if (x.second <= 1) continue;
    if (x.first < span) return false;
    span += x.first * (x.second - 1ll);
  }
  return true;
}

// Checks a call and fills the kernels' arguments.
int fill(rnn_ctx* ctx, const rnn_diffattn* d, const void* q, const void* k, const void* v, const float* lambda,
         const void* o, Args& a) {
  RNN_REQUIRE(ctx != nullptr, "null context");
  RNN_REQUIRE(d != nullptr, "diffattn: null description");
  RNN_REQUIRE(d->dtype == RNN_F32 || d->dtype == RNN_BF16, "diffattn: unknown dtype %d", d->dtype);
  RNN_REQUIRE(d->causal >= RNN_CAUSAL_NONE && d->causal <= RNN_CAUSAL_END, "diffattn: unknown causal mode %d",
              d->causal);
  RNN_REQUIRE(d->n >= 0 && d->tq >= 0 && d->tk >= 0 && d->h >= 1 && d->hkv >= 1 && d->h % d->hkv == 0,
              "diffattn: bad shape n=%d tq=%d tk=%d h=%d hkv=%d", d->n, d->tq, d->tk, d->h, d->hkv);
  RNN_REQUIRE(d->dh >= 1, "diffattn: dh=%d", d->dh);
  if (d->dh > 64) return set_error(RNN_ERR_UNSUPPORTED, "diffattn: dh=%d, at most 64 columns a half", d->dh);
  // the kernels count a (sequence, key head)'s rows in int, to the end of a block of up to 128
  RNN_REQUIRE(d->n * (long long)d->hkv < (1ll << 31) && d->tk < (1 << 30) && d->tq < (1 << 30) &&
                  (long long)(d->h / d->hkv) * d->tq < (1ll << 31) - 128,
              "diffattn: shape too large");
  RNN_REQUIRE(d->q_batch >= 0 && d->q_row >= 0 && d->q_head >= 0 && d->k_batch >= 0 && d->k_row >= 0 &&
                  d->k_head >= 0 && d->v_batch >= 0 && d->v_row >= 0 && d->v_head >= 0 && d->o_batch >= 0 &&
                  d->o_row >= 0 && d->o_head >= 0 && d->kmask_batch >= 0,
              "diffattn: negative stride");
  const int w = 2 * d->dh;
  const size_t esz = d->dtype == RNN_F32 ? 4 : 2;
  const bool rows = d->n > 0 && d->tq > 0, keys = d->n > 0 && d->tk > 0;
  RNN_REQUIRE(!rows || (q != nullptr && o != nullptr && lambda != nullptr), "diffattn: null pointer");
  RNN_REQUIRE(!keys || (k != nullptr && v != nullptr), "diffattn: null pointer");
  for (const void* p : {q, k, v, o})
    RNN_REQUIRE(reinterpret_cast<uintptr_t>(p) % esz == 0, "diffattn: misaligned pointer");
  RNN_REQUIRE(reinterpret_cast<uintptr_t>(lambda) % 4 == 0 && reinterpret_cast<uintptr_t>(d->klen) % 4 == 0,
              "diffattn: misaligned pointer");
  RNN_RANGE(q, extent(d->n, d->tq, d->h, d->q_batch, d->q_row, d->q_head, w) * esz);
  RNN_RANGE(k, extent(d->n, d->tk, d->hkv, d->k_batch, d->k_row, d->k_head, w) * esz);
  RNN_RANGE(v, extent(d->n, d->tk, d->hkv, d->v_batch, d->v_row, d->v_head, w) * esz);
  RNN_RANGE(o, extent(d->n, d->tq, d->h, d->o_batch, d->o_row, d->o_head, w) * esz);
  if (rows) RNN_RANGE(lambda, d->h * sizeof(float));
  if (d->klen) RNN_RANGE(d->klen, d->n * sizeof(int));
  if (d->kmask && keys) RNN_RANGE(d->kmask, (size_t)((d->n - 1) * d->kmask_batch + d->tk));
  a = Args{};
  a.n = d->n, a.h = d->h, a.hkv = d->hkv, a.grp = d->h / d->hkv, a.dh = d->dh;
  a.tq = d->tq, a.tk = d->tk, a.causal = d->causal;
  a.scale = d->scale;
  a.slog2 = d->scale * 1.4426950408889634f;
  a.qb = d->q_batch, a.qr = d->q_row, a.qh = d->q_head;
  a.kb = d->k_batch, a.kr = d->k_row, a.kh = d->k_head;
  a.vb = d->v_batch, a.vr = d->v_row, a.vh = d->v_head;
  a.ob = d->o_batch, a.orow = d->o_row, a.oh = d->o_head;
  // the stride of an axis of one element is never used: 0 keeps it out of the alignment rules
  if (a.n <= 1) a.qb = a.kb = a.vb = a.ob = 0;
  if (a.tq <= 1) a.qr = a.orow = 0;
  if (a.tk <= 1) a.kr = a.vr = 0;
  if (a.h <= 1) a.qh = a.oh = 0;
  if (a.hkv <= 1) a.kh = a.vh = 0;
  a.q = q, a.k = k, a.v = v, a.lam = lambda;
  a.klen = d->klen, a.kmask = d->kmask, a.kmb = d->kmask_batch;
  a.nsplit = 1;
  return RNN_OK;
}

// Whether all strides are multiples of e elements.
bool multiples(std::initializer_list<long long> s, long long e) {
  for (long long x : s)
    if (x % e) return false;
  return true;
}
bool aligned(std::initializer_list<const void*> ps, size_t bytes) {
  for (const void* p : ps)
    if (reinterpret_cast<uintptr_t>(p) % bytes) return false;
  return true;
}

}  // namespace

int join_parts(rnn_ctx* ctx, const Args& a) { return join_launch<__nv_bfloat16, 128>(ctx, a); }
int join_rows_bf16(rnn_ctx* ctx, const Args& a) { return join_rows_launch<__nv_bfloat16, 128>(ctx, a); }
int join_rows_f32(rnn_ctx* ctx, const Args& a) { return join_rows_launch<float, 64>(ctx, a); }
int join_rows_f32_wide(rnn_ctx* ctx, const Args& a) { return join_rows_launch<float, 128>(ctx, a); }

}  // namespace diff
}  // namespace rnn

using namespace rnn;

extern "C" int rnn_diffattn_fwd_dev(rnn_ctx* ctx, const rnn_diffattn* d, const void* q, const void* k, const void* v,
                                    const float* lambda, void* o, void* o2, float* lse) {
  diff::Args a;
  RNN_TRY(diff::fill(ctx, d, q, k, v, lambda, o, a));
  RNN_REQUIRE((o2 == nullptr) == (lse == nullptr), "diffattn: o2 and lse are written both or neither");
  RNN_REQUIRE(diff::disjoint(a.n, a.tq, a.h, a.ob, a.orow, a.oh, 2 * a.dh), "diffattn: output rows or heads overlap");
  if (a.n == 0 || a.tq == 0) return RNN_OK;
  const size_t esz = d->dtype == RNN_F32 ? 4 : 2;
  const size_t nrow = (size_t)a.n * a.h * a.tq;
  if (o2) {
    RNN_REQUIRE(diff::aligned({o2}, 2 * esz) && diff::aligned({lse}, 4), "diffattn: misaligned pointer");
    RNN_RANGE(o2, nrow * 2 * a.dh * esz);
    RNN_RANGE(lse, nrow * 2 * sizeof(float));
  }
  a.o = o, a.o2 = o2, a.lse = lse;
  a.vec = a.dh % (16 / esz) == 0 && diff::aligned({q, k, v}, 16) &&
          diff::multiples({a.qb, a.qr, a.qh, a.kb, a.kr, a.kh, a.vb, a.vr, a.vh}, 16 / esz);
  a.pair = diff::multiples({a.ob, a.orow, a.oh}, 2) && diff::aligned({o}, 2 * esz);
  if (d->dtype == RNN_F32) return diff::f32_tc_ok(a, false) ? diff::f32_tc_fwd(ctx, a) : diff::fwd_type<float>(ctx, a);
  if (diff::dec_ok(a)) return diff::dec_fwd(ctx, a);
  return diff::tc_fwd_ok(a) ? diff::tc_fwd(ctx, a) : diff::fwd_type<__nv_bfloat16>(ctx, a);
}

extern "C" int rnn_diffattn_bwd_dev(rnn_ctx* ctx, const rnn_diffattn* d, const rnn_diffattn* g, const void* q,
                                    const void* k, const void* v, const float* lambda, const void* o, const void* o2, const float* lse,
                                    const void* dout, void* dq, void* dk, void* dv, float* dlambda) {
  diff::Args a;
  RNN_TRY(diff::fill(ctx, d, q, k, v, lambda, o, a));
  if (g == nullptr) g = d;
  RNN_REQUIRE(g->q_batch >= 0 && g->q_row >= 0 && g->q_head >= 0 && g->k_batch >= 0 && g->k_row >= 0 &&
                  g->k_head >= 0 && g->v_batch >= 0 && g->v_row >= 0 && g->v_head >= 0 && g->o_batch >= 0 &&
                  g->o_row >= 0 && g->o_head >= 0,
              "diffattn: negative stride");
  auto of = [](int count, long long stride) { return count <= 1 ? 0 : stride; };
  a.dqb = of(a.n, g->q_batch), a.dqr = of(a.tq, g->q_row), a.dqh = of(a.h, g->q_head);
  a.dkb = of(a.n, g->k_batch), a.dkr = of(a.tk, g->k_row), a.dkh = of(a.hkv, g->k_head);
  a.dvb = of(a.n, g->v_batch), a.dvr = of(a.tk, g->v_row), a.dvh = of(a.hkv, g->v_head);
  a.gb = of(a.n, g->o_batch), a.gr = of(a.tq, g->o_row), a.gh = of(a.h, g->o_head);
  RNN_REQUIRE(diff::disjoint(a.n, a.tq, a.h, a.dqb, a.dqr, a.dqh, 2 * a.dh) &&
                  diff::disjoint(a.n, a.tk, a.hkv, a.dkb, a.dkr, a.dkh, 2 * a.dh) &&
                  diff::disjoint(a.n, a.tk, a.hkv, a.dvb, a.dvr, a.dvh, 2 * a.dh),
              "diffattn: gradient rows or heads overlap");
  const bool rows = a.n > 0 && a.tq > 0, keys = a.n > 0 && a.tk > 0;
  if (!rows && !keys) return RNN_OK;
  const size_t esz = d->dtype == RNN_F32 ? 4 : 2;
  const size_t nrow = (size_t)a.n * a.h * a.tq;
  RNN_REQUIRE(!rows || (o2 && lse && dout && dq && dlambda), "diffattn: null pointer");
  RNN_REQUIRE(!keys || (dk && dv), "diffattn: null pointer");
  RNN_REQUIRE(diff::aligned({o2, dout, dq, dk, dv}, esz) && diff::aligned({lse, dlambda}, 4),
              "diffattn: misaligned pointer");
  const int w = 2 * a.dh;
  RNN_RANGE(dq, diff::extent(a.n, a.tq, a.h, a.dqb, a.dqr, a.dqh, w) * esz);
  RNN_RANGE(dk, diff::extent(a.n, a.tk, a.hkv, a.dkb, a.dkr, a.dkh, w) * esz);
  RNN_RANGE(dv, diff::extent(a.n, a.tk, a.hkv, a.dvb, a.dvr, a.dvh, w) * esz);
  RNN_RANGE(dout, diff::extent(a.n, a.tq, a.h, a.gb, a.gr, a.gh, w) * esz);
  RNN_RANGE(o2, nrow * w * esz);
  RNN_RANGE(lse, nrow * 2 * sizeof(float));
  if (rows) RNN_RANGE(dlambda, a.h * sizeof(float));
  a.fo = o, a.fo2 = o2, a.flse = lse, a.dout = dout;
  a.dq = dq, a.dk = dk, a.dv = dv, a.dlam = dlambda;
  a.vec = a.dh % (16 / esz) == 0 && diff::aligned({q, k, v, dout}, 16) &&
          diff::multiples({a.qb, a.qr, a.qh, a.kb, a.kr, a.kh, a.vb, a.vr, a.vh, a.gb, a.gr, a.gh}, 16 / esz);
  a.pair = a.dh % 2 == 0 && diff::aligned({dq, dk, dv}, 2 * esz) &&
           diff::multiples({a.dqb, a.dqr, a.dqh, a.dkb, a.dkr, a.dkh, a.dvb, a.dvr, a.dvh}, 2);
  const bool tensor = d->dtype == RNN_BF16 && diff::tc_bwd_ok(a);
  a.kparts = tensor ? diff::tc_bwd_parts(ctx, a) : 1;
  const size_t sums = (nrow * 3 + 3) / 4 * 4, keep = a.kparts > 1 ? (size_t)a.kparts * a.n * a.hkv * a.tk * 256 : 0;
  RNN_TRY(ensure_ws(ctx, (sums + keep) * sizeof(float)));
  a.dsum = static_cast<float*>(ctx->ws);
  a.dlrow = a.dsum + 2 * nrow;
  a.kpart = a.dsum + sums;
  if (tensor) return diff::tc_bwd(ctx, a);
  if (d->dtype == RNN_F32) return diff::f32_tc_ok(a, true) ? diff::f32_tc_bwd(ctx, a) : diff::bwd_type<float>(ctx, a);
  return diff::bwd_type<__nv_bfloat16>(ctx, a);
}
