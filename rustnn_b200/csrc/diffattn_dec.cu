// Differential attention of a few new tokens over a long cache: bf16, at most
// 16 packed rows (query heads of a key head x new tokens).
//
// The call is a read of the cache, so the kernel is laid out around it: tiles
// of 64 keys come by tensor copies, three stages deep, two blocks an SM (190 KB
// in flight), and a block's four warps take 16 keys of each tile.  The products
// are turned round, keys and value columns as the MMA's 16 rows, the packed
// rows as its 8 columns:
//   S_m^T = k_m q_m^T,   A^T += v^T (P_1 - r P_2)^T,   B^T += v^T P_2^T,
// so that up to 8 rows cost half of what 16-row products would and a lane's
// accumulators all belong to two rows.  As in the other kernels (diffattn.cu on
// A, B and r) the references change only where a slice's sums show they must: each
// slice adds its 16 keys' sums of both maps over 8 lanes for that comparison, and
// nothing else passes between lanes.  P_1 - r P_2 and P_2 are rounded to bf16 for
// the products with v (the tensors' own type): outputs are 2.3e-3 from the formula
// in the mean square, of which rounding the output is 1.7e-3.
//
// Keys are split over blocks, several parts per resident block: sequences of
// different lengths then balance by themselves.  Parts are joined by a second
// kernel.  Measured with a cold L2: 8 sequences of up to 32768 keys, 16 heads on 4
// of 64: 90 us, 4.5 TB/s of a copy's 6.55, and the join 7; on the kernels of
// mma.sync, which read a tile through all four warps, 274 together.
#include <algorithm>

#include "diffattn_tc.cuh"

namespace rnn {
namespace diff {
namespace {

constexpr int DEC_THREADS = 160, DEC_WARPS = 4, DEC_STAGES = 3, TILE = 64;
constexpr uint32_t PART = TILE * 128;     // 64 columns of a tile, bytes
constexpr uint32_t STAGE = 4 * PART;      // k halves, v parts
constexpr float FAR = 20.0f, FAR_SUM = 1048576.0f;
constexpr int W = 128, RJ = 2 * W + 4;    // floats of a row's partial result

struct alignas(64) DecParams {
  CUtensorMap k, v;
  Args a;
  int* dev_error;
};
struct DecShared {
  uint64_t full[DEC_STAGES], empty[DEC_STAGES];
  int abort_flag;
};
constexpr size_t DEC_SMEM = 1024 + DEC_STAGES * STAGE + sizeof(DecShared);

__device__ __forceinline__ void ldm(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldm_t(uint32_t (&r)[4], uint32_t addr) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
// The transpose of an 8 x 8 block of bf16, one register a lane.
__device__ __forceinline__ uint32_t turn8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
__device__ __forceinline__ void mma16(float (&d)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
// Over the 8 lanes that hold a row's 16 keys.
__device__ __forceinline__ float keys_max(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, o));
  return x;
}
__device__ __forceinline__ float keys_sum(float x) {
#pragma unroll
  for (int o = 4; o < 32; o <<= 1) x += __shfl_xor_sync(0xffffffffu, x, o);
  return x;
}

// NB: blocks of 8 packed rows.
template <int NB, bool MASK>
__global__ void __launch_bounds__(DEC_THREADS) dec_kernel(const __grid_constant__ DecParams p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  DecShared& sh = *reinterpret_cast<DecShared*>(base + DEC_STAGES * STAGE);
  volatile int* abort_flag = &sh.abort_flag;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int rows = a.grp * a.tq, nbh = a.n * a.hkv;
  const int bh = static_cast<int>(blockIdx.x), b = bh / a.hkv, kvh = bh - b * a.hkv;
  const int len = key_len(a, b);
  const int kbeg = static_cast<int>(blockIdx.y) * a.split_keys;
  const int kend = min(row_limit(a, a.tq - 1, len), kbeg + a.split_keys);
  const int nt = kend > kbeg ? (kend - kbeg + TILE - 1) / TILE : 0;
  const int wide = 2 * a.dh > 64 ? 2 : 1, ksteps = (a.dh + 15) / 16, msteps = a.dh / 8;

  if (tid == 0) {
    for (int i = 0; i < DEC_STAGES; i++) {
      mbar_init(&sh.full[i], 1);
      mbar_init(&sh.empty[i], DEC_WARPS);
    }
    sh.abort_flag = 0;
    fence_barrier_init();
  }
  __syncthreads();

  // lanes: g keys or columns, 2q and 2q + 1 rows of a block
  const int g = lane >> 2, q = lane & 3;
  float A[NB][8][4], B[NB][8][4];
  float m1[NB][2], m2[NB][2], l1[NB][2], l2[NB][2], r[NB][2], lam[NB][2];
  if (warp < DEC_WARPS) {
    int lim[NB][2], low = kend;
    uint32_t qf[NB][2][4][2];
    const __nv_bfloat16* qp =
        static_cast<const __nv_bfloat16*>(a.q) + b * a.qb + static_cast<long long>(kvh) * a.grp * a.qh;
#pragma unroll
    for (int nb = 0; nb < NB; nb++) {
#pragma unroll
      for (int e = 0; e < 2; e++) {
        const int row = nb * 8 + 2 * q + e;
        m1[nb][e] = m2[nb][e] = -CUDART_INF_F;
        l1[nb][e] = l2[nb][e] = 0.0f;
        lim[nb][e] = row < rows ? min(kend, row_limit(a, row % a.tq, len)) : 0;
        lam[nb][e] = row < rows ? __ldg(a.lam + kvh * a.grp + row / a.tq) : 0.0f;
        r[nb][e] = lam[nb][e];
        low = min(low, row < rows ? lim[nb][e] : kend);
      }
      // q as the MMA's column operand: row g, columns 2q, 2q + 1 (+ 8)
      const int row = nb * 8 + g;
      const __nv_bfloat16* x = qp + (row / a.tq) * a.qh + (row % a.tq) * a.qr;
#pragma unroll
      for (int h = 0; h < 2; h++)
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const int c = ks * 16 + e * 8 + 2 * q;
            qf[nb][h][ks][e] =
                row < rows && c < a.dh ? __ldg(reinterpret_cast<const unsigned int*>(x + h * a.dh + c)) : 0u;
          }
#pragma unroll
      for (int i = 0; i < 8; i++)
#pragma unroll
        for (int e = 0; e < 4; e++) A[nb][i][e] = B[nb][i][e] = 0.0f;
    }
    const int full = __reduce_min_sync(0xffffffffu, low);
    const float c2 = a.slog2;
    int st = 0, ph = 0;
    // whether a masked call's key `lane` of the warp's 16 counts, a tile ahead
    const uint8_t* mask = MASK ? a.kmask + b * a.kmb : nullptr;
    auto counts = [&](int j) { return lane < 16 && j + lane < len && mask[j + lane] != 0; };
    bool next = MASK && nt > 0 && counts(kbeg + warp * 16);
    for (int t = 0; t < nt; t++) {
      const int j0 = kbeg + t * TILE + warp * 16;
      const uint32_t seen = MASK ? __ballot_sync(0xffffffffu, next) : 0xffffu;
      if (MASK && t + 1 < nt) next = counts(j0 + TILE);
      if (!warp_wait(&sh.full[st], ph, abort_flag, p.dev_error)) break;
      if (j0 < kend) {
        const uint32_t kt = smem_u32(base) + st * STAGE, vt = kt + 2 * PART;
        if (MASK ? seen != 0xffffu : j0 + 16 > len && len < a.tk) {
          // what is hidden may be NaN, and P = 0 there
          uint8_t* v = base + st * STAGE + 2 * PART;
          for (int x = (MASK ? 0 : max(0, len - j0) * 8) + lane; x < 16 * 8; x += 32)
            if (!MASK || !(seen >> (x >> 3) & 1))
              for (int c = 0; c < wide; c++)
                *reinterpret_cast<uint4*>(v + c * PART + (warp * 16 + (x >> 3)) * 128 + (x & 7) * 16) =
                    make_uint4(0, 0, 0, 0);
          fence_async_smem();  // a later copy lands in the same place
          __syncwarp();
        }
        float s1[NB][4], s2[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int e = 0; e < 4; e++) s1[nb][e] = s2[nb][e] = 0.0f;
        const int kr = warp * 16 + (lane & 15);
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
          if (ks < ksteps) {
            uint32_t k1[4], k2[4];
            const uint32_t at = kr * 128 + (((ks * 2 + (lane >> 4)) ^ (kr & 7)) << 4);
            ldm(k1, kt + at);
            ldm(k2, kt + PART + at);
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
              mma16(s1[nb], k1, qf[nb][0][ks][0], qf[nb][0][ks][1]);
              mma16(s2[nb], k2, qf[nb][1][ks][0], qf[nb][1][ks][1]);
            }
          }
        const bool edge = j0 + 16 > full;
        bool far = false;
        float x1[NB][4], x2[NB][4];
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int e = 0; e < 4; e++) {
            float u = s1[nb][e] * c2, v = s2[nb][e] * c2;
            if ((edge && j0 + g + (e >> 1) * 8 >= lim[nb][e & 1]) || (MASK && !(seen >> (g + (e >> 1) * 8) & 1)))
              u = v = -CUDART_INF_F;
            s1[nb][e] = u;
            s2[nb][e] = v;
            const float n1 = m1[nb][e & 1], n2 = m2[nb][e & 1];
            x1[nb][e] = ex2(u - (n1 == -CUDART_INF_F ? 0.0f : n1));
            x2[nb][e] = ex2(v - (n2 == -CUDART_INF_F ? 0.0f : n2));
            far |= !(x1[nb][e] <= FAR_SUM) || !(x2[nb][e] <= FAR_SUM) ||
                   (n1 == -CUDART_INF_F && u != -CUDART_INF_F);
          }
        // references and ratios: changed where a score is far above a reference,
        // or the ratio half off lam l_1 / l_2 (what it is off by is what the
        // rounding of P_2 is multiplied with)
#pragma unroll
        for (int nb = 0; nb < NB; nb++)
#pragma unroll
          for (int e = 0; e < 2; e++) {
            const float q1 = lam[nb][e] * keys_sum(l1[nb][e] + x1[nb][e] + x1[nb][e + 2]);
            const float q2 = r[nb][e] * keys_sum(l2[nb][e] + x2[nb][e] + x2[nb][e + 2]);
            far |= fabsf(q1 - q2) > 0.5f * fabsf(q1);
          }
        if (__builtin_expect(__any_sync(0xffffffffu, far), 0)) {
#pragma unroll
          for (int nb = 0; nb < NB; nb++)
#pragma unroll
            for (int e = 0; e < 2; e++) {
              const float t1 = keys_max(fmaxf(s1[nb][e], s1[nb][e + 2]));
              const float t2 = keys_max(fmaxf(s2[nb][e], s2[nb][e + 2]));
              float f1 = 1.0f, f2 = 1.0f;
              if (m1[nb][e] == -CUDART_INF_F || t1 > m1[nb][e] + FAR) {
                f1 = m1[nb][e] == -CUDART_INF_F ? 1.0f : ex2(m1[nb][e] - t1);
                m1[nb][e] = t1;
              }
              if (m2[nb][e] == -CUDART_INF_F || t2 > m2[nb][e] + FAR) {
                f2 = m2[nb][e] == -CUDART_INF_F ? 1.0f : ex2(m2[nb][e] - t2);
                m2[nb][e] = t2;
              }
              const float n1 = m1[nb][e] == -CUDART_INF_F ? 0.0f : m1[nb][e];
              const float n2 = m2[nb][e] == -CUDART_INF_F ? 0.0f : m2[nb][e];
#pragma unroll
              for (int i = e; i < 4; i += 2) {
                x1[nb][i] = ex2(s1[nb][i] - n1);
                x2[nb][i] = ex2(s2[nb][i] - n2);
              }
              l1[nb][e] *= f1;
              l2[nb][e] *= f2;
              const float q1 = keys_sum(l1[nb][e] + x1[nb][e] + x1[nb][e + 2]);
              const float q2 = keys_sum(l2[nb][e] + x2[nb][e] + x2[nb][e + 2]);
              const float now = q1 > 0.0f && q2 > 0.0f ? lam[nb][e] * __fdividef(q1, q2) : r[nb][e];
              const float de = r[nb][e] * f1 - now * f2;
              r[nb][e] = now;
#pragma unroll
              for (int i = 0; i < 8; i++)
#pragma unroll
                for (int k = e; k < 4; k += 2) {
                  A[nb][i][k] = f1 * A[nb][i][k] + de * B[nb][i][k];
                  B[nb][i][k] *= f2;
                }
            }
        }
        uint32_t pd[NB][2], pe[NB][2];
#pragma unroll
        for (int nb = 0; nb < NB; nb++) {
#pragma unroll
          for (int e = 0; e < 2; e++) {
            l1[nb][e] += x1[nb][e] + x1[nb][e + 2];
            l2[nb][e] += x2[nb][e] + x2[nb][e + 2];
          }
#pragma unroll
          for (int e = 0; e < 2; e++) {
            pd[nb][e] = turn8(pack2(x1[nb][2 * e] - r[nb][0] * x2[nb][2 * e],
                                    x1[nb][2 * e + 1] - r[nb][1] * x2[nb][2 * e + 1]));
            pe[nb][e] = turn8(pack2(x2[nb][2 * e], x2[nb][2 * e + 1]));
          }
        }
        // v columns as rows: keys (lane >> 4) * 8 + (lane & 7), columns of chunk (lane >> 3) & 1
        const int vr = warp * 16 + (lane >> 4) * 8 + (lane & 7);
#pragma unroll
        for (int i = 0; i < 8; i++)
          if (i < msteps) {
            uint32_t f[4];
            const int ch = (i & 3) * 2 + ((lane >> 3) & 1);
            ldm_t(f, vt + (i >> 2) * PART + vr * 128 + ((ch ^ (vr & 7)) << 4));
#pragma unroll
            for (int nb = 0; nb < NB; nb++) {
              mma16(A[nb][i], f, pd[nb][0], pd[nb][1]);
              mma16(B[nb][i], f, pe[nb][0], pe[nb][1]);
            }
          }
      }
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.empty[st]);
      if (++st == DEC_STAGES) {
        st = 0;
        ph ^= 1;
      }
    }
  } else if (elect_one() && nt > 0) {
    int t = 0;
    for (; t < nt; t++) {
      const int st = t % DEC_STAGES;
      if (t >= DEC_STAGES && !wait(&sh.empty[st], (t / DEC_STAGES - 1) & 1, abort_flag, p.dev_error)) break;
      const uint32_t dst = smem_u32(base) + st * STAGE;
      mbar_arrive_expect_tx(&sh.full[st], (2 + wide) * PART);
      for (int h = 0; h < 2; h++) tma_5d(dst + h * PART, &p.k, 0, h, kvh, kbeg + t * TILE, b, &sh.full[st]);
      for (int c = 0; c < wide; c++)
        tma_5d(dst + (2 + c) * PART, &p.v, c * 64, 0, kvh, kbeg + t * TILE, b, &sh.full[st]);
    }
    // what was asked for lands before the tiles' memory is used for the join
    for (int i = max(0, t - DEC_STAGES); i < t; i++) settle(&sh.full[i % DEC_STAGES], (i / DEC_STAGES) & 1);
  }

  // join the warps through shared memory
  __syncthreads();
  float* sj = reinterpret_cast<float*>(base);
  if (warp < DEC_WARPS) {
#pragma unroll
    for (int nb = 0; nb < NB; nb++)
#pragma unroll
      for (int e = 0; e < 2; e++) {
        float* x = sj + (warp * NB * 8 + nb * 8 + 2 * q + e) * RJ;
        const float s = keys_sum(l1[nb][e]), u = keys_sum(l2[nb][e]);
#pragma unroll
        for (int i = 0; i < 8; i++)
#pragma unroll
          for (int k = 0; k < 2; k++) {
            const float y = B[nb][i][e + 2 * k];
            x[i * 16 + k * 8 + g] = A[nb][i][e + 2 * k] + r[nb][e] * y;
            x[W + i * 16 + k * 8 + g] = y;
          }
        if (g == 0) {
          x[2 * W] = m1[nb][e];
          x[2 * W + 1] = s;
          x[2 * W + 2] = m2[nb][e];
          x[2 * W + 3] = u;
        }
      }
  }
  __syncthreads();
  for (int row = warp; row < rows; row += DEC_THREADS / 32) {
    float M1 = -CUDART_INF_F, M2 = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < DEC_WARPS; w++) {
      M1 = fmaxf(M1, sj[(w * NB * 8 + row) * RJ + 2 * W]);
      M2 = fmaxf(M2, sj[(w * NB * 8 + row) * RJ + 2 * W + 2]);
    }
    float w1[DEC_WARPS], w2[DEC_WARPS], L1 = 0.0f, L2 = 0.0f;
#pragma unroll
    for (int w = 0; w < DEC_WARPS; w++) {
      const float* s = sj + (w * NB * 8 + row) * RJ + 2 * W;
      w1[w] = ex2(s[0] - (M1 == -CUDART_INF_F ? 0.0f : M1));
      w2[w] = ex2(s[2] - (M2 == -CUDART_INF_F ? 0.0f : M2));
      L1 += w1[w] * s[1];
      L2 += w2[w] * s[3];
    }
    const long long at = (static_cast<long long>(blockIdx.y) * nbh + bh) * rows + row;
    const int head = kvh * a.grp + row / a.tq, i = row % a.tq;
    const float i1 = inverse(L1), i2 = inverse(L2);
    const float lm = L2 == 0.0f ? 0.0f : __ldg(a.lam + head);
    for (int c = lane; c < 2 * a.dh; c += 32) {
      float x = 0.0f, y = 0.0f;
#pragma unroll
      for (int w = 0; w < DEC_WARPS; w++) {
        x += w1[w] * sj[(w * NB * 8 + row) * RJ + c];
        y += w2[w] * sj[(w * NB * 8 + row) * RJ + W + c];
      }
      if (a.nsplit > 1) {
        a.part[at * (2 * W) + c] = x;
        a.part[at * (2 * W) + W + c] = y;
      } else {
        static_cast<__nv_bfloat16*>(a.o)[b * a.ob + head * a.oh + i * a.orow + c] =
            __float2bfloat16_rn(x * i1 - lm * (y * i2));
        if (a.o2)
          static_cast<__nv_bfloat16*>(a.o2)[((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh) + c] =
              __float2bfloat16_rn(y * i2);
      }
    }
    if (lane == 0) {
      if (a.nsplit > 1) {
        *reinterpret_cast<float4*>(a.stat + at * 4) = make_float4(M1, L1, M2, L2);
      } else if (a.lse) {
        float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
        s[0] = log_sum(M1, L1);
        s[a.tq] = log_sum(M2, L2);
      }
    }
  }
}

template <int NB, bool MASK>
int dec_launch(rnn_ctx* ctx, DecParams& p) {
  Args& a = p.a;
  static std::atomic<unsigned long long> optin{0};
  RNN_TRY(tc::ensure_smem_optin((dec_kernel<NB, MASK>), optin, ctx->device, static_cast<int>(DEC_SMEM)));
  const long long nbh = static_cast<long long>(a.n) * a.hkv, rows = static_cast<long long>(a.grp) * a.tq;
  // Parts: about four for each of the two blocks an SM holds, of at least 256
  // keys, so that a part's start and the join stay small beside its read.
  const int tiles = (a.tk + TILE - 1) / TILE;
  const long long want = std::max(1ll, 8ll * ctx->num_sms / nbh);
  const int per = static_cast<int>(std::max<long long>(4, (tiles + want - 1) / want));
  a.split_keys = per * TILE;
  a.nsplit = std::max(1, (tiles + per - 1) / per);
  if (a.nsplit > 1) {
    const size_t part = static_cast<size_t>(a.nsplit) * nbh * rows * 2 * W * sizeof(float);
    const size_t stat = static_cast<size_t>(a.nsplit) * nbh * rows * 4 * sizeof(float);
    RNN_TRY(ensure_ws(ctx, part + stat));
    a.part = static_cast<float*>(ctx->ws);
    a.stat = a.part + part / sizeof(float);
  }
  dec_kernel<NB, MASK><<<dim3(static_cast<unsigned>(nbh), a.nsplit), DEC_THREADS, DEC_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  return a.nsplit > 1 ? join_parts(ctx, a) : RNN_OK;
}

}  // namespace

bool dec_ok(const Args& a) {
  if (static_cast<long long>(a.grp) * a.tq > 16) return false;
  if (a.dh % 8 || a.dh > 64 || a.tk < 1) return false;
  if (reinterpret_cast<uintptr_t>(a.q) % 4 || (a.qb | a.qr | a.qh) % 2) return false;
  return map_ok(a.k, a.n, a.tk, a.hkv, a.dh, a.kb, a.kr, a.kh) &&
         map_ok(a.v, a.n, a.tk, a.hkv, 2 * a.dh, a.vb, a.vr, a.vh);
}

int dec_fwd(rnn_ctx* ctx, const Args& a) {
  DecParams p;
  p.a = a;
  p.dev_error = ctx->dev_error;
  RNN_TRY(encode_map(&p.k, a.k, a.n, a.tk, a.hkv, 2, a.dh, a.kb, a.kr, a.kh, TILE));
  RNN_TRY(encode_map(&p.v, a.v, a.n, a.tk, a.hkv, 1, 2 * a.dh, a.vb, a.vr, a.vh, TILE));
  if (a.kmask)
    return static_cast<long long>(a.grp) * a.tq <= 8 ? dec_launch<1, true>(ctx, p) : dec_launch<2, true>(ctx, p);
  return static_cast<long long>(a.grp) * a.tq <= 8 ? dec_launch<1, false>(ctx, p) : dec_launch<2, false>(ctx, p);
}

}  // namespace diff
}  // namespace rnn
