// Differential attention forward on tcgen05: bf16, halves of 8 .. 64 columns
// (multiples of 8).
//
// A block owns 128 queries of one head.  Its 8 softmax warps are two teams, one
// thread per query, that take the 64-key tiles alternately, so that the
// exponentials of one team (the bound: two per query and key, 16 a clock and SM)
// run while the tensor cores form scores and the products with v for the other.
// Warp 8 copies tiles; warps 9 and 10 issue MMAs, 10 the scores of the first map,
// 9 the others (an issuing warp stalls while the tensor cores are busy, and one
// warp alone left them idle at each of its waits); warp 11 clears values
// that are masked or beyond a sequence's length.  Tensor memory (512 columns):
//   [0, 128)    A = sum (P_1 - r P_2) v        [128, 256)  B = sum P_2 v
//   [256, 384)  S_1 | S_2 of even tiles        [384, 512)  the same of odd tiles
// The bf16 maps overwrite S_2 alone: S_1 of a team's next tile is formed as soon
// as its scores are in registers, S_2 right after the products with v, behind
// the exponentials of the first map.
//
// A row's references (maxima m_1, m_2 and the ratio r) sit in shared memory and
// change rarely: a map's maximum when a tile exceeds it by 2^20 (sums and
// products are f32 and bf16, whose range allows that, so that most tiles need
// no maximum at all: their sums tell), the ratio when it is half off
// lam l_1 / l_2.  They pass from tile to tile with a token per pair of warps
// that own the same rows; who changes one waits for the products so far and
// rescales A and B.  With P_1 and P_2 in units of 2^m:
//   A <- alpha_1 A + (r alpha_1 - r' alpha_2) B,  B <- alpha_2 B,
// and at the end o = (A + (r - lam l_1/l_2) B) / l_1.
//
// Measured: 2 x 8192 x 8192 causal, 8 heads on 4 of 64: 503 us, 0.55 PF/s of the
// formula's products; a tile of 64 keys takes 2045 clocks, of which the
// exponentials alone are 1024 and the MMAs about 950.  Short calls pay a block's
// start and end: 128 x 64 x 256, 6 heads of 32: 55 us, of which 24 are tiles.
#include <algorithm>

#include "diffattn_tc.cuh"

namespace rnn {
namespace diff {

typedef CUresult (*EncodeFn)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                             const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                             CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

static EncodeFn encode_fn() {
  static const EncodeFn fn = [] {
    void* p = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &p, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeFn>(p);
    return static_cast<EncodeFn>(nullptr);
  }();
  return fn;
}

bool map_ok(const void* base, int n, int t, int heads, int cols, long long sb, long long sr, long long sh) {
  auto fits = [](int count, long long s) { return count <= 1 || (s > 0 && s % 8 == 0 && s < (1ll << 38)); };
  return reinterpret_cast<uintptr_t>(base) % 16 == 0 && cols % 8 == 0 && fits(n, sb) && fits(t, sr) && fits(heads, sh);
}

int encode_map(CUtensorMap* m, const void* base, int n, int t, int heads, int halves, int cols, long long sb,
               long long sr, long long sh, int rows) {
  EncodeFn fn = encode_fn();
  RNN_REQUIRE(fn != nullptr, "diffattn: cuTensorMapEncodeTiled unavailable");
  // the stride of an axis of one element is never used; any valid one will do
  auto bytes = [](int count, long long s) { return static_cast<cuuint64_t>(count <= 1 ? 16 : s * 2); };
  const cuuint64_t dims[5] = {(cuuint64_t)cols, (cuuint64_t)halves, (cuuint64_t)heads, (cuuint64_t)t, (cuuint64_t)n};
  const cuuint64_t strides[4] = {bytes(halves, cols), bytes(heads, sh), bytes(t, sr), bytes(n, sb)};
  const cuuint32_t box[5] = {64, 1, 1, (cuuint32_t)rows, 1};
  const cuuint32_t estr[5] = {1, 1, 1, 1, 1};
  const CUresult r = fn(m, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 5, const_cast<void*>(base), dims, strides, box, estr,
                        CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_128B,
                        CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  RNN_REQUIRE(r == CUDA_SUCCESS, "diffattn: cuTensorMapEncodeTiled failed (CUresult %d)", (int)r);
  return RNN_OK;
}

namespace {

constexpr int QROWS = 128, KEYS = 64, STAGES = 5;
constexpr int FWD_THREADS = 384;
constexpr int SOFT_WARPS = 8, WARP_COPY = 8, WARP_MMA = 9, WARP_SCORE = 10, WARP_CLEAR = 11;
constexpr uint32_t Q_BYTES = 2 * QROWS * 128;      // two halves, rows of 128 bytes
constexpr uint32_t HALF_BYTES = KEYS * 128;        // one half of k, or 64 columns of v
constexpr uint32_t STAGE_BYTES = 4 * HALF_BYTES;   // k halves, then v columns
constexpr uint32_t COL_B = 128, COL_S = 256;
constexpr float RAISE = 20.0f, RAISE_SUM = 1048576.0f;

struct alignas(64) FwdParams {
  CUtensorMap q, k, v;
  Args a;
  int* dev_error;  // the context's error word
  int o16;         // 16-byte stores of o are aligned
};

struct FwdShared {
  uint64_t q_full, kv_full[STAGES], kv_empty[STAGES], landed[STAGES], s1_full[2], s2_full[2], s1_free[2], p_full[2];
  uint64_t pv_last, o_full, tok[4], drain[2];
  uint32_t tmem;
  int abort_flag;
  uint2 seen[STAGES];    // masked calls: which keys of a tile count
  float4 ref[QROWS];     // a row's m_1, m_2, r
  float4 sum[2][QROWS];  // m_1, l_1, m_2, l_2 of a team
};
constexpr size_t FWD_SMEM = 1024 + Q_BYTES + STAGES * STAGE_BYTES + sizeof(FwdShared);

// What a thread does with its row's 64 scores of one map.
template <bool MASK>
__device__ __forceinline__ void mask_scores(float (&s)[2][32], int visible, uint2 seen) {
#pragma unroll
  for (int c = 0; c < KEYS; c++)
    if (c >= visible || (MASK && !((c < 32 ? seen.x : seen.y) >> (c & 31) & 1))) s[c >> 5][c & 31] = -CUDART_INF_F;
}
__device__ __forceinline__ float max_of(const float (&s)[2][32]) {
  float m[4] = {s[0][0], s[0][1], s[0][2], s[0][3]};
#pragma unroll
  for (int c = 4; c < KEYS; c++) m[c & 3] = fmaxf(m[c & 3], s[c >> 5][c & 31]);
  return fmaxf(fmaxf(m[0], m[1]), fmaxf(m[2], m[3]));
}
// s <- 2^(s c2 - u); returns the sum.
__device__ __forceinline__ float exp_sum(float (&s)[2][32], float c2, float u) {
  const f32x2 cc = pair(c2, c2), uu = pair(-u, -u);
  f32x2 t[2] = {0ull, 0ull};
#pragma unroll
  for (int i = 0; i < KEYS / 2; i++) {
    float& x = s[i >> 4][(2 * i) & 31];
    float& y = s[i >> 4][(2 * i + 1) & 31];
    unpair(fma2(pair(x, y), cc, uu), x, y);
    x = ex2(x);
    y = ex2(y);
    t[i & 1] = add2(t[i & 1], pair(x, y));
  }
  float x, y;
  unpair(add2(t[0], t[1]), x, y);
  return x + y;
}
// A row's exponentials of one map, from the scores at tensor memory address t
// to s, at reference u; returns their sum.  The maximum is only looked for where
// it matters: when a row has no reference yet (u = -inf) or the sum shows that
// a score passed it by about 2^20; rows beyond that get their tile's maximum.
template <bool MASK>
__device__ __forceinline__ float exponentials(uint32_t t, float (&s)[2][32], float& u, float c2, bool edge,
                                              int visible, uint2 seen) {
  bool look = __any_sync(0xffffffffu, u == -CUDART_INF_F && visible > 0);
  while (true) {
    tmem_ld(t, s[0]);
    tmem_ld(t + 32, s[1]);
    tmem_landed(s[0]);
    tmem_landed(s[1]);
    if (__builtin_expect(edge, 0)) mask_scores<MASK>(s, visible, seen);
    if (__builtin_expect(look, 0)) {
      const float top = max_of(s) * c2;
      if (u == -CUDART_INF_F || top > u + RAISE) u = top;
    }
    const float sum = exp_sum(s, c2, u == -CUDART_INF_F ? 0.0f : u);
    if (__builtin_expect(look || __all_sync(0xffffffffu, sum <= RAISE_SUM), 1)) return sum;
    look = true;
  }
}
// Moves a row's reference m to the reference u of the tile's exponentials if
// that is far above it (al: the factor of what was summed before; true), else
// keeps it (f: the factor of this tile).
__device__ __forceinline__ bool raise(float& m, float u, float& al, float& f) {
  if (u == m || u == -CUDART_INF_F) return false;
  if (m == -CUDART_INF_F) {
    m = u;
    return false;
  }
  if (u > m + RAISE) {
    al = ex2(m - u);
    m = u;
    return true;
  }
  f = ex2(u - m);
  return false;
}
// Writes P_1 - r P_2 and P_2 as bf16 operands of 32 columns each: the type of the
// tensors, and half the MMAs that two planes of a map would take.  Outputs are then
// 2.3e-3 from the formula in the mean square, of which rounding the output is 1.7e-3.
__device__ __forceinline__ void store_maps(uint32_t dst, const float (&s1)[2][32], const float (&s2)[2][32], float r) {
  const f32x2 rr = pair(-r, -r);
#pragma unroll
  for (int h = 0; h < 2; h++) {
    uint32_t d[16], e[16];
#pragma unroll
    for (int i = 0; i < 16; i++) {
      float z0, z1;
      unpair(fma2(pair(s2[h][2 * i], s2[h][2 * i + 1]), rr, pair(s1[h][2 * i], s1[h][2 * i + 1])), z0, z1);
      d[i] = pack2(z0, z1);
      e[i] = pack2(s2[h][2 * i], s2[h][2 * i + 1]);
    }
    tmem_st(dst + h * 16, d);
    tmem_st(dst + 32 + h * 16, e);
  }
}
__device__ __forceinline__ void soft_sync() { asm volatile("bar.sync 1, 256;" ::: "memory"); }

template <bool MASK>
__global__ void __launch_bounds__(FWD_THREADS, 1) tc_fwd_kernel(const __grid_constant__ FwdParams p) {
  extern __shared__ uint8_t raw[];
  const Args& a = p.a;
  uint8_t* base = raw + ((1024 - (smem_u32(raw) & 1023)) & 1023);
  const uint32_t sq = smem_u32(base), skv = sq + Q_BYTES;
  FwdShared& sh = *reinterpret_cast<FwdShared*>(base + Q_BYTES + STAGES * STAGE_BYTES);
  volatile int* abort_flag = &sh.abort_flag;
  int* dev_error = p.dev_error;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int ntile = (a.tq + QROWS - 1) / QROWS, nbh = a.n * a.h;
  const int tile = ntile - 1 - static_cast<int>(blockIdx.x) / nbh;  // longest causal rows first
  const int bh = static_cast<int>(blockIdx.x) % nbh;
  const int b = bh / a.h, head = bh - b * a.h, kvh = head / a.grp;
  const int i0 = tile * QROWS;
  const int len = key_len(a, b);
  // this block's part of the keys: all of them, or split_keys (a multiple of KEYS)
  const int kbeg = static_cast<int>(blockIdx.y) * a.split_keys;
  const int kend = min(row_limit(a, min(i0 + QROWS, a.tq) - 1, len), kbeg + a.split_keys);
  const int nt = max(kend - kbeg + KEYS - 1, 0) / KEYS;
  // Values that a row must not meet are cleared: the last tile's that lie in a
  // cache beyond the sequence, any tile's that are masked.
  const uint8_t* mask = MASK ? a.kmask + b * a.kmb : nullptr;
  const int clear0 = MASK ? 0 : nt > 0 && kbeg + nt * KEYS > len && len < a.tk ? nt - 1 : nt;  // first tile to be cleared
  // phase of a tile's arrival: a stage's uses so far, of one barrier or the other
  auto clears = [&](int j) { return j >= clear0 && clear0 > 0 ? 0u : static_cast<uint32_t>(j / STAGES) & 1u; };
  const int wide = 2 * a.dh > 64 ? 2 : 1;  // 64-column parts of v
  const int ksteps = (a.dh + 15) / 16;

  if (tid == 0) {
    mbar_init(&sh.q_full, 1);
    for (int i = 0; i < STAGES; i++) {
      mbar_init(&sh.kv_full[i], 1);
      mbar_init(&sh.kv_empty[i], 1);
      mbar_init(&sh.landed[i], 1);
    }
    for (int i = 0; i < 2; i++) {
      mbar_init(&sh.s1_full[i], 1);
      mbar_init(&sh.s2_full[i], 1);
      mbar_init(&sh.s1_free[i], 4);
      mbar_init(&sh.p_full[i], 4);
    }
    mbar_init(&sh.pv_last, 1);
    mbar_init(&sh.o_full, 1);
    for (int i = 0; i < 4; i++) {
      mbar_init(&sh.tok[i], 1);
    }
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
  // registers: 384 threads x 168 at launch; the softmax teams hold a row's 128
  // scores (256 x 216 + 128 x 72 = 384 x 168)
  if (warp < SOFT_WARPS) {
    asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
    const int team = warp >> 2, w = warp & 3, row = w * 32 + lane, i = i0 + row;
    const uint32_t lanes = static_cast<uint32_t>(w * 32) << 16;
    const uint32_t ts = tmem + lanes + COL_S + team * 128;
    const int lim = i < a.tq ? row_limit(a, i, len) : 0;
    const int full = __reduce_min_sync(0xffffffffu, lim);
    const float lam = __ldg(a.lam + head), c2 = a.slog2;
    float m1 = -CUDART_INF_F, m2 = -CUDART_INF_F, l1 = 0.0f, l2 = 0.0f, r = lam;

    for (int j = team; j < nt; j += 2) {
      const int j0 = kbeg + j * KEYS;
      bool edge = j0 + KEYS > full;
      const uint32_t par = (j >> 1) & 1;
      float s1[2][32], s2[2][32];
      // the references the exponentials are taken at: the row's, as far as this
      // team knows them
      float u1 = m1, u2 = m2;
      uint2 seen = make_uint2(0xffffffffu, 0xffffffffu);
      if (MASK) {  // from the clearing warp
        if (!warp_wait(&sh.kv_full[j % STAGES], (j / STAGES) & 1, abort_flag, dev_error)) break;
        seen = sh.seen[j % STAGES];
        edge |= (seen.x & seen.y) != 0xffffffffu;
      }
      if (!warp_wait(&sh.s1_full[team], par, abort_flag, dev_error)) break;
      tc_fence_after();
      const float sum1 = exponentials<MASK>(ts, s1, u1, c2, edge, lim - j0, seen);
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.s1_free[team]);
      if (!warp_wait(&sh.s2_full[team], par, abort_flag, dev_error)) break;
      tc_fence_after();
      const float sum2 = exponentials<MASK>(ts + 64, s2, u2, c2, edge, lim - j0, seen);

      // The row's references as tile j - 1 left them.  Where they are what the
      // exponentials were taken at (nearly always), only the sums go on; else
      // the sums and maps of this tile move to what the references become.
      bool change = true;
      float4 ref = make_float4(-CUDART_INF_F, -CUDART_INF_F, lam, 0.0f);
      float4 other = make_float4(-CUDART_INF_F, 0.0f, -CUDART_INF_F, 0.0f);  // the other team's sums
      if (j > 0) {
        if (!warp_wait(&sh.tok[w], (j - 1) & 1, abort_flag, dev_error)) break;
        ref = sh.ref[row];
        other = sh.sum[team ^ 1][row];
        // The ratio has to stay near lam l_1 / l_2: what it is off by is what the
        // rounding of P_2 is multiplied with.
        const float q1 = lam * (l1 + sum1 + other.y), q2 = ref.z * (l2 + sum2 + other.w);
        change = ref.x != u1 || ref.y != u2 || ref.x != m1 || ref.y != m2 || fabsf(q1 - q2) > 0.5f * fabsf(q1);
      }
      r = ref.z;
      if (__builtin_expect(!__any_sync(0xffffffffu, change), 1)) {
        l1 += sum1;
        l2 += sum2;
        sh.sum[team][row] = make_float4(m1, l1, m2, l2);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.tok[w]);
      } else {
        if (ref.x != m1) l1 *= ex2(m1 - ref.x);
        if (ref.y != m2) l2 *= ex2(m2 - ref.y);
        m1 = ref.x;
        m2 = ref.y;
        float al1 = 1.0f, al2 = 1.0f, f1 = 1.0f, f2 = 1.0f, rn = r;
        bool event = raise(m1, u1, al1, f1);
        event |= raise(m2, u2, al2, f2);
        l1 = l1 * al1 + sum1 * f1;
        l2 = l2 * al2 + sum2 * f2;
        // the sums so far: own ones, and the other team's as it gave them with its
        // last token (which tiles they cover does not depend on timing)
        float q1 = l1, q2 = l2;
        if (other.y > 0.0f) q1 += other.y * ex2(other.x - m1);
        if (other.w > 0.0f) q2 += other.w * ex2(other.z - m2);
        const float want = lam * __fdividef(q1, q2);
        if (q1 > 0.0f && q2 > 0.0f && (j == 0 || fabsf(want - r) > 0.25f * fabsf(want))) {
          rn = want;
          event = true;
        }
        sh.sum[team][row] = make_float4(m1, l1, m2, l2);
        sh.ref[row] = make_float4(m1, m2, rn, 0.0f);
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.tok[w]);
        if (j > 0 && __any_sync(0xffffffffu, event)) {
          // the products up to tile j - 1, which the scores of tile j + 1 follow
          if (!(j + 1 < nt ? warp_wait(&sh.s2_full[team ^ 1], ((j + 1) >> 1) & 1, abort_flag, dev_error)
                           : warp_wait(&sh.pv_last, 0, abort_flag, dev_error)))
            break;
          tc_fence_after();
          const float de = r * al1 - rn * al2;
#pragma unroll 1
          for (int c = 0; c < 2 * a.dh; c += 16) {
            float x[16], y[16];
            tmem_ld(tmem + lanes + c, x);
            tmem_ld(tmem + lanes + COL_B + c, y);
            tmem_landed(x);
            tmem_landed(y);
#pragma unroll
            for (int k = 0; k < 16; k++) {
              x[k] = al1 * x[k] + de * y[k];
              y[k] *= al2;
            }
            tmem_st(tmem + lanes + c, x);
            tmem_st(tmem + lanes + COL_B + c, y);
          }
        }
        r = rn;
        if (__any_sync(0xffffffffu, f1 != 1.0f || f2 != 1.0f)) {
#pragma unroll
          for (int c = 0; c < KEYS; c++) {
            s1[c >> 5][c & 31] *= f1;
            s2[c >> 5][c & 31] *= f2;
          }
        }
      }
      store_maps(ts + 64, s1, s2, r);
      tmem_wait_st();
      tc_fence_before();
      __syncwarp();
      if (lane == 0) mbar_arrive(&sh.p_full[team]);
    }

    // join the teams' sums at the final references
    soft_sync();
    const float4 last = nt > 0 ? sh.ref[row] : make_float4(-CUDART_INF_F, -CUDART_INF_F, 0.0f, 0.0f);
    if (last.x != m1) l1 *= ex2(m1 - last.x);
    if (last.y != m2) l2 *= ex2(m2 - last.y);
    sh.sum[team][row] = make_float4(0.0f, l1, 0.0f, l2);
    soft_sync();
    const float L1 = sh.sum[0][row].y + sh.sum[1][row].y, L2 = sh.sum[0][row].w + sh.sum[1][row].w;
    // o = (A + (r - lam l_1 / l_2) B) / l_1; where the first map is 0, -lam B / l_2
    const bool one = L1 != 0.0f, two = L2 != 0.0f;
    const float i1 = one ? 1.0f / L1 : 1.0f, i2 = inverse(L2);
    const float rest = one ? last.z - lam * L1 * i2 : two ? -lam * i2 : 0.0f;
    bool ok = true;
    if (nt > 0) {
      ok = warp_wait(&sh.o_full, 0, abort_flag, dev_error);
      tc_fence_after();
    }
    __nv_bfloat16* o = static_cast<__nv_bfloat16*>(a.o) + b * a.ob + head * a.oh + i * a.orow;
    __nv_bfloat16* o2 =
        a.o2 ? static_cast<__nv_bfloat16*>(a.o2) + ((static_cast<long long>(b) * a.tq + i) * a.h + head) * (2 * a.dh)
             : nullptr;
    const bool whole = a.nsplit == 1;
    // a part's sums of the maps' products with v, for join_kernel: A + r B and B
    const long long idx = (static_cast<long long>(b) * a.hkv + kvh) * (static_cast<long long>(a.grp) * a.tq) +
                          static_cast<long long>(head - kvh * a.grp) * a.tq + i;
    const long long at = blockIdx.y * (static_cast<long long>(nbh) * a.tq) + idx;
    if (!whole && team == 0 && i < a.tq)
      *reinterpret_cast<float4*>(a.stat + at * 4) = make_float4(last.x, L1, last.y, L2);
    // 16 columns at a time, the two threads of a row in turn
    for (int c = team * 16; ok && c < 2 * a.dh; c += 32) {
      float x[16] = {}, y[16] = {};
      if (nt > 0) {
        tmem_ld(tmem + lanes + c, x);
        tmem_ld(tmem + lanes + COL_B + c, y);
        tmem_landed(x);
        tmem_landed(y);
      }
      if (!whole) {
        if (i < a.tq) {
          float4* px = reinterpret_cast<float4*>(a.part + at * 256 + c);
#pragma unroll
          for (int k = 0; k < 4; k++) {
            px[k] = make_float4(x[4 * k] + last.z * y[4 * k], x[4 * k + 1] + last.z * y[4 * k + 1],
                                x[4 * k + 2] + last.z * y[4 * k + 2], x[4 * k + 3] + last.z * y[4 * k + 3]);
            px[32 + k] = make_float4(y[4 * k], y[4 * k + 1], y[4 * k + 2], y[4 * k + 3]);
          }
        }
        __syncwarp();
        continue;
      }
      uint32_t po[8], p2[8];
#pragma unroll
      for (int k = 0; k < 8; k++) {
        // a map without a key has no part in the products but what 0 * inf or 0 * NaN left
        const float y0 = two ? y[2 * k] : 0.0f, y1 = two ? y[2 * k + 1] : 0.0f;
        const float x0 = ((one ? x[2 * k] : 0.0f) + rest * y0) * i1;
        const float x1 = ((one ? x[2 * k + 1] : 0.0f) + rest * y1) * i1;
        po[k] = pack2(x0, x1);
        p2[k] = pack2(y0 * i2, y1 * i2);
      }
      if (i < a.tq) {
        if (p.o16) {
          *reinterpret_cast<uint4*>(o + c) = make_uint4(po[0], po[1], po[2], po[3]);
          *reinterpret_cast<uint4*>(o + c + 8) = make_uint4(po[4], po[5], po[6], po[7]);
        } else {
#pragma unroll
          for (int k = 0; k < 8; k++) {
            const __nv_bfloat162 z = *reinterpret_cast<__nv_bfloat162*>(&po[k]);
            o[c + 2 * k] = z.x;
            o[c + 2 * k + 1] = z.y;
          }
        }
        if (o2) {
          *reinterpret_cast<uint4*>(o2 + c) = make_uint4(p2[0], p2[1], p2[2], p2[3]);
          *reinterpret_cast<uint4*>(o2 + c + 8) = make_uint4(p2[4], p2[5], p2[6], p2[7]);
        }
      }
      __syncwarp();
    }
    if (whole && a.lse && team == 0 && i < a.tq) {
      float* s = a.lse + (static_cast<long long>(b) * a.h + head) * 2 * a.tq + i;
      s[0] = log_sum(last.x, L1);
      s[a.tq] = log_sum(last.y, L2);
    }
  } else {
    asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
    if (warp == WARP_COPY) {
      if (elect_one() && nt > 0) {
        mbar_arrive_expect_tx(&sh.q_full, Q_BYTES);
        for (int half = 0; half < 2; half++)
          tma_5d(sq + half * (QROWS * 128), &p.q, 0, half, head, i0, b, &sh.q_full);
        int j = 0;
        for (; j < nt; j++) {
          const int st = j % STAGES;
          if (j >= STAGES && !wait(&sh.kv_empty[st], (j / STAGES - 1) & 1, abort_flag, dev_error)) break;
          const uint32_t dst = skv + st * STAGE_BYTES;
          // a tile to be cleared lands for the clearing warp, which passes it on
          uint64_t* bar = j >= clear0 ? &sh.landed[st] : &sh.kv_full[st];
          mbar_arrive_expect_tx(bar, (2 + wide) * HALF_BYTES);
          for (int half = 0; half < 2; half++)
            tma_5d(dst + half * HALF_BYTES, &p.k, 0, half, kvh, kbeg + j * KEYS, b, bar);
          for (int c = 0; c < wide; c++)
            tma_5d(dst + (2 + c) * HALF_BYTES, &p.v, c * 64, 0, kvh, kbeg + j * KEYS, b, bar);
        }
        // what was asked for lands before the block may end, aborting or not
        settle(&sh.q_full, 0);
        for (int t = max(0, j - STAGES); t < j; t++)
          settle(t >= clear0 ? &sh.landed[t % STAGES] : &sh.kv_full[t % STAGES], clears(t));
      }
      __syncwarp();
    } else if (warp == WARP_CLEAR) {
      Seen keys;
      if (clear0 < nt) keys.load(mask, kbeg + clear0 * KEYS, len);
      for (int j = clear0; j < nt; j++) {
        const int st = j % STAGES;
        const uint2 seen = keys.bits();
        if (j + 1 < nt) keys.load(mask, kbeg + (j + 1) * KEYS, len);
        if (!warp_wait(&sh.landed[st], clears(j), abort_flag, dev_error)) break;
        clear_hidden(base + Q_BYTES + st * STAGE_BYTES + 2 * HALF_BYTES, seen, wide);
        if (lane == 0) sh.seen[st] = seen;
        fence_async_smem();
        __syncwarp();
        if (lane == 0) mbar_arrive(&sh.kv_full[st]);
      }
    } else if (nt > 0) {
      const uint32_t lead = elect_one() ? 1u : 0u;
      const uint32_t id_s = idesc_bf16(QROWS, KEYS, false);
      const uint64_t dq = desc_k(sq), dkv = desc_k(skv);
      auto done = [&](uint64_t* bar, uint32_t parity) { return warp_wait(bar, parity, abort_flag, dev_error); };
      auto landed = [&](int j, int st) { return done(&sh.kv_full[st], (j / STAGES) & 1); };
      // scores of one map of tile j (stage st); descriptors count 16 bytes
      auto scores = [&](int j, int st, int half) {
        const uint64_t q = dq + half * (QROWS * 128 / 16), k = dkv + (st * STAGE_BYTES + half * HALF_BYTES) / 16;
        const uint32_t d = tmem + COL_S + (j & 1) * 128 + half * KEYS;
#pragma unroll
        for (int ks = 0; ks < 4; ks++)
          if (ks < ksteps) mma_ss(d, q + ks * 2, k + ks * 2, id_s, ks > 0, lead);
        commit(half ? &sh.s2_full[j & 1] : &sh.s1_full[j & 1], lead);
      };
      bool ok = done(&sh.q_full, 0);
      int st = 0;
      if (warp == WARP_SCORE) {
        for (int j = 0; ok && j < nt; j++) {
          // the team has the scores of tile j - 2 in registers
          if (!(ok = landed(j, st) && (j < 2 || done(&sh.s1_free[j & 1], ((j >> 1) - 1) & 1)))) break;
          tc_fence_after();
          scores(j, st, 0);
          if (++st == STAGES) st = 0;
        }
      } else {
        const uint32_t id_o = idesc_bf16(QROWS, 64, true);
        const uint64_t dv = desc_mn(skv + 2 * HALF_BYTES, 0);
        for (int j = 0; ok && j < min(nt, 2); j++)
          if ((ok = landed(j, j))) {
            tc_fence_after();
            scores(j, j, 1);
          }
        int st2 = 2;
        for (int j = 0; ok && j < nt; j++) {
          if (!(ok = (j + 2 >= nt || landed(j + 2, st2)) && done(&sh.p_full[j & 1], (j >> 1) & 1))) break;
          tc_fence_after();
          const uint64_t v = dv + st * (STAGE_BYTES / 16);
          const uint32_t s = tmem + COL_S + (j & 1) * 128 + KEYS;
          for (int c = 0; c < wide; c++) {
#pragma unroll
            for (int ks = 0; ks < KEYS / 16; ks++) {
              const uint64_t d = v + (c * HALF_BYTES + ks * 2048) / 16;
              mma_ts(tmem + c * 64, s + ks * 8, d, id_o, j > 0 || ks > 0, lead);
              mma_ts(tmem + COL_B + c * 64, s + 32 + ks * 8, d, id_o, j > 0 || ks > 0, lead);
            }
          }
          // the scores of tile j are long done: its maps came of them
          commit(&sh.kv_empty[st], lead);
          if (j + 2 == nt) commit(&sh.pv_last, lead);
          if (j + 1 == nt) commit(&sh.o_full, lead);
          // The next scores of the second map overwrite the maps that these
          // products read.  This warp's MMAs have one accumulator shape
          // (128 x 64), which makes them execute in the order of issue.
          if (j + 2 < nt) scores(j + 2, st2, 1);
          if (++st == STAGES) st = 0;
          if (++st2 == STAGES) st2 = 0;
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

}  // namespace

// A block costs about 5 us beside its tiles, whose time does not go by dh, and
// holds one head's rows, while the kernels of mma.sync pack the rows of all heads
// that share keys and run several blocks an SM.  So they keep what is short on
// both sides (256 x 32 x 32, 4 heads of 32: 20 us against 41 here), what is little
// work (128 x 64 x 64 of 8: 12 and, backward, 27 against 24 and 54; 32 x 1000 x 4
// of 16: 50 against 79; but 64 x 100 x 100 of 8: 19 and 45 against 16 and 35) and
// rows too few to fill a tile (64 x 3 x 1024, 32 heads on 4: 96 against 346; 64 x 9 x 512, 8 on
// 2: 50 against 62).  The rest is faster here: 64 x 24 x 256, 8 of 32: 39 against
// 51; 128 x 33 x 1000, 8 of 64: 181 against 508; 32 x 1000 x 16: 102 against 131
// (the others timed with a mask of keys that hides none).
bool big_enough(const Args& a) {
  return std::max(a.tq, a.tk) >= 64 && static_cast<long long>(a.tq) * a.tk * a.dh >= 65536;
}
bool tc_fwd_ok(const Args& a) {
  if (a.dh % 8 || a.dh > 64 || !(a.slog2 > 0.0f) || a.slog2 > 1e30f) return false;
  if (a.tq < 16 || !big_enough(a)) return false;
  if (reinterpret_cast<uintptr_t>(a.o2) % 16) return false;
  return map_ok(a.q, a.n, a.tq, a.h, a.dh, a.qb, a.qr, a.qh) && map_ok(a.k, a.n, a.tk, a.hkv, a.dh, a.kb, a.kr, a.kh) &&
         map_ok(a.v, a.n, a.tk, a.hkv, 2 * a.dh, a.vb, a.vr, a.vh);
}

// When the rows leave SMs idle the keys are split over blocks.  A part's start
// and end and the join cost about seven tiles' time (1.06 us each).  Measured
// whole and split: 1 x 128 x 8192, 16 heads: 133 and 34 us; 1 x 64 x 16384, 4
// heads: 293 and 31; 4 x 128 x 1024, 8 heads: 24 and 21; but 2 x 256 x 512, 8
// heads: 14 and 16 in four parts.
static long long key_parts(const rnn_ctx* ctx, long long blocks, int tiles) {
  const long long parts = std::min<long long>(ctx->num_sms / blocks, tiles / 4);
  return parts > 1 && tiles - tiles / parts > 7 ? parts : 1;
}

int tc_fwd(rnn_ctx* ctx, const Args& a) {
  FwdParams p;
  p.a = a;
  p.dev_error = ctx->dev_error;
  auto m8 = [](long long s) { return s % 8 == 0; };
  p.o16 = reinterpret_cast<uintptr_t>(a.o) % 16 == 0 && m8(a.ob) && m8(a.orow) && m8(a.oh);
  RNN_TRY(encode_map(&p.q, a.q, a.n, a.tq, a.h, 2, a.dh, a.qb, a.qr, a.qh, QROWS));
  RNN_TRY(encode_map(&p.k, a.k, a.n, a.tk, a.hkv, 2, a.dh, a.kb, a.kr, a.kh, KEYS));
  RNN_TRY(encode_map(&p.v, a.v, a.n, a.tk, a.hkv, 1, 2 * a.dh, a.vb, a.vr, a.vh, KEYS));
  const long long blocks = (a.tq + QROWS - 1ll) / QROWS * a.n * a.h;
  RNN_REQUIRE(blocks < (1ll << 31), "diffattn: too many rows");
  static std::atomic<unsigned long long> optin[2];
  const auto kernel = a.kmask ? tc_fwd_kernel<true> : tc_fwd_kernel<false>;
  RNN_TRY(tc::ensure_smem_optin(kernel, optin[a.kmask != nullptr], ctx->device, static_cast<int>(FWD_SMEM)));
  const int tiles = (a.tk + KEYS - 1) / KEYS;
  const long long parts = key_parts(ctx, blocks, tiles);
  p.a.split_keys = static_cast<int>((tiles + parts - 1) / parts) * KEYS;
  p.a.nsplit = (a.tk + p.a.split_keys - 1) / p.a.split_keys;
  if (p.a.nsplit > 1) {
    const size_t rows = static_cast<size_t>(a.n) * a.h * a.tq;
    RNN_TRY(ensure_ws(ctx, rows * p.a.nsplit * (256 + 4) * sizeof(float)));
    p.a.part = static_cast<float*>(ctx->ws);
    p.a.stat = p.a.part + rows * p.a.nsplit * 256;
  }
  kernel<<<dim3(static_cast<unsigned>(blocks), p.a.nsplit), FWD_THREADS, FWD_SMEM, ctx->stream>>>(p);
  RNN_CHECK_LAUNCH();
  return p.a.nsplit > 1 ? join_rows_bf16(ctx, p.a) : RNN_OK;
}

}  // namespace diff
}  // namespace rnn
