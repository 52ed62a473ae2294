// Products of 8-bit rows:  y[m][n] = xs[m] ws[n] sum_k x[m][k] w[n][k] (+ bias[n]),  bf16 or fp32 out.
// The sum is exact: int32 holds K <= 131056 products of 128 128, so that every way of cutting K gives the same bits.
//
// The matrix instruction is v_mfma_i32_16x16x64_i8 with the weight as its first operand: lane l holds 16 bytes of row l & 15
// at byte 16 (l >> 4), and gets the sums of columns 4 (l >> 4) .. + 3 of row l & 15 of x, so that it stores four neighbours.
#include <cmath>

#include "int8_rows.h"

namespace k8s {
namespace q8 {

struct GemmArgs {
  const uint8_t *x, *w;
  const float *xs, *ws, *bias;
  void* y;
  long ldx, ldw, ldy;
  int M, N, K, f32;
  int splits;    // runs of K; with more than one, int32 sums go to `part` (any order of adding gives the same): [splits][M][ldp],
  int* part;     // of 256 x 256 tiles [tile - whole][splits][256][256]
  long ldp;      // a multiple of 8, at least N
  int whole;     // 256 x 256: tiles in front whose K is not cut
};
__device__ const i32x4 kZeros = {0, 0, 0, 0};

// Whether rows of y take pieces of V values (columns start at multiples of V).
template <int V>
__device__ __forceinline__ bool aligned_rows(const GemmArgs& a) {
  return (a.ldy & (V - 1)) == 0 && ((uintptr_t)a.y & 15) == 0;
}

// R rows by C pieces of V neighbouring columns: row(i) and col(j) are the row and the first column, at(i, j, e) an integer sum.
// Scales and bias are asked for together, in front of the first store (a load behind a store waits for both).
template <int R, int C, int V, typename Row, typename Col, typename At>
__device__ __forceinline__ void put_block(const GemmArgs& a, Row row, Col col, At at) {
  float f[R], w[C][V], b[C][V] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) f[i] = a.xs[min(row(i), a.M - 1)];
#pragma unroll
  for (int j = 0; j < C; ++j)
#pragma unroll
    for (int e = 0; e < V; ++e) w[j][e] = a.ws[min(col(j) + e, a.N - 1)];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < C; ++j)
#pragma unroll
      for (int e = 0; e < V; ++e) b[j][e] = a.bias[min(col(j) + e, a.N - 1)];
  }
  const bool wide = aligned_rows<V>(a);
  auto value = [&](int i, int j, int e) { return fmaf((float)at(i, j, e) * f[i], w[j][e], b[j][e]); };
  if (a.f32) {
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int m = row(i), n = col(j);
        if (m >= a.M) continue;
        float* const o = (float*)a.y + (long)m * a.ldy + n;
        if (wide && n + V <= a.N) {
#pragma unroll
          for (int e = 0; e < V; e += 4)
            *reinterpret_cast<f32x4*>(o + e) = f32x4{value(i, j, e), value(i, j, e + 1), value(i, j, e + 2), value(i, j, e + 3)};
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (n + e < a.N) o[e] = value(i, j, e);
        }
      }
  } else {
    typedef uint16_t out_t __attribute__((ext_vector_type(V)));
#pragma unroll
    for (int i = 0; i < R; ++i)
#pragma unroll
      for (int j = 0; j < C; ++j) {
        const int m = row(i), n = col(j);
        if (m >= a.M) continue;
        uint16_t* const o = (uint16_t*)a.y + (long)m * a.ldy + n;
        out_t v;
#pragma unroll
        for (int e = 0; e < V; ++e) v[e] = f2bf(value(i, j, e));
        if (wide && n + V <= a.N) {
          *reinterpret_cast<out_t*>(o) = v;
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e)
            if (n + e < a.N) o[e] = v[e];
        }
      }
  }
}
__device__ __forceinline__ void put4(const GemmArgs& a, int m, int n, const i32x4& s) {
  put_block<1, 1, 4>(a, [&](int) { return m; }, [&](int) { return n; }, [&](int, int, int e) { return s[e]; });
}
// The same for other rows: R times 16 rows by C times 32 columns of a wave turn in its own LDS (kTurn numbers), 16 by 32 at a time, so that
// a store has neighbouring lanes at neighbouring columns.  row(i) and col(j) are where they begin; lane (r, g) holds sums
// at(i, j, e) of row r, e < 8: of columns V (g + 4 (e / V)) + e % V.
// us of 3655 x 1772 x 2048 and, in fp32, of 484 x 21381 x 432 and 800 x 36639 x 9136: value by value from where they are 47.3, 49.2 and
// 409, turned with each piece's scales asked for behind the last one's stores 47.0, 33.1 and 337, with all of them in front 35.2, 22.1 and
// 332 (the next widths that rows start evenly with: 29.6, 22.7 and 322).
constexpr int kTurnRow = 36, kTurn = 16 * kTurnRow;
template <int R, int C, int V, typename Row, typename Col, typename At>
__device__ __forceinline__ void put_turned(const GemmArgs& a, float* lds, int lane, Row row, Col col, At at) {
  const int r = lane & 15, g = lane >> 4, c = lane & 31, hi = lane >> 5;
  float f[R], w[C], b[C] = {};
#pragma unroll
  for (int i = 0; i < R; ++i) f[i] = a.xs[min(row(i) + r, a.M - 1)];
#pragma unroll
  for (int j = 0; j < C; ++j) w[j] = a.ws[min(col(j) + c, a.N - 1)];
  if (a.bias) {
#pragma unroll
    for (int j = 0; j < C; ++j) b[j] = a.bias[min(col(j) + c, a.N - 1)];
  }
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < C; ++j) {
#pragma unroll
      for (int e = 0; e < 8; e += 4)
        *reinterpret_cast<f32x4*>(lds + r * kTurnRow + V * (g + 4 * (e / V)) + e % V) =
            f32x4{(float)at(i, j, e) * f[i], (float)at(i, j, e + 1) * f[i], (float)at(i, j, e + 2) * f[i], (float)at(i, j, e + 3) * f[i]};
      wave_lds_fence();
      float v[8];
#pragma unroll
      for (int k = 0; k < 8; ++k) v[k] = fmaf(lds[(2 * k + hi) * kTurnRow + c], w[j], b[j]);
      wave_lds_fence();
      const int m = row(i) + hi, n = col(j) + c;
      const long o = (long)m * a.ldy + n;
#pragma unroll
      for (int k = 0; k < 8; ++k) {
        if (m + 2 * k >= a.M || n >= a.N) continue;
        if (a.f32)
          ((float*)a.y)[o + 2 * k * a.ldy] = v[k];
        else
          ((uint16_t*)a.y)[o + 2 * k * a.ldy] = f2bf(v[k]);
      }
    }
}

// ------------------------------------------------------------ few rows: the weight streams by
// A workgroup has 16 columns and up to 16 rows; its eight waves cut K into eight runs and meet in LDS.  What bounds it is the weight's
// way: one row of 28672 x 4096 25 us (4.7 TB/s), of 6144 x 4096 8.2 (2 to 3 of them the launch), of 128256 x 4096 102 (5.1 TB/s); 16 rows
// read x as often as w (143 us), so that others take over.  us of one row of 4096 x 4096 / 28672 x 4096 in other forms: eight steps asked
// for at once 6.7 / 27.4, 16 waves 6.5 / 29.1, waves taking turns over K 6.4 / 30.5, two strips 7.6 / 31.0, non-temporal 5.6 / 24.6,
// this one 5.8 / 23.2.
constexpr int kWaves = 8;
__global__ void __launch_bounds__(64 * kWaves) few_kernel(GemmArgs a) {
  __shared__ i32x4 red[kWaves][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16;
  const uint8_t* const w = a.w + (size_t)min(n0 + r, a.N - 1) * a.ldw;
  const uint8_t* const x = a.x + (size_t)min(r, a.M - 1) * a.ldx;
  const int steps = (a.K + 63) >> 6, per = (steps + kWaves - 1) / kWaves, s1 = min(steps, (wv + 1) * per);
  i32x4 acc = {0, 0, 0, 0};
  constexpr int U = 4;
  for (int s = wv * per; s < s1; s += U) {
    i32x4 wf[U], xf[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // a piece behind the row's end: the row's last one is read again, and zeros of x take it out
      const int k = 64 * (s + u) + 16 * g;
      const bool in = s + u < s1 && k < a.K;
      const int kc = in ? k : a.K - 16;
      wf[u] = *reinterpret_cast<const i32x4*>(w + kc);
      xf[u] = *reinterpret_cast<const i32x4*>(x + kc);
      if (!in) xf[u] = i32x4{0, 0, 0, 0};
    }
#pragma unroll
    for (int u = 0; u < U; ++u) acc = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u], acc, 0, 0, 0);
  }
  red[wv][lane] = acc;
  __syncthreads();
  if (wv) return;
#pragma unroll
  for (int k = 1; k < kWaves; ++k) acc += red[k][lane];
  put4(a, r, n0 + 4 * g, acc);
}

// ------------------------------------------------------------ staging through LDS
// A stage holds rows of 128 bytes of K: 16-byte piece c of row r at c ^ ((r >> 1) & 7), so that the 16 lanes of a fragment's
// read hit 16 different bank groups.  The DMA writes LDS in lane order, so that the exchange is in its source address.
typedef __attribute__((address_space(3))) void lds_t;
template <int POLICY = 0>  // 2: non-temporal
__device__ __forceinline__ void dma16(const uint8_t* src, uint8_t* dst) {
  __builtin_amdgcn_global_load_lds(src, (lds_t*)dst, 16, 0, POLICY);
}
__device__ __forceinline__ void bar() {
  __builtin_amdgcn_sched_barrier(0);
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
}
template <int N>
using ic = std::integral_constant<int, N>;

// Workgroup b of n, such that the workgroups of one XCD (every eighth) have neighbouring numbers.
__device__ __forceinline__ int near_number(int b, int n) {
  const int xcd = b & 7, q = n >> 3, r = n & 7;
  return (xcd < r ? xcd * (q + 1) : r * (q + 1) + (xcd - r) * q) + (b >> 3);
}
// Tile t of n_mt x n_nt, in groups of 4 tiles of M by all of N.
__device__ __forceinline__ void tile_at(int t, int n_mt, int n_nt, int& tm, int& tn) {
  const int per = 4 * n_nt, first = t / per * 4, gm = min(n_mt - first, 4), u = t % per;
  tm = first + u % gm;
  tn = u / gm;
}
__device__ __forceinline__ void put_part(const GemmArgs& a, int slice, int m, int n, const i32x4& v) {
  if (m < a.M && n < a.N) *reinterpret_cast<i32x4*>(a.part + ((size_t)slice * a.M + m) * a.ldp + n) = v;
}

// ------------------------------------------------------------ middle sizes: tiles of BM x BN behind a ring of stages
// Waves 2 x WN; NB stages of 128 bytes of K, NB - 1 of them on their way while one is multiplied; one barrier a stage.  Up to
// 128 rows the weight's way bounds it (48 rows of 128256 x 4096 118 to 134 us, 4.1 to 4.7 TB/s), from then on the stages' way into
// LDS (some 25 bytes a clock and unit): weights from memory, 256 x 4096 x 4096 17.6 us (490 TOP/s), 1024 x 4096 x 4096 28.8 (1190).
template <int BM, int BN, int NB, int WN>
__global__ void __launch_bounds__(128 * WN, 2) ring_kernel(GemmArgs a, int n_mt, int n_nt) {
  constexpr int STAGE = (BM + BN) * 128, I = (BM + BN) / (16 * WN);  // DMAs a wave and stage
  constexpr int FM = BM / 32, FN = BN / (16 * WN);
  __shared__ __attribute__((aligned(1024))) uint8_t sm[NB * STAGE];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int t0 = near_number(blockIdx.x, n_mt * n_nt * a.splits), slice = t0 % a.splits;
  int tm, tn;
  tile_at(t0 / a.splits, n_mt, n_nt, tm, tn);
  const int m0 = tm * BM, n0 = tn * BN;
  const int all = (a.K + 127) >> 7, per = (all + a.splits - 1) / a.splits, kt0 = slice * per, nt = min(all - kt0, per);
  // One row of tiles over an uncut K streams the weight by, and it need not stay in the caches: 17 and 48 rows of 128256 x 4096 take
  // 7 and 4 % less, of 28672 x 4096 7 and 5 % (with K in four runs 4096 x 14336 took 9 % more).
  const bool once = n_mt == 1 && a.splits == 1;

  const uint8_t* src[I];
  int lch[I];
#pragma unroll
  for (int i = 0; i < I; ++i) {
    const int R = 8 * (I * wv + i) + (lane >> 3);  // row of the stage: x's, then w's
    lch[i] = 16 * ((lane & 7) ^ ((R >> 1) & 7));
    src[i] = R < BM ? a.x + (size_t)min(m0 + R, a.M - 1) * a.ldx : a.w + (size_t)min(n0 + R - BM, a.N - 1) * a.ldw;
  }
  auto issue = [&](int stage, int kt) {
    const int k = 128 * (kt0 + kt);
#pragma unroll
    for (int i = 0; i < I; ++i) {
      // (zeros behind K: in both operands, since both may be rows of one tensor that goes on)
      const uint8_t* p = k + lch[i] < a.K ? src[i] + k + lch[i] : reinterpret_cast<const uint8_t*>(&kZeros);
      uint8_t* const to = sm + stage * STAGE + (I * wv + i) * 1024;
      if (once && 8 * (I * wv + i) >= BM)
        dma16<2>(p, to);
      else
        dma16(p, to);
    }
  };
  const int r = lane & 15, g = lane >> 4;
  const int f0 = r * 128 + 16 * (g ^ ((r >> 1) & 7));
  const int wr = wv / WN, wc = wv % WN;
  const int xo = wr * (BM / 2) * 128 + f0, wo = (BM + wc * (BN / WN)) * 128 + f0;
  i32x4 acc[FM][FN] = {};
#pragma unroll
  for (int j = 0; j < NB - 1; ++j) issue(j, min(j, nt - 1));
  for (int i = 0; i < nt; ++i) {
    asm volatile("s_waitcnt vmcnt(%0)" ::"n"((NB - 2) * I) : "memory");
    bar();
    issue((i + NB - 1) % NB, min(i + NB - 1, nt - 1));
    const uint8_t* s = sm + (i % NB) * STAGE;
    i32x4 xf[2][FM], wf[2][FN];
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
#pragma unroll
      for (int f = 0; f < FN; ++f) wf[ks][f] = *reinterpret_cast<const i32x4*>(s + ((wo + 2048 * f) ^ (64 * ks)));
#pragma unroll
      for (int f = 0; f < FM; ++f) xf[ks][f] = *reinterpret_cast<const i32x4*>(s + ((xo + 2048 * f) ^ (64 * ks)));
    }
    __builtin_amdgcn_sched_barrier(0);  // every read is asked for before the first product
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int f = 0; f < FM; ++f)
#pragma unroll
        for (int j = 0; j < FN; ++j) acc[f][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[ks][j], xf[ks][f], acc[f][j], 0, 0, 0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");  // no DMA outlives the workgroup's LDS
  auto row = [&](int f) { return m0 + wr * (BM / 2) + 16 * f + r; };
  auto col = [&](int j) { return n0 + wc * (BN / WN) + 16 * j + 4 * g; };
  if (a.splits > 1) {
#pragma unroll
    for (int f = 0; f < FM; ++f)
#pragma unroll
      for (int j = 0; j < FN; ++j) put_part(a, slice, row(f), col(j), acc[f][j]);
    return;
  }
  if (aligned_rows<4>(a)) {
    put_block<FM, FN, 4>(a, row, col, [&](int f, int j, int e) { return acc[f][j][e]; });
    return;
  }
  bar();  // (every wave is done with the stages)
  static_assert(FN == 2 && (BM + BN) % (16 * WN) == 0, "32 columns and whole DMAs a wave");
  put_turned<FM, 1, 4>(a, reinterpret_cast<float*>(sm) + wv * kTurn, lane, [&](int f) { return m0 + wr * (BM / 2) + 16 * f; },
                       [&](int) { return n0 + wc * (BN / WN); }, [&](int f, int, int e) { return acc[f][e >> 2][e & 3]; });
}

// ------------------------------------------------------------ large: tiles of 256 x 256, eight phases for two stages
// Eight waves, 2 x 4, on one compute unit.  A stage of 128 bytes of K is four half tiles (x rows 0-127 and 128-255, w rows
// likewise) of 16 KB, two stages in LDS.  A stage's product has four phases, one a quadrant of 128 x 128: a phase reads its new
// fragments (8 of x or 4 of w), asks for one half tile of a later stage, and issues 16 matrix instructions; every fragment is
// read once a stage.  Waves 4-7 run one barrier behind waves 0-3, so that on each SIMD one wave multiplies while the other
// reads.  A half tile is asked for two phases after its place was last read and waited for (four half tiles later still on
// their way) one phase before it is read.  Rows of w are staged so that a lane's two fragments are eight neighbouring columns.
// us: 4001 x 28672 x 4096 386 to 414 (2.27 to 2.43 POP/s), 4096 x 4096 x 14336 177 to 180 (2.7), 4096 x 4096 x 4096 59 to 62 (2.3); a large bf16
// product of the library reaches 1.46 PFLOP/s, whose bytes a matrix instruction are the same.  A stage takes 1.5 us, of which the
// matrix instructions are 1.0: LDS moves as much in the time as it can (192 KB read, 64 KB written a stage); 6 us of each tile
// are its start and its stores.  What whole rounds of 256 tiles leave has its K cut: 2048 x 10240 x 8192 (320 tiles) 185 -> 155.
constexpr int HALF = 128 * 128, BUF = 4 * HALF, OX0 = 0, OX1 = HALF, OW0 = 2 * HALF, OW1 = 3 * HALF;
__global__ void __launch_bounds__(512, 1) big_kernel(GemmArgs a, int n_mt, int n_nt) {
  __shared__ __attribute__((aligned(1024))) uint8_t sm[2 * BUF];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int wr = wv >> 2, wc = wv & 3;
  const int b = blockIdx.x;
  const bool cut = b >= a.whole && a.splits > 1;
  const int u0 = near_number(b < a.whole ? b : b - a.whole, b < a.whole ? a.whole : gridDim.x - a.whole);
  const int tile = b < a.whole ? u0 : a.whole + u0 / a.splits, slice = cut ? u0 % a.splits : 0;
  int tm, tn;
  tile_at(tile, n_mt, n_nt, tm, tn);
  const int m0 = tm * 256, n0 = tn * 256;
  // an even count of stages a run: those behind K are zeros
  const int all = (a.K + 127) >> 7, runs = cut ? a.splits : 1, nt = ((all + runs - 1) / runs + 1) & ~1, kt0 = slice * nt;

  const uint8_t* const zeros = reinterpret_cast<const uint8_t*>(&kZeros);
  const uint8_t *xs[2][2], *ws[2][2];
  int lch[2];
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int R = 16 * wv + 8 * i + (lane >> 3), rho = R & 31;
    lch[i] = 16 * ((lane & 7) ^ ((R >> 1) & 7));
#pragma unroll
    for (int h = 0; h < 2; ++h) {
      const int n = n0 + 128 * h + (R & ~31) + 8 * ((rho >> 2) & 3) + 4 * (rho >> 4) + (rho & 3);
      xs[h][i] = a.x + (size_t)min(m0 + 128 * h + R, a.M - 1) * a.ldx + lch[i];
      ws[h][i] = a.w + (size_t)min(n, a.N - 1) * a.ldw + lch[i];
    }
  }
  auto issue = [&](const uint8_t* const* src, int at, int kt) {
    const int k = 128 * (kt0 + kt);
#pragma unroll
    for (int i = 0; i < 2; ++i) dma16(k + lch[i] < a.K ? src[i] + k : zeros, sm + at + (2 * wv + i) * 1024);
  };
  const int r = lane & 15, g = lane >> 4;
  const int f0 = r * 128 + 16 * (g ^ ((r >> 1) & 7));
  const int xo = 64 * wr * 128 + f0, wo = 32 * wc * 128 + f0;
  i32x4 acc[4][4][2] = {};
  i32x4 xf[4][2], wf0[2][2], wf1[2][2];

  issue(xs[0], OX0, 0);
  issue(ws[0], OW0, 0);
  issue(ws[1], OW1, 0);
  issue(xs[1], OX1, 0);
  issue(xs[0], BUF + OX0, 1);
  issue(ws[0], BUF + OW0, 1);
  asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
  bar();
  if (wr == 1) bar();

  auto phase = [&](auto PHc, auto Bc, int u) {
    constexpr int PH = decltype(PHc)::value, B0 = decltype(Bc)::value * BUF, B1 = BUF - B0;
    auto read_x = [&](int at) {
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) xf[i][ks] = *reinterpret_cast<const i32x4*>(sm + B0 + at + ((xo + 2048 * i) ^ (64 * ks)));
    };
    auto read_w = [&](i32x4(&w)[2][2], int at) {
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int ks = 0; ks < 2; ++ks) w[j][ks] = *reinterpret_cast<const i32x4*>(sm + B0 + at + ((wo + 2048 * j) ^ (64 * ks)));
    };
    if constexpr (PH == 1) {
      read_w(wf0, OW0);
      read_x(OX0);
      issue(ws[1], B1 + OW1, min(u + 1, nt - 1));
    } else if constexpr (PH == 2) {
      read_w(wf1, OW1);
      issue(xs[1], B1 + OX1, min(u + 1, nt - 1));
    } else if constexpr (PH == 3) {
      read_x(OX1);
      issue(xs[0], B0 + OX0, min(u + 2, nt - 1));
    } else {
      issue(ws[0], B0 + OW0, min(u + 2, nt - 1));
    }
    if constexpr (PH != 3) asm volatile("s_waitcnt vmcnt(8)" ::: "memory");
    bar();
    __builtin_amdgcn_s_setprio(1);
#pragma unroll
    for (int ks = 0; ks < 2; ++ks)
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 2; ++j) {
          const i32x4 w = PH == 1 || PH == 4 ? wf0[j][ks] : wf1[j][ks];
          acc[PH - 1][i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(w, xf[i][ks], acc[PH - 1][i][j], 0, 0, 0);
        }
    __builtin_amdgcn_s_setprio(0);
    bar();
  };
  for (int u = 0; u < nt; u += 2) {
    phase(ic<1>{}, ic<0>{}, u);
    phase(ic<2>{}, ic<0>{}, u);
    phase(ic<3>{}, ic<0>{}, u);
    phase(ic<4>{}, ic<0>{}, u);
    phase(ic<1>{}, ic<1>{}, u + 1);
    phase(ic<2>{}, ic<1>{}, u + 1);
    phase(ic<3>{}, ic<1>{}, u + 1);
    phase(ic<4>{}, ic<1>{}, u + 1);
  }
  if (wr == 0) bar();
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");

  // quadrant (x half, w half) is 0 (0,0), 1 (0,1), 2 (1,1), 3 (1,0)
  auto row = [&](int i) { return m0 + 128 * (i >> 2) + 64 * wr + 16 * (i & 3) + r; };
  auto col = [&](int j) { return n0 + 128 * j + 32 * wc + 8 * g; };
  auto quad = [](int i, int j) { return i >= 4 ? 3 - j : j; };
  if (cut) {
    int* const p = a.part + ((size_t)(tile - a.whole) * a.splits + slice) * 65536;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 2; ++j)
#pragma unroll
        for (int e = 0; e < 2; ++e)
          *reinterpret_cast<i32x4*>(p + (row(i) - m0) * 256 + col(j) - n0 + 4 * e) = acc[quad(i, j)][i & 3][e];
    return;
  }
  if (aligned_rows<8>(a)) {
    put_block<8, 2, 8>(a, row, col, [&](int i, int j, int e) { return acc[quad(i, j)][i & 3][e >> 2][e & 3]; });
    return;
  }
  bar();  // (every wave is done with the stages)
  put_turned<8, 2, 8>(a, reinterpret_cast<float*>(sm) + wv * kTurn, lane, [&](int i) { return m0 + 128 * (i >> 2) + 64 * wr + 16 * (i & 3); },
                      [&](int j) { return n0 + 128 * j + 32 * wc; }, [&](int i, int j, int e) { return acc[quad(i, j)][i & 3][e >> 2][e & 3]; });
}

// the runs' sums, scaled: four neighbours a thread
__global__ void __launch_bounds__(256) join_kernel(GemmArgs a) {
  const int per = (a.N + 3) >> 2;
  const long i = blockIdx.x * 256L + threadIdx.x;
  if (i >= (long)per * a.M) return;
  const int m = (int)(i / per), n = 4 * (int)(i % per);
  i32x4 s = {0, 0, 0, 0};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) s += *reinterpret_cast<const i32x4*>(a.part + ((size_t)k * a.M + m) * a.ldp + n);
  put4(a, m, n, s);
}

// the same of the cut tiles of 256 x 256: grid (tiles, 64)
__global__ void __launch_bounds__(256) join_big_kernel(GemmArgs a, int n_mt, int n_nt) {
  int tm, tn;
  tile_at(a.whole + blockIdx.x, n_mt, n_nt, tm, tn);
  const int row = 4 * blockIdx.y + (threadIdx.x >> 6), c = 4 * (threadIdx.x & 63);
  if (tm * 256 + row >= a.M || tn * 256 + c >= a.N) return;
  const int* p = a.part + (size_t)blockIdx.x * a.splits * 65536 + row * 256 + c;
  i32x4 s = {0, 0, 0, 0};
#pragma unroll 4
  for (int k = 0; k < a.splits; ++k) s += *reinterpret_cast<const i32x4*>(p + (size_t)k * 65536);
  put4(a, tm * 256 + row, tn * 256 + c, s);
}

// ------------------------------------------------------------ the choice
// Rows and columns of a tile by kind.
constexpr int kEdge[8][2] = {{16, 16}, {32, 64}, {64, 64}, {64, 128}, {128, 64}, {128, 128}, {256, 256}, {128, 256}};

// Estimated us of a product.  Its tiles take rounds over the 256 compute units, a round `per` stages of 128 bytes of K and a fixed part;
// the smaller of the middle tiles lie two on a unit, where a stage takes longer.  Beside that stands the weight's way from memory: the third
// root of the cubes' sum, roughly, since the one hides in the other until they are alike.  Few rows: the weight's way with the
// rows' reads beside it, against the latency of each wave's turns over K (four steps of 64 bytes a turn), and what a workgroup
// costs beside its loads, which shows where K is short.  The constants are a fit to times of every kind and cut at 480 sizes: 1 to
// 4096 rows by 16 weights of 512 x 512 to 128256 x 4096 (K from 512 to 28672), the weights from memory.  The choice is 1.3 % from
// the best one on average; furthest off are 13 and 16 rows of 5120 x 5120, 16.0 and 17.2 us where
// 32 x 64 tiles in four runs take 14.1, and one row of 128256 x 4096, which goes to tiles, 120 us for 102.
// Tiles of 128 x 256 came later (96 sizes, 72 to 1000 rows: 0.4 % from the best one, without them 4.1; 512 rows of 14336 x 4096 take
// 18 % less, 41 us, 128 of 40000 x 4096 15 %, 256 of 28672 x 4096 10 %, 100 of 128256 x 4096 6 %).
inline double cost(int M, int N, int K, int kind, int splits) {
  constexpr double kStart = 2.62, kByte = 0.150e-6, kJoin = 2.46, kJoinByte = 0.328e-6;
  // us a stage alone on a unit, by twos (of the three largest, a round full and nearly empty), a round's fixed part
  constexpr double c[8][3] = {{}, {.260, .434, 1.54}, {.361, .525, 1.44}, {.453, .809, 1.60}, {.592, .800, 2.00}, {.643, .542, 2.61}, {1.44, .995, 5.61}, {1.13, .826, 2.97}};
  const double bytes = (double)N * K;
  if (kind == 0) {
    const double turns = (K + 64 * kWaves * 4 - 1) / (64 * kWaves * 4), stream = bytes * (0.168e-6 + 0.00664e-6 * (M - 1));
    const double wait = turns * (1.04 + 0.0501 * (M - 1));
    return kStart + pow(pow(stream, 4.09) + pow(wait, 4.09), 1 / 4.09) + 0.00247 * ((N + 15) / 16) * (K > 1024 ? 1024. / K : 1.);
  }
  const int stages = (K + 127) / 128, per = (stages + splits - 1) / splits;
  const long tiles = (long)((M - 1) / kEdge[kind][0] + 1) * ((N - 1) / kEdge[kind][1] + 1);
  const double a = c[kind][0], b = c[kind][1], e = c[kind][2];
  double t, joined = (double)splits * M * N;
  if (kind == 6) {
    const long whole = tiles / 256, rest = tiles % 256 * splits;
    t = whole * (stages * a + e) + (rest ? per * (b + (a - b) * rest / 256.) + e : 0);
    joined = 65536. * rest;
  } else if (kind == 5 || kind == 7) {
    const long whole = tiles * splits / 256, rest = tiles * splits % 256;
    t = whole * (per * a + e) + (rest ? per * (b + (a - b) * rest / 256.) + e : 0);
  } else {
    const long whole = tiles * splits / 512, rest = tiles * splits % 512;
    t = whole * (per * b + e) + (rest ? per * (rest > 256 ? b : a) + e : 0);
  }
  return kStart + pow(pow(t, 2.82) + pow(bytes * kByte, 2.82), 1 / 2.82) + (splits > 1 ? kJoin + kJoinByte * 4 * joined : 0);
}
// Whether `splits` runs of K are possible: none of them empty, and of 256 x 256 tiles only as many as the rest of a round holds.
inline bool can_cut(int M, int N, int K, int kind, int splits) {
  if (splits == 1) return true;
  const int stages = (K + 127) / 128, per = (stages + splits - 1) / splits;
  if (kind == 0 || (splits - 1) * per >= stages) return false;
  const long tiles = (long)((M - 1) / kEdge[kind][0] + 1) * ((N - 1) / kEdge[kind][1] + 1);
  return kind == 6 ? tiles % 256 && tiles % 256 * splits <= 256 : tiles * splits <= 2048;
}

template <int BM, int BN, int NB, int WN>
void ring(const GemmArgs& a, hipStream_t st) {
  const int n_mt = (a.M + BM - 1) / BM, n_nt = (a.N + BN - 1) / BN;
  hipLaunchKernelGGL((ring_kernel<BM, BN, NB, WN>), dim3(n_mt * n_nt * a.splits), dim3(128 * WN), 0, st, a, n_mt, n_nt);
}

}  // namespace q8
}  // namespace k8s

// The kernel (kind) and cut of K for these sizes: kind | runs << 8.
K8S_API int k8s_int8_gemm_plan(int M, int N, int K) {
  using namespace k8s::q8;
  static const int runs[] = {1, 2, 3, 4, 6, 8, 12, 16};
  if (M <= 0 || N <= 0 || K <= 0) return 1 << 8;
  double best = 0;
  int plan = 0;
  for (int kind = M <= 16 ? 0 : 1; kind < 8; ++kind)
    for (int s : runs) {
      if (!can_cut(M, N, K, kind, s)) continue;
      const double t = cost(M, N, K, kind, s);
      if (!plan || t < best) best = t, plan = kind | s << 8;
    }
  return plan;
}

// int32 numbers of workspace that the plan needs
K8S_API long k8s_int8_gemm_part(int M, int N, int kind, int splits) {
  using namespace k8s::q8;
  if (splits <= 1 || kind < 0 || kind > 7) return 0;
  const long tiles = (long)((M - 1) / kEdge[kind][0] + 1) * ((N - 1) / kEdge[kind][1] + 1);
  return kind == 6 ? tiles % 256 * splits * 65536L : (long)splits * M * ((N + 7) / 8 * 8);
}

// x [M][ldx], w [N][ldw] int8, 16-byte aligned rows, K % 16 == 0; y bf16, or fp32 with f32.  kind: 0 few rows (M <= 16), then tiles
// of kEdge; those take K in `splits` runs of at least a stage, which leave their sums in `part` (k8s_int8_gemm_part numbers).
K8S_API int k8s_int8_gemm(const void* x, long ldx, const float* xs, const void* w, long ldw, const float* ws, const float* bias, void* y,
                          long ldy, int f32, int M, int N, int K, int kind, int splits, void* part, long parts, void* stream) {
  using namespace k8s::q8;
  if (M <= 0 || N <= 0) return 0;
  if (kind < 0 || kind > 7 || (kind == 0 && M > 16) || K <= 0 || (K & 15) || K > 131056 || splits < 1) return (int)hipErrorInvalidValue;
  if (!can_cut(M, N, K, kind, splits) || (splits > 1 && (!part || parts < k8s_int8_gemm_part(M, N, kind, splits)))) return (int)hipErrorInvalidValue;
  const int n_mt = (M - 1) / kEdge[kind][0] + 1, n_nt = (N - 1) / kEdge[kind][1] + 1;
  if ((long)n_mt * n_nt * splits > 0x7fffffffL || ((long)((N + 3) / 4) * M + 255) / 256 > 0x7fffffffL) return (int)hipErrorInvalidValue;
  GemmArgs a{(const uint8_t*)x, (const uint8_t*)w, xs, ws, bias, y, ldx, ldw, ldy, M, N, K, f32, splits, (int*)part, (N + 7) / 8 * 8, 0};
  hipStream_t st = (hipStream_t)stream;
  switch (kind) {
    case 0: hipLaunchKernelGGL(few_kernel, dim3(n_nt), dim3(64 * kWaves), 0, st, a); break;
    case 1: ring<32, 64, 5, 2>(a, st); break;
    case 2: ring<64, 64, 4, 2>(a, st); break;
    case 3: ring<64, 128, 3, 4>(a, st); break;
    case 4: ring<128, 64, 3, 2>(a, st); break;
    case 5: ring<128, 128, 4, 4>(a, st); break;
    case 7: ring<128, 256, 3, 8>(a, st); break;
    default: {
      // the tiles of whole rounds take all of K; those of the last, partial one are cut
      a.whole = splits > 1 ? n_mt * n_nt / 256 * 256 : n_mt * n_nt;
      const int rest = n_mt * n_nt - a.whole;
      hipLaunchKernelGGL(big_kernel, dim3(a.whole + rest * splits), dim3(512), 0, st, a, n_mt, n_nt);
      if (rest) hipLaunchKernelGGL(join_big_kernel, dim3(rest, 64), dim3(256), 0, st, a, n_mt, n_nt);
      return (int)hipGetLastError();
    }
  }
  if (splits > 1) hipLaunchKernelGGL(join_kernel, dim3((unsigned)(((long)((N + 3) / 4) * M + 255) / 256)), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}
