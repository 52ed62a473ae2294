// Products of 8-bit rows:  y[m][n] = xs[m] ws[n] sum_k x[m][k] w[n][k] (+ bias[n]),  bf16 or fp32 out.
// The sum is exact: int32 holds K <= 131056 products of 128 128, so that every way of cutting K gives the same bits.
//
// The matrix instruction is v_mfma_i32_16x16x64_i8 with the weight as its first operand: lane l holds 16 bytes of row l & 15
// at byte 16 (l >> 4), and gets the sums of columns 4 (l >> 4) .. + 3 of row l & 15 of x, so that it stores four neighbours.
#include "int8_rows.h"

namespace k8s {
namespace q8 {

struct GemmArgs {
  const uint8_t *x, *w;
  const float *xs, *ws, *bias;
  void* y;
  long ldx, ldw, ldy;
  int M, N, K, f32;
};

// four neighbouring outputs of row m from column n on
__device__ __forceinline__ void put4(const GemmArgs& a, int m, int n, const i32x4& s) {
  if (m >= a.M || n >= a.N) return;
  const float f = a.xs[m];
  float v[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int c = min(n + i, a.N - 1);
    v[i] = (float)s[i] * f * a.ws[c];
    if (a.bias) v[i] += a.bias[c];
  }
  const long at = (long)m * a.ldy + n;
  const bool whole = n + 4 <= a.N;
  if (a.f32) {
    float* const o = (float*)a.y + at;
    if (whole && ((uintptr_t)o & 15) == 0) {
      *reinterpret_cast<f32x4*>(o) = f32x4{v[0], v[1], v[2], v[3]};
      return;
    }
    for (int i = 0; i < 4 && n + i < a.N; ++i) o[i] = v[i];
  } else {
    uint16_t* const o = (uint16_t*)a.y + at;
    if (whole && ((uintptr_t)o & 7) == 0) {
      *reinterpret_cast<u16x4*>(o) = u16x4{f2bf(v[0]), f2bf(v[1]), f2bf(v[2]), f2bf(v[3])};
      return;
    }
    for (int i = 0; i < 4 && n + i < a.N; ++i) o[i] = f2bf(v[i]);
  }
}

// ------------------------------------------------------------ few rows: the weight streams by
// A workgroup has 16 columns and up to 16 MF rows; its eight waves cut K into eight runs and meet in LDS.
constexpr int kWaves = 8;
template <int MF>
__global__ void __launch_bounds__(64 * kWaves) few_kernel(GemmArgs a) {
  __shared__ i32x4 red[kWaves][MF][64];
  const int lane = threadIdx.x & 63, wv = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
  const int r = lane & 15, g = lane >> 4;
  const int n0 = blockIdx.x * 16, m0 = blockIdx.y * 16 * MF;
  const uint8_t* const w = a.w + (size_t)min(n0 + r, a.N - 1) * a.ldw;
  const uint8_t* x[MF];
#pragma unroll
  for (int f = 0; f < MF; ++f) x[f] = a.x + (size_t)min(m0 + 16 * f + r, a.M - 1) * a.ldx;
  const int steps = (a.K + 63) >> 6, per = (steps + kWaves - 1) / kWaves;
  const int s1 = min(steps, (wv + 1) * per);
  i32x4 acc[MF] = {};
  constexpr int U = MF <= 2 ? 4 : 2;
  for (int s = wv * per; s < s1; s += U) {
    i32x4 wf[U], xf[U][MF];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      // a piece behind the row's end: the row's last one is read again, and zeros of x take it out
      const int k = 64 * (s + u) + 16 * g;
      const bool in = s + u < s1 && k < a.K;
      const int kc = in ? k : a.K - 16;
      wf[u] = ldw_nt<i32x4>(w + kc);
#pragma unroll
      for (int f = 0; f < MF; ++f) {
        xf[u][f] = *reinterpret_cast<const i32x4*>(x[f] + kc);
        if (!in) xf[u][f] = i32x4{0, 0, 0, 0};
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int f = 0; f < MF; ++f) acc[f] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[u], xf[u][f], acc[f], 0, 0, 0);
  }
#pragma unroll
  for (int f = 0; f < MF; ++f) red[wv][f][lane] = acc[f];
  __syncthreads();
  for (int i = threadIdx.x; i < 64 * MF; i += 64 * kWaves) {
    const int f = i >> 6, l = i & 63;
    i32x4 s = red[0][f][l];
#pragma unroll
    for (int k = 1; k < kWaves; ++k) s += red[k][f][l];
    put4(a, m0 + 16 * f + (l & 15), n0 + 4 * (l >> 4), s);
  }
}

// ------------------------------------------------------------ tiles of 128 x 128
// Four waves of 64 x 64 each; K in steps of 128 bytes, two stages in LDS (2 x 32 KB) filled through registers.
constexpr int TB = 128, PITCH = 128 + 16;
__global__ void __launch_bounds__(256, 2) tile_kernel(GemmArgs a) {
  __shared__ __attribute__((aligned(16))) uint8_t sm[2][2][TB * PITCH];
  const int tid = threadIdx.x, lane = tid & 63, wv = tid >> 6;
  const int r = lane & 15, g = lane >> 4;
  const int m0 = blockIdx.y * TB, n0 = blockIdx.x * TB;
  const int wm = 64 * (wv >> 1), wn = 64 * (wv & 1);
  i32x4 rx[4], rw[4];
  const int c = tid & 7, row = tid >> 3;  // 16-byte piece c of rows row, row + 32 ..
  auto load = [&](int kt) {
    const int k = 128 * kt + 16 * c;
    const bool in = k < a.K;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int rr = row + 32 * i;
      rx[i] = rw[i] = i32x4{0, 0, 0, 0};
      if (in) {
        rx[i] = *reinterpret_cast<const i32x4*>(a.x + (size_t)min(m0 + rr, a.M - 1) * a.ldx + k);
        rw[i] = *reinterpret_cast<const i32x4*>(a.w + (size_t)min(n0 + rr, a.N - 1) * a.ldw + k);
      }
    }
  };
  auto keep = [&](int b) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      *reinterpret_cast<i32x4*>(&sm[b][0][(row + 32 * i) * PITCH + 16 * c]) = rx[i];
      *reinterpret_cast<i32x4*>(&sm[b][1][(row + 32 * i) * PITCH + 16 * c]) = rw[i];
    }
  };
  i32x4 acc[4][4] = {};
  const int nt = (a.K + 127) >> 7;
  load(0);
  keep(0);
  for (int kt = 0; kt < nt; ++kt) {
    __syncthreads();
    if (kt + 1 < nt) load(kt + 1);
    const int b = kt & 1;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      i32x4 wf[4], xf[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        xf[i] = *reinterpret_cast<const i32x4*>(&sm[b][0][(wm + 16 * i + r) * PITCH + 64 * ks + 16 * g]);
        wf[i] = *reinterpret_cast<const i32x4*>(&sm[b][1][(wn + 16 * i + r) * PITCH + 64 * ks + 16 * g]);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_i32_16x16x64_i8(wf[j], xf[i], acc[i][j], 0, 0, 0);
    }
    if (kt + 1 < nt) keep(b ^ 1);
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) put4(a, m0 + wm + 16 * i + r, n0 + wn + 16 * j + 4 * g, acc[i][j]);
}

}  // namespace q8
}  // namespace k8s

// x [M][ldx], w [N][ldw] int8, 16-byte aligned rows, K % 16 == 0; y bf16, or fp32 with f32.
K8S_API int k8s_int8_gemm(const void* x, long ldx, const float* xs, const void* w, long ldw, const float* ws, const float* bias, void* y,
                          long ldy, int f32, int M, int N, int K, void* stream) {
  using namespace k8s::q8;
  if (M <= 0 || N <= 0) return 0;
  if (K <= 0 || (K & 15) || K > 131056) return (int)hipErrorInvalidValue;
  const GemmArgs a{(const uint8_t*)x, (const uint8_t*)w, xs, ws, bias, y, ldx, ldw, ldy, M, N, K, f32};
  hipStream_t st = (hipStream_t)stream;
  const dim3 strips((N + 15) / 16);
  if (M <= 16)
    hipLaunchKernelGGL(few_kernel<1>, strips, dim3(64 * kWaves), 0, st, a);
  else if (M <= 32)
    hipLaunchKernelGGL(few_kernel<2>, strips, dim3(64 * kWaves), 0, st, a);
  else if (M <= 64)
    hipLaunchKernelGGL(few_kernel<4>, strips, dim3(64 * kWaves), 0, st, a);
  else {
    if ((M + TB - 1) / TB > 65535) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(tile_kernel, dim3((N + TB - 1) / TB, (M + TB - 1) / TB), dim3(256), 0, st, a);
  }
  return (int)hipGetLastError();
}
