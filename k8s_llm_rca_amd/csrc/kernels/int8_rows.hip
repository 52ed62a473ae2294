// Rows of 8-bit integers with a scale each (int8_rows.h), made where the rows are:
//   rows:  y = x
//   gate:  y = silu(g) u,                x = [g | u]
//   norm:  y = h w / sqrt(mean h^2 + eps),  h = x (+ r, rounded to the rows' type and written back to r)
// One pass over memory: a row stays in the registers of its threads between its maximum and its integers (rows too long for that are
// read again).  Behind a norm the sum of squares and the maximum of |h w| leave in one exchange: the norm's factor is the
// same for the whole row, so it does not change the integers, only the scale.
// What bounds it is memory: a norm of 8192 x 8192 bf16 with its residual 87 to 92 us (470 MB: 5.1 to 5.4 TB/s; a large copy moves
// 5.1, of which it reads a smaller part), a gate of 4096 x 14336 53 us (5.5 TB/s); a few rows are 3 us of launch, load and exchange.
#include "int8_rows.h"

namespace k8s {
namespace q8 {

struct RowArgs {
  const void* x;
  void* res;
  const void* w;
  uint8_t* q;
  float* scale;
  int T, H;
  long ldx, ldq;  // elements between rows
  float eps;
};

template <typename E>
__device__ __forceinline__ void load8(const E* p, float (&v)[8]) {
  if constexpr (sizeof(E) == 2) {
    const u16x8 a = *reinterpret_cast<const u16x8*>(p);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = bf2f(a[j]);
  } else {
    const f32x4 a = *reinterpret_cast<const f32x4*>(p), b = *reinterpret_cast<const f32x4*>(p + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) v[j] = a[j], v[j + 4] = b[j];
  }
}
template <typename E>
__device__ __forceinline__ void store8(E* p, const float (&v)[8]) {
  if constexpr (sizeof(E) == 2) {
    u16x8 a;
#pragma unroll
    for (int j = 0; j < 8; ++j) a[j] = f2bf(v[j]);
    *reinterpret_cast<u16x8*>(p) = a;
  } else {
    *reinterpret_cast<f32x4*>(p) = f32x4{v[0], v[1], v[2], v[3]};
    *reinterpret_cast<f32x4*>(p + 4) = f32x4{v[4], v[5], v[6], v[7]};
  }
}

enum { ROWS = 0, GATE = 1, NORM = 2 };

// W waves a row; NC pieces of 8 a thread stay in registers (0: the row is read twice)
template <int MODE, typename E, int W, int NC>
__global__ void __launch_bounds__(W >= 4 ? 64 * W : 256) rows_kernel(RowArgs a) {
  constexpr int TPR = 64 * W, RPB = W >= 4 ? 1 : 4 / W;
  const int t = threadIdx.x % TPR;
  const int row = blockIdx.x * RPB + threadIdx.x / TPR;
  if (RPB > 1 && row >= a.T) return;  // (W == 1: no barrier follows)
  const int nv = a.H >> 3;
  const E* const x = (const E*)a.x + (size_t)row * a.ldx;
  E* const r = MODE == NORM && a.res ? (E*)a.res + (size_t)row * a.H : nullptr;
  const E* const w = (const E*)a.w;

  // piece i of the row: y without the norm's factor; `first`: the pass that adds the residual
  float ss = 0.f;
  auto piece = [&](int i, float (&y)[8], bool first) {
    if constexpr (MODE == GATE) {
      float u[8];
      load8(x + 8 * i, y);
      load8(x + a.H + 8 * i, u);
      // (hardware exponential and reciprocal: y and the maximum are off by 2^-18 at most, an integer by a thousandth of its step)
#pragma unroll
      for (int j = 0; j < 8; ++j) y[j] = silu_hw(y[j]) * u[j];
    } else if constexpr (MODE == NORM) {
      float g[8];
      load8(w + 8 * i, g);
      if (r && !first) {
        load8(r + 8 * i, y);
      } else {
        load8(x + 8 * i, y);
        if (r) {
          float b[8];
          load8(r + 8 * i, b);
#pragma unroll
          for (int j = 0; j < 8; ++j) {
            y[j] += b[j];
            if constexpr (sizeof(E) == 2) y[j] = bf2f(f2bf(y[j]));
          }
          store8(r + 8 * i, y);
        }
      }
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        if (first) ss = fmaf(y[j], y[j], ss);
        y[j] *= g[j];
      }
    } else {
      load8(x + 8 * i, y);
    }
  };
  uint32_t top = 0;
  auto largest = [&](const float (&y)[8]) {
#pragma unroll
    for (int j = 0; j < 8; ++j) top = max(top, abs_bits(y[j]));
  };
  float y[NC ? NC : 1][8];
  if constexpr (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = t + c * TPR;
      if (i < nv) {
        piece(i, y[c], true);
        largest(y[c]);
      }
    }
  } else {
    for (int i = t; i < nv; i += TPR) {
      piece(i, y[0], true);
      largest(y[0]);
    }
  }
#pragma unroll
  for (int o = 32; o > 0; o >>= 1) {
    top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    if constexpr (MODE == NORM) ss += __shfl_xor(ss, o, 64);
  }
  if constexpr (W > 1) {
    __shared__ uint32_t tops[W];
    __shared__ float sums[W];
    if ((threadIdx.x & 63) == 0) {
      tops[threadIdx.x >> 6] = top;
      sums[threadIdx.x >> 6] = ss;
    }
    __syncthreads();
    top = 0;
    ss = 0.f;
#pragma unroll
    for (int k = 0; k < W; ++k) {
      top = max(top, tops[k]);
      ss += sums[k];
    }
  }
  Step s = row_step(top, MODE == NORM ? kLeast : kTiny);
  uint8_t* const q = a.q + (size_t)row * a.ldq;
  if constexpr (MODE == NORM) {
    const float f = 1.f / sqrtf(ss / (float)a.H + a.eps);
    s.scale *= f;
    if (__uint_as_float(top) * f < kTiny) s = {0.f, 0.f, 0.f};
    if (!(ss < INFINITY)) s = {0.f, 0.f, __uint_as_float(0x7fc00000u)};  // (squares that left fp32: no zeros for them)
  }
  if (t == 0) a.scale[row] = s.scale;
  if constexpr (NC > 0) {
#pragma unroll
    for (int c = 0; c < NC; ++c) {
      const int i = t + c * TPR;
      if (i < nv) *reinterpret_cast<u32x2*>(q + 8 * i) = pack8(y[c], s);
    }
  } else {
    for (int i = t; i < nv; i += TPR) {
      piece(i, y[0], false);
      *reinterpret_cast<u32x2*>(q + 8 * i) = pack8(y[0], s);
    }
  }
}

// Waves a row.  Few rows wait for their own loads and exchange: a piece a lane, two up to 8192 wide, up to four beyond that.  Many rows fill
// the chip by themselves: fewer waves a row, up to four pieces a lane.  us of a norm with its residual, bf16, the same rows again and
// again, at 32 / 8192 rows: 1024 wide by 1 wave
// 3.7 / 10.0, by 4 3.2 / 16.0; 2048 wide by 1 4.7 / 19.7, by 4 3.2 / 22.2; 4096 wide by 4 3.8 / 37.0, by 8 3.3 / 38.4; 8192 wide by 4
// 4.9 / 77.8, by 8 3.9 / 77.2, by 16 3.9 / 82.1; 14336 wide by 8 4.8 / 156, by 16 4.5 / 152.
template <int MODE, typename E>
int launch(const RowArgs& a, hipStream_t st) {
  const int nv = a.H >> 3;
  const bool many = a.T > 1024;
  if (nv <= (many ? 256 : 64))
    hipLaunchKernelGGL((rows_kernel<MODE, E, 1, 4>), dim3((a.T + 3) / 4), dim3(256), 0, st, a);
  else if (nv <= (many ? 512 : 256))
    hipLaunchKernelGGL((rows_kernel<MODE, E, 4, 4>), dim3(a.T), dim3(256), 0, st, a);
  else if (nv <= 1024)
    hipLaunchKernelGGL((rows_kernel<MODE, E, 8, 4>), dim3(a.T), dim3(512), 0, st, a);
  else if (nv <= 4096)
    hipLaunchKernelGGL((rows_kernel<MODE, E, 16, 4>), dim3(a.T), dim3(1024), 0, st, a);
  else  // (over 32768 wide: the row is read twice)
    hipLaunchKernelGGL((rows_kernel<MODE, E, 16, 0>), dim3(a.T), dim3(1024), 0, st, a);
  return (int)hipGetLastError();
}

}  // namespace q8
}  // namespace k8s

// mode: 0 rows, 1 gate, 2 norm; f32: the rows' type (and the residual's and the norm weight's) is fp32, else bf16.  H % 8 == 0, rows 16-byte aligned.
K8S_API int k8s_int8_rows(int mode, int f32, const void* x, long ldx, void* res, const void* w, void* q, long ldq, float* scale, int T, int H,
                          float eps, void* stream) {
  using namespace k8s::q8;
  if (T <= 0) return 0;
  if (mode < 0 || mode > 2 || H <= 0 || (H & 7) || (mode == NORM && !w)) return (int)hipErrorInvalidValue;
  hipStream_t st = (hipStream_t)stream;
  const long size = f32 ? 4 : 2;
  constexpr int kMost = 1 << 21;  // rows a launch: 2^31 threads (a grid holds fewer than 2^32)
  for (int t0 = 0; t0 < T;) {
    const int n = T - t0 < kMost ? T - t0 : kMost;
    const RowArgs a{(const char*)x + t0 * ldx * size, res ? (char*)res + (long)t0 * H * size : nullptr, w, (uint8_t*)q + t0 * ldq, scale + t0, n, H, ldx,
                    ldq, eps};
    const int rc = mode == ROWS ? (f32 ? launch<ROWS, float>(a, st) : launch<ROWS, uint16_t>(a, st))
                   : mode == GATE ? (f32 ? launch<GATE, float>(a, st) : launch<GATE, uint16_t>(a, st))
                                  : (f32 ? launch<NORM, float>(a, st) : launch<NORM, uint16_t>(a, st));
    if (rc) return rc;
    t0 += n;
  }
  return 0;
}
