// A paged cache of keys and values in 8 bits, one scale a token and head (int8_rows.h):
//   k [blocks][nkv][BS][128], v [blocks][nkv][128][BS] (transposed pages, as in the bf16 cache), scales [blocks][nkv][BS].
// Tokens are rotated and written in one pass: q heads are rotated in place, a k head is rotated in fp32 and quantised from
// there, a v head is quantised as it is.
#include "int8_rows.h"

namespace k8s {
namespace q8 {

struct WriteArgs {
  uint16_t* qkv;
  long ld;
  const int* pos;
  const float* cos_sin;
  const int* slots;
  uint8_t *k, *v;
  float *ks, *vs;
  int T, nq, nkv, BS, max_pos;
  long cap;  // slots of the pool
};

// Eight lanes a head: lane j has dims 8j .. 8j+7 and their partners 64 on.
__global__ void __launch_bounds__(256) write_kernel(WriteArgs a) {
  const int heads = a.nq + 2 * a.nkv, j = threadIdx.x & 7;
  const long unit = (blockIdx.x * 256L + threadIdx.x) >> 3;
  const bool live = unit < (long)a.T * heads;  // (all eight lanes of a head, so that the exchange below has its partners)
  if (!live) return;
  const int t = (int)(unit / heads), h = (int)(unit % heads);
  uint16_t* const p = a.qkv + (size_t)t * a.ld + h * 128 + 8 * j;
  const u16x8 lo = *reinterpret_cast<const u16x8*>(p), hi = *reinterpret_cast<const u16x8*>(p + 64);
  float x[8], y[8];
  if (h < a.nq + a.nkv) {
    // (a position outside the table takes its last row: no read behind it)
    const int ps = min(max(a.pos[t], 0), a.max_pos - 1);
    const float* cs = a.cos_sin + (size_t)ps * 128 + 8 * j;
#pragma unroll
    for (int e = 0; e < 8; ++e) rope_pair(bf2f(lo[e]), bf2f(hi[e]), cs[e], cs[64 + e], x[e], y[e]);
  } else {
#pragma unroll
    for (int e = 0; e < 8; ++e) x[e] = bf2f(lo[e]), y[e] = bf2f(hi[e]);
  }
  if (h < a.nq) {
    u16x8 o0, o1;
#pragma unroll
    for (int e = 0; e < 8; ++e) o0[e] = f2bf(x[e]), o1[e] = f2bf(y[e]);
    *reinterpret_cast<u16x8*>(p) = o0;
    *reinterpret_cast<u16x8*>(p + 64) = o1;
    return;
  }
  uint32_t top = 0;
#pragma unroll
  for (int e = 0; e < 8; ++e) top = max(top, max(abs_bits(x[e]), abs_bits(y[e])));
#pragma unroll
  for (int o = 1; o < 8; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
  const long slot = a.slots ? a.slots[t] : -1;
  if (slot < 0 || slot >= a.cap) return;
  const Step s = row_step(top);
  const u32x2 q0 = pack8(x, s), q1 = pack8(y, s);
  const bool key = h < a.nq + a.nkv;
  const size_t page = (size_t)(slot / a.BS) * a.nkv + (h - a.nq - (key ? 0 : a.nkv));
  const int off = (int)(slot % a.BS);
  if (key) {
    uint8_t* d = a.k + (page * a.BS + off) * 128 + 8 * j;
    *reinterpret_cast<u32x2*>(d) = q0;
    *reinterpret_cast<u32x2*>(d + 64) = q1;
    if (j == 0) a.ks[page * a.BS + off] = s.scale;
  } else {
    uint8_t* d = a.v + (page * 128 + 8 * j) * (size_t)a.BS + off;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[(size_t)e * a.BS] = (uint8_t)(q0[e >> 2] >> (8 * (e & 3)));
      d[(size_t)(64 + e) * a.BS] = (uint8_t)(q1[e >> 2] >> (8 * (e & 3)));
    }
    if (j == 0) a.vs[page * a.BS + off] = s.scale;
  }
}

}  // namespace q8
}  // namespace k8s

// cap: slots of the pool (blocks * BS); a row whose slot is negative or past it is rotated and not kept
K8S_API int k8s_int8_write(void* qkv, long ld, const int* pos, const float* cos_sin, int max_pos, const int* slots, void* k, void* v, float* ks,
                           float* vs, int T, int nq, int nkv, int BS, long cap, void* stream) {
  using namespace k8s::q8;
  if (T <= 0) return 0;
  if (nq < 0 || nkv <= 0 || BS <= 0 || max_pos <= 0) return (int)hipErrorInvalidValue;
  const WriteArgs a{(uint16_t*)qkv, ld, pos, cos_sin, slots, (uint8_t*)k, (uint8_t*)v, ks, vs, T, nq, nkv, BS, max_pos, cap};
  const long blocks = ((long)T * (nq + 2 * nkv) * 8 + 255) / 256;
  if (blocks > 0x7fffffffL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(write_kernel, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a);
  return (int)hipGetLastError();
}
