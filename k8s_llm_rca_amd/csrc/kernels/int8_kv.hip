// A paged cache of keys and values in 8 bits, one scale a token and head (int8_rows.h):
//   k [blocks][nkv][BS][128], v [blocks][nkv][128][BS] (transposed pages, as in the bf16 cache), scales [blocks][nkv][BS].
// Tokens are rotated and written in one pass: q heads are rotated in place, a k head is rotated in fp32 and quantised from
// there, a v head is quantised as it is.  What bounds it is memory: 8000 rows of 32 + 2 x 8 heads 43 us
// (five sequences; 181 MB: 4.2 TB/s); rows of
// many pages the single bytes of their values (1024 rows in as many pages 34 us).
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

constexpr int kTokens = 64, kCols = kTokens + 16, kPitch = 84;  // of a workgroup that writes values; bytes of its LDS rows

// Whether the row is kept, and where.
__device__ __forceinline__ int slot_of(const WriteArgs& a, int t) {
  const int s = t < a.T && a.slots ? a.slots[t] : -1;
  return s < a.cap ? s : -1;
}

// Eight lanes a head (lane j has dims 8j .. 8j+7 and their partners 64 on), which read their cosines once for all heads that they
// take; a token's heads go by eights to `parts` waves in turn, of which this is wave `part`.  VALUES: the value heads, too,
// byte by byte.
template <bool VALUES>
__device__ __forceinline__ void rotate(const WriteArgs& a, int t, int part, int parts, int lane) {
  if (t >= a.T) return;
  const int j = lane & 7, heads = a.nq + (VALUES ? 2 : 1) * a.nkv;
  uint16_t* const row = a.qkv + (size_t)t * a.ld + 8 * j;
  // (a position outside the table takes its last row: no read behind it)
  const float* const cs = a.cos_sin + (size_t)min(max(a.pos[t], 0), a.max_pos - 1) * 128 + 8 * j;
  const int slot = slot_of(a, t), blk = max(slot, 0) / a.BS, off = max(slot, 0) - blk * a.BS;
  f32x4 co[2], si[2];
#pragma unroll
  for (int e = 0; e < 2; ++e) {
    co[e] = *reinterpret_cast<const f32x4*>(cs + 4 * e);
    si[e] = *reinterpret_cast<const f32x4*>(cs + 64 + 4 * e);
  }
  constexpr int U = 5;
  for (int h0 = 8 * part + (lane >> 3); h0 < heads; h0 += 8 * U * parts) {
    u16x8 lo[U], hi[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint16_t* const p = row + min(h0 + 8 * u * parts, heads - 1) * 128;
      lo[u] = *reinterpret_cast<const u16x8*>(p);
      hi[u] = *reinterpret_cast<const u16x8*>(p + 64);
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int h = h0 + 8 * u * parts;
      if (h >= heads) break;
      float x[8], y[8];
      const bool turned = !VALUES || h < a.nq + a.nkv;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        x[e] = bf2f(lo[u][e]), y[e] = bf2f(hi[u][e]);
        if (turned) rope_pair(x[e], y[e], co[e >> 2][e & 3], si[e >> 2][e & 3], x[e], y[e]);
      }
      if (h < a.nq) {
        u16x8 o0, o1;
#pragma unroll
        for (int e = 0; e < 8; ++e) o0[e] = f2bf(x[e]), o1[e] = f2bf(y[e]);
        *reinterpret_cast<u16x8*>(row + h * 128) = o0;
        *reinterpret_cast<u16x8*>(row + h * 128 + 64) = o1;
        continue;
      }
      uint32_t top = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) top = max(top, max(abs_bits(x[e]), abs_bits(y[e])));
#pragma unroll
      for (int o = 1; o < 8; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
      if (slot < 0) continue;
      const Step s = row_step(top);
      const u32x2 q0 = pack8(x, s), q1 = pack8(y, s);
      const size_t page = (size_t)blk * a.nkv + h - a.nq - (turned ? 0 : a.nkv), at = page * a.BS + off;
      if (turned) {
        *reinterpret_cast<u32x2*>(a.k + at * 128 + 8 * j) = q0;
        *reinterpret_cast<u32x2*>(a.k + at * 128 + 64 + 8 * j) = q1;
      } else {
        uint8_t* const d = a.v + (page * 128 + 8 * j) * a.BS + off;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          d[(size_t)e * a.BS] = (uint8_t)(q0[e >> 2] >> (8 * (e & 3)));
          d[(size_t)(64 + e) * a.BS] = (uint8_t)(q1[e >> 2] >> (8 * (e & 3)));
        }
      }
      if (j == 0) (turned ? a.ks : a.vs)[at] = s.scale;
    }
  }
}

// Values of up to 64 rows of one head, turned in LDS: a dim's tokens lie side by side in a page, so that 16 rows whose slots
// follow one another from a multiple of 16 on leave as 16 bytes a dim; of others fours that do so as 4 bytes, the rest byte by
// byte.  Column c of a dim is row c - (first row's slot mod 16), which lines the runs up.  us with the fours / without: 1055 rows of
// 81 sequences, 16 + 2 x 16 heads, 14.5 / 21.5, 2652 of 22 17.1 / 22.4, 8000 of 5, 32 + 2 x 8 heads, 47.1 / 51.9.
__device__ __forceinline__ void values(const WriteArgs& a, int t0, int head) {
  __shared__ alignas(16) uint8_t sm[128 * kPitch];  // (read as words)
  __shared__ int slots[kCols], whole[kCols / 16], piece[kCols];
  __shared__ size_t first[kCols];  // where the column's first dim lies in the cache
  const int tid = threadIdx.x, j = tid & 7;
  u16x8 in[kTokens / 32][2];
#pragma unroll
  for (int i = 0; i < kTokens / 32; ++i) {
    const uint16_t* const p = a.qkv + (size_t)min(t0 + 32 * i + (tid >> 3), a.T - 1) * a.ld + (a.nq + a.nkv + head) * 128 + 8 * j;
    in[i][0] = *reinterpret_cast<const u16x8*>(p);
    in[i][1] = *reinterpret_cast<const u16x8*>(p + 64);
  }
  const int shift = max(slot_of(a, t0), 0) & 15;
  int mine = -1;
  if (tid < 128) {
    mine = tid >= shift && tid < shift + kTokens ? slot_of(a, t0 + tid - shift) : -1;
    const int blk = max(mine, 0) / a.BS;
    if (tid < kCols) {
      slots[tid] = mine;
      first[tid] = ((size_t)blk * a.nkv + head) * 128 * a.BS + max(mine, 0) - blk * a.BS;
    }
    // sixteen columns that follow one another from a multiple of 16 on (as a page is one, they share it)
    const int lead = __shfl(mine, tid & 48, 64);
    const uint64_t run = __ballot(lead >= 0 && (lead & 15) == 0 && mine == lead + (tid & 15));
    if (tid < kCols && (tid & 15) == 0) whole[tid >> 4] = ((run >> (tid & 63)) & 0xffff) == 0xffff;
  }
  __syncthreads();
  if (tid < kCols) {  // bytes that leave from this column: four, if their slots are a whole piece of four, else its own, if no such piece has it
    const int s = slots[tid], b = tid - (s & 3);
    bool four = s >= 0 && b >= 0 && b + 3 < kCols;
    if (four)
      for (int e = 0; e < 4; ++e) four &= slots[b + e] == s - (s & 3) + e;
    piece[tid] = s < 0 ? 0 : !four ? 1 : s & 3 ? 0 : 4;
  }
#pragma unroll
  for (int i = 0; i < kTokens / 32; ++i) {
    const int row = 32 * i + (tid >> 3);
    float x[8], y[8];
    uint32_t top = 0;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      x[e] = bf2f(in[i][0][e]), y[e] = bf2f(in[i][1][e]);
      top = max(top, max(abs_bits(x[e]), abs_bits(y[e])));
    }
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) top = max(top, (uint32_t)__shfl_xor((int)top, o, 64));
    const Step s = row_step(top);
    const u32x2 q0 = pack8(x, s), q1 = pack8(y, s);
    uint8_t* const d = sm + 8 * j * kPitch + shift + row;
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      d[e * kPitch] = (uint8_t)(q0[e >> 2] >> (8 * (e & 3)));
      d[(64 + e) * kPitch] = (uint8_t)(q1[e >> 2] >> (8 * (e & 3)));
    }
    const int slot = slots[shift + row];
    if (j == 0 && slot >= 0) {
      const int blk = slot / a.BS;
      a.vs[((size_t)blk * a.nkv + head) * a.BS + slot - blk * a.BS] = s.scale;
    }
  }
  __syncthreads();
  for (int i = tid; i < 128 * (kCols / 16); i += 256) {
    const int d = i / (kCols / 16), g = i % (kCols / 16);
    if (!whole[g]) continue;
    const uint32_t* const p = reinterpret_cast<const uint32_t*>(sm + d * kPitch + 16 * g);
    *reinterpret_cast<u32x4*>(a.v + first[16 * g] + (size_t)d * a.BS) = u32x4{p[0], p[1], p[2], p[3]};
  }
  // (a lane a dim here: all lanes of a wave do the same)
  for (int g = 0; g < kCols / 16; ++g) {
    if (whole[g]) continue;
    const int d = tid & 127, c0 = 16 * g + 8 * (tid >> 7);
#pragma unroll
    for (int e = 0; e < 8; ++e) {
      const int n = __builtin_amdgcn_readfirstlane(piece[c0 + e]);
      const uint8_t* const p = sm + d * kPitch + c0 + e;
      uint8_t* const to = a.v + first[c0 + e] + (size_t)d * a.BS;
      if (n == 4)
        *reinterpret_cast<uint32_t*>(to) = pack4(p[0], p[1], p[2], p[3]);
      else if (n)
        *to = *p;
    }
  }
}

// TURN: the first v_blocks workgroups have the values, the others four waves of rotations each.
template <bool TURN>
__global__ void __launch_bounds__(256) write_kernel(WriteArgs a, int v_blocks, int parts) {
  const int b = blockIdx.x;
  if constexpr (TURN)
    if (b < v_blocks) return values(a, b / a.nkv * kTokens, b % a.nkv);
  const int w = (b - v_blocks) * 4 + (threadIdx.x >> 6);
  rotate<!TURN>(a, w / parts, w % parts, parts, threadIdx.x & 63);
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
  // The turn through LDS pays from some tokens and heads on.  us byte by byte / turned, rows of one sequence: 32 + 2 x 8 heads at 512 rows
  // 7.9 / 7.7, 768 10.8 / 8.2; 8 + 2 x 1 heads at 4096 rows 9.7 / 8.8, 6000 12.3 / 10.0; 16 + 2 x 16 heads at 256 rows 7.5 / 6.9.  Of 13
  // rows a sequence: 32 + 2 x 8 heads at 512 rows 9.8 / 10.3, 768 11.8 / 10.9; 8 + 2 x 1 heads at 4096 9.9 / 11.2; 16 + 2 x 16 heads
  // at 128 rows 6.7 / 9.0, 400 11.2 / 9.9.  Of one row: 32 + 2 x 8 heads at 512 rows 11.2 / 13.8, 1024 34.8 / 34.8, 2000 82.5 / 75.2.
  const bool turn = slots && (long)T * nkv >= 5000;
  // few tokens: a wave eight heads, so that no wave takes them one after another (one row of 32 + 2 x 8 heads 4.8 -> 3.3 us, 128 rows
  // 7.0 -> 4.2)
  const int eights = (nq + (turn || !slots ? 1 : 2) * nkv + 7) / 8, parts = T >= 2048 ? 1 : T * eights <= 2048 ? eights : 2048 / T;
  const long v_blocks = turn ? ((long)T + kTokens - 1) / kTokens * nkv : 0, blocks = v_blocks + ((long)T * parts + 3) / 4;
  if (blocks > 0x7fffffffL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(turn ? write_kernel<true> : write_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, (hipStream_t)stream, a, (int)v_blocks, parts);
  return (int)hipGetLastError();
}
