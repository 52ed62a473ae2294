// Attention over the 8-bit paged cache (int8_kv.hip), for reply tokens and for chunks of prompts:
//   S = scale ks[j] (q . k[j]),  O = sum_j softmax(S)[j] vs[j] v[j],  key j of row t visible while j < ctx - qlen + t + 1.
// An int8 is a bf16 exactly, so that both products run on the bf16 matrix instructions with the integers as they are: the
// key's scale multiplies its score, the value's scale the weight, which is rounded to bf16 with it (the one rounding that is
// not fp32's: 2^-9 of a weight, as the bf16 cache's attention has it).
//
// A wave holds 16 rows (token, q head) of one kv head and walks 64 keys at a time.  v_mfma_f32_16x16x32_bf16, S^T = K Q^T:
// row rho of key tile (u, t) is key 16 (rho >> 2) + 8 u + 4 t + (rho & 3), so that lane group g = lane >> 4 is left with the
// scores of keys 16 g .. 16 g + 15, whose values of one dim are one 16-byte load, and weights go to the second product
// without leaving their lane.  Dims of K and Q are taken as 64 c + 16 g + [0, 16) by lane group g: one 16-byte load, two steps.
#include "int8_rows.h"

namespace k8s {
namespace q8 {

constexpr int D = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnArgs {
  const uint16_t* q;
  long ldq;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int* bt;       // [S][bt_stride] block ids
  int bt_stride, NB;   // (a context behind the table's end, a page outside the pool: clamped, never read)
  const int *ctx, *q_start;
  int S, nq, nkv, G, BS;
  float scale_log2;
  uint16_t* out;
  long ldo;
  // replies: a list of (row, part | -1, end key, q row | (tokens - 1) << 24), parts of part_size keys
  const int4* items;
  int n_items;
  const int* d_items;  // {items, keys a part} on the device, or null
  float *part_o, *part_ml;
  int n_parts, part_size;
  // chunks: tiles of rows and runs of 64-key pages
  const int *tile_seq, *tile_tok0, *tile_len, *tile_kv0, *tile_kv1, *tile_slot;
  int n_tiles, tile_waves;
  const int *m_tok0, *m_len, *m_slot0, *m_np;
  int n_merge, slot_rows;
};

struct State {
  bf16x8 qf[4];
  f32x4 o[8];
  float m, l;  // running maximum (log2) of row lane & 15, this lane's part of its sum
};

__device__ __forceinline__ void load_q(State& st, const AttnArgs& a, long row, int head, bool valid, int g) {
  const uint16_t* p = a.q + row * a.ldq + head * D + 16 * g;
#pragma unroll
  for (int c = 0; c < 2; ++c)
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      u16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
      if (valid) z = *reinterpret_cast<const u16x8*>(p + 64 * c + 8 * s);
      st.qf[2 * c + s] = __builtin_bit_cast(bf16x8, z);
    }
#pragma unroll
  for (int d = 0; d < 8; ++d) st.o[d] = f32x4{0.f, 0.f, 0.f, 0.f};
  st.m = -INFINITY;
  st.l = 0.f;
}

// Keys [k0, k1) (k0 a multiple of 64) of one sequence; row lane & 15 sees keys below lim, every row those below kmin.
__device__ __forceinline__ void walk(State& st, const AttnArgs& a, const int* bt, int kvh, int k0, int k1, int kmin, int lim, int lane) {
  const int r = lane & 15, g = lane >> 4;
  for (int kb = k0; kb < k1; kb += 64) {
    const int blk = min(max(__builtin_amdgcn_readfirstlane(bt[kb / a.BS]), 0), a.NB - 1);
    const size_t page = (size_t)blk * a.nkv + kvh;
    const int off = kb % a.BS;
    const uint8_t* kp = a.k + (page * a.BS + off) * D + 16 * g;
    const uint8_t* vp = a.v + page * D * a.BS + off + 16 * g;
    const float* ksp = a.ks + page * a.BS + off + 16 * g;
    const float* vsp = a.vs + page * a.BS + off + 16 * g;
    u32x4 kf[4][2], vf[8];
    f32x4 ks[4], vs[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      const int key = 16 * (r >> 2) + 4 * t + (r & 3);
#pragma unroll
      for (int c = 0; c < 2; ++c) kf[t][c] = *reinterpret_cast<const u32x4*>(kp + key * D + 64 * c);
      ks[t] = *reinterpret_cast<const f32x4*>(ksp + 4 * t);
      vs[t] = *reinterpret_cast<const f32x4*>(vsp + 4 * t);
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) vf[d] = *reinterpret_cast<const u32x4*>(vp + (16 * d + r) * a.BS);
    f32x4 sc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16x8(kf[t][c][0], kf[t][c][1]), st.qf[2 * c], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16x8(kf[t][c][2], kf[t][c][3]), st.qf[2 * c + 1], acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] = acc[i] * (ks[t][i] * a.scale_log2);
    }
    if (kb + 64 > kmin) {  // keys that a row does not see: no weight, whatever stands there (a scale may be a NaN)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          if (kb + 16 * g + 4 * t + i >= lim) sc[t][i] = -INFINITY;
          if (kb + 16 * g + 4 * t + i >= k1) vs[t][i] = 0.f;
        }
    }
    float top = -INFINITY;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) top = fmaxf(top, sc[t][i]);
    top = fmaxf(top, __shfl_xor(top, 16, 64));
    top = fmaxf(top, __shfl_xor(top, 32, 64));
    // the maximum moves only when it would grow by more than 8: weights up to 2^8, and O is seldom rescaled
    const bool up = top > st.m + 8.f;
    const float m = up ? top : st.m;
    const float alpha = up ? __builtin_amdgcn_exp2f(st.m - m) : 1.f;
    const float sub = m == -INFINITY ? 0.f : m;
    bf16x8 pf[2];
    float sum = 0.f;
#pragma unroll
    for (int t = 0; t < 4; ++t)
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float e = __builtin_amdgcn_exp2f(sc[t][i] - sub);
        sum += e;
        // (a row's own limit may lie in front of the wave's: its weight there is zero, and so is the product, unless the scale is a NaN)
        pf[t >> 1][4 * (t & 1) + i] = (__bf16)(sc[t][i] == -INFINITY ? 0.f : e * vs[t][i]);
      }
    st.l = st.l * alpha + sum;
    st.m = m;
    if (__ballot(up)) {
      float ar[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) ar[i] = __shfl(alpha, 4 * g + i, 64);
#pragma unroll
      for (int d = 0; d < 8; ++d)
#pragma unroll
        for (int i = 0; i < 4; ++i) st.o[d][i] *= ar[i];
    }
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[0], to_bf16x8(vf[d][0], vf[d][1]), st.o[d], 0, 0, 0);
      st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[1], to_bf16x8(vf[d][2], vf[d][3]), st.o[d], 0, 0, 0);
    }
  }
}

// rows 4 g + i of the wave: their maxima and whole sums
__device__ __forceinline__ void row_stats(const State& st, int g, float (&m)[4], float (&l)[4]) {
  float s = st.l + __shfl_xor(st.l, 16, 64);
  s += __shfl_xor(s, 32, 64);
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    m[i] = __shfl(st.m, 4 * g + i, 64);
    l[i] = __shfl(s, 4 * g + i, 64);
  }
}
__device__ __forceinline__ void put_row(const State& st, int i, float f, uint16_t* o, int r) {
#pragma unroll
  for (int d = 0; d < 8; ++d) o[16 * d + r] = f2bf(st.o[d][i] * f);
}
__device__ __forceinline__ void put_part(const State& st, int i, float m, float l, float* o, float* ml, int r) {
#pragma unroll
  for (int d = 0; d < 8; ++d) o[16 * d + r] = st.o[d][i];
  if (r == 0) {
    ml[0] = m;
    ml[1] = l;
  }
}

// ------------------------------------------------------------------ replies
__global__ void __launch_bounds__(64, 2) reply_kernel(AttnArgs a) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int n_items = a.d_items ? __builtin_amdgcn_readfirstlane(a.d_items[0]) : a.n_items;
  const int part_size = a.d_items ? __builtin_amdgcn_readfirstlane(a.d_items[1]) : a.part_size;
  const int total = n_items * a.nkv;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int it = w / a.nkv, kvh = w - it * a.nkv;
    const int4 item = a.items[it];
    const int seq = item.x, k1 = min(item.z, a.bt_stride * a.BS), qrow = item.w & 0xFFFFFF, nt = (item.w >> 24) + 1;
    const bool whole = item.y < 0;
    const int part = whole ? 0 : item.y, k0 = part * part_size;
    const int qi = r / a.G;
    const bool valid = qi < nt;
    int lim = k1, kmin = k1;
    if (nt > 1) {
      lim = min(k1, a.ctx[seq + min(qi, nt - 1)]);
      kmin = min(k1, __builtin_amdgcn_readfirstlane(a.ctx[seq]));
    }
    State st;
    load_q(st, a, qrow + (valid ? qi : 0), kvh * a.G + (valid ? r - qi * a.G : 0), valid, g);
    walk(st, a, a.bt + (size_t)seq * a.bt_stride, kvh, k0, k1, kmin, lim, lane);
    float m[4], l[4];
    row_stats(st, g, m, l);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int row = 4 * g + i;
      if (row >= nt * a.G) continue;
      const int ti = row / a.G, head = kvh * a.G + row - ti * a.G;
      if (whole) {
        put_row(st, i, l[i] == 0.f ? 0.f : 1.f / l[i], a.out + (qrow + ti) * a.ldo + head * D, r);
      } else {
        const size_t at = ((size_t)(seq + ti) * a.nq + head) * a.n_parts + part;
        put_part(st, i, m[i], l[i], a.part_o + at * D, a.part_ml + at * 2, r);
      }
    }
  }
  // rows without a key are on no list
  for (int s = blockIdx.x; s < a.S; s += gridDim.x)
    if (a.ctx[s] <= 0)
      for (int c = lane; c < a.nq * D; c += 64) a.out[a.q_start[s] * a.ldo + c] = 0;
}

// rows of more than one part: grid (nq, S), a thread a dim
__global__ void __launch_bounds__(D) reply_merge_kernel(AttnArgs a) {
  const int head = blockIdx.x, seq = blockIdx.y, d = threadIdx.x;
  const int part_size = a.d_items ? a.d_items[1] : a.part_size;
  const int np = min(a.n_parts, (a.ctx[seq] + part_size - 1) / part_size);
  if (np <= 1) return;
  const size_t at = ((size_t)seq * a.nq + head) * a.n_parts;
  float M = -INFINITY, L = 0.f, O = 0.f;
  for (int p = 0; p < np; ++p) M = fmaxf(M, a.part_ml[(at + p) * 2]);
  for (int p = 0; p < np; ++p) {
    const float m = a.part_ml[(at + p) * 2], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    L = fmaf(a.part_ml[(at + p) * 2 + 1], f, L);
    O = fmaf(a.part_o[(at + p) * D + d], f, O);
  }
  a.out[a.q_start[seq] * a.ldo + head * D + d] = f2bf(L == 0.f ? 0.f : O / L);
}

// ------------------------------------------------------------------ chunks
// grid: tiles * nkv * tile_waves, a wave each
__global__ void __launch_bounds__(64, 2) chunk_kernel(AttnArgs a) {
  const int lane = threadIdx.x, r = lane & 15, g = lane >> 4;
  const int w = blockIdx.x % a.tile_waves, kvh = blockIdx.x / a.tile_waves % a.nkv, tile = blockIdx.x / a.tile_waves / a.nkv;
  const int seq = a.tile_seq[tile], tok0 = a.tile_tok0[tile], len = a.tile_len[tile], rows = len * a.G;
  if (16 * w >= rows) return;
  const int qs = a.q_start[seq], base = a.ctx[seq] - (a.q_start[seq + 1] - qs) + (tok0 - qs);
  const int row = 16 * w + r, tt = min(row, rows - 1) / a.G, head = kvh * a.G + min(row, rows - 1) % a.G;
  const bool valid = row < rows;
  const int lo = 16 * w / a.G, hi = min(rows - 1, 16 * w + 15) / a.G;
  const int k0 = a.tile_kv0[tile] * 64, k1 = max(k0, (int)min(min((long)base + hi + 1, a.tile_kv1[tile] * 64L), (long)a.bt_stride * a.BS));
  State st;
  load_q(st, a, tok0 + tt, head, valid, g);
  walk(st, a, a.bt + (size_t)seq * a.bt_stride, kvh, k0, k1, base + lo + 1, base + tt + 1, lane);
  float m[4], l[4];
  row_stats(st, g, m, l);
  const int slot = a.tile_slot[tile];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int rr = 16 * w + 4 * g + i;
    if (rr >= rows) continue;
    if (slot < 0) {
      put_row(st, i, l[i] == 0.f ? 0.f : 1.f / l[i], a.out + (long)(tok0 + rr / a.G) * a.ldo + (kvh * a.G + rr % a.G) * D, r);
    } else {
      const size_t at = ((size_t)slot * a.nkv + kvh) * a.slot_rows + rr;
      put_part(st, i, m[i], l[i], a.part_o + at * D, a.part_ml + at * 2, r);
    }
  }
}

// grid (n_merge * nkv, rows / 2): two rows a workgroup, a thread a dim
__global__ void __launch_bounds__(2 * D) chunk_merge_kernel(AttnArgs a) {
  const int kvh = blockIdx.x % a.nkv, mi = blockIdx.x / a.nkv, row = blockIdx.y * 2 + (threadIdx.x >> 7), d = threadIdx.x & (D - 1);
  if (row >= a.m_len[mi] * a.G) return;
  const int slot0 = a.m_slot0[mi], np = a.m_np[mi];
  float M = -INFINITY, L = 0.f, O = 0.f;
  auto at = [&](int p) { return ((size_t)(slot0 + p) * a.nkv + kvh) * a.slot_rows + row; };
  for (int p = 0; p < np; ++p) M = fmaxf(M, a.part_ml[at(p) * 2]);
  for (int p = 0; p < np; ++p) {
    const float m = a.part_ml[at(p) * 2], f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
    L = fmaf(a.part_ml[at(p) * 2 + 1], f, L);
    O = fmaf(a.part_o[at(p) * D + d], f, O);
  }
  a.out[(long)(a.m_tok0[mi] + row / a.G) * a.ldo + (kvh * a.G + row % a.G) * D + d] = f2bf(L == 0.f ? 0.f : O / L);
}

}  // namespace q8
}  // namespace k8s

K8S_API int k8s_int8_attn_reply(const void* q, long ldq, const void* k, const void* v, const float* ks, const float* vs, int NB, const int* bt,
                                int bt_stride, const int* ctx, const int* q_start, int S, int nq, int nkv, int BS, float scale, void* out,
                                long ldo, float* part_o, float* part_ml, int n_parts, int part_size, const void* items, int n_items,
                                const int* d_items, int grid, void* stream) {
  using namespace k8s::q8;
  if (S <= 0) return 0;
  if (nkv <= 0 || nq % nkv || nq / nkv > 16 || BS <= 0 || (BS & 63) || grid <= 0 || NB <= 0) return (int)hipErrorInvalidValue;
  if (n_parts > 1 && (!part_o || !part_ml || part_size <= 0 || (part_size & 63))) return (int)hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const uint16_t*)q, a.ldq = ldq, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs, a.bt = bt;
  a.bt_stride = bt_stride, a.NB = NB, a.ctx = ctx, a.q_start = q_start, a.S = S, a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.BS = BS;
  a.scale_log2 = scale * kLog2e, a.out = (uint16_t*)out, a.ldo = ldo, a.part_o = part_o, a.part_ml = part_ml, a.n_parts = n_parts;
  a.part_size = part_size, a.items = (const int4*)items, a.n_items = n_items, a.d_items = d_items;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(reply_kernel, dim3(grid), dim3(64), 0, st, a);
  if (n_parts > 1) hipLaunchKernelGGL(reply_merge_kernel, dim3(nq, S), dim3(D), 0, st, a);
  return (int)hipGetLastError();
}

// tiles of up to `rows` (token, q head) rows; split tiles leave parts of slot_rows rows a slot and kv head
K8S_API int k8s_int8_attn_chunk(const void* q, long ldq, const void* k, const void* v, const float* ks, const float* vs, int NB, const int* bt,
                                int bt_stride, const int* ctx, const int* q_start, int nq, int nkv, int BS, float scale, void* out, long ldo,
                                const int* tile_seq, const int* tile_tok0, const int* tile_len, const int* tile_kv0, const int* tile_kv1,
                                const int* tile_slot, int n_tiles, int rows, const int* m_tok0, const int* m_len, const int* m_slot0,
                                const int* m_np, int n_merge, float* part_o, float* part_ml, int slot_rows, void* stream) {
  using namespace k8s::q8;
  if (n_tiles <= 0) return 0;
  if (nkv <= 0 || nq % nkv || BS <= 0 || (BS & 63) || NB <= 0 || rows <= 0 || rows > slot_rows) return (int)hipErrorInvalidValue;
  if (n_merge > 0 && (!part_o || !part_ml)) return (int)hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const uint16_t*)q, a.ldq = ldq, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs, a.bt = bt;
  a.bt_stride = bt_stride, a.NB = NB, a.ctx = ctx, a.q_start = q_start, a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.BS = BS;
  a.scale_log2 = scale * kLog2e, a.out = (uint16_t*)out, a.ldo = ldo, a.part_o = part_o, a.part_ml = part_ml;
  a.tile_seq = tile_seq, a.tile_tok0 = tile_tok0, a.tile_len = tile_len, a.tile_kv0 = tile_kv0, a.tile_kv1 = tile_kv1, a.tile_slot = tile_slot;
  a.n_tiles = n_tiles, a.tile_waves = (rows + 15) / 16, a.m_tok0 = m_tok0, a.m_len = m_len, a.m_slot0 = m_slot0, a.m_np = m_np;
  a.n_merge = n_merge, a.slot_rows = slot_rows;
  hipStream_t st = (hipStream_t)stream;
  const long blocks = (long)n_tiles * nkv * a.tile_waves;
  if (blocks > 0x7fffffffL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(chunk_kernel, dim3((unsigned)blocks), dim3(64), 0, st, a);
  if (n_merge > 0) hipLaunchKernelGGL(chunk_merge_kernel, dim3(n_merge * nkv, (rows + 1) / 2), dim3(2 * D), 0, st, a);
  return (int)hipGetLastError();
}
