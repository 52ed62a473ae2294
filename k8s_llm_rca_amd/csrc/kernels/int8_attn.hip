// Attention over the 8-bit paged cache (int8_kv.hip), for reply tokens and for chunks of prompts:
//   S = scale ks[j] (q . k[j]),  O = sum_j softmax(S)[j] vs[j] v[j],  key j of row t visible while j < ctx - qlen + t + 1.
// An int8 is a bf16 exactly, so that both products run on the bf16 matrix instructions with the integers as they are: the
// key's scale multiplies its score, the value's scale the weight, which is rounded to bf16 with it (the one rounding that is
// not fp32's: 2^-8 of a weight, as the bf16 cache's attention has it).  Maxima, sums and O are fp32's.
//
// Replies: a wave holds 16 rows (token, q head) of one kv head and walks 64 keys at a time, a run of keys of a list that the host
// made (long contexts in parts, which meet in a second launch).  What bounds it is the cache's way from memory: 96 replies over 1500
// to 6000 keys of 8 heads 148 + 5 us, 5.3 TB/s (a large weight alone is read at 6.9); one reply over 5003 keys 8 + 4 us, which is
// latency: loads, softmax and exchange of two chunks a wave, and the second launch.  v_mfma_f32_16x16x32_bf16, S^T = K Q^T:
// row rho of key tile (u, t) is key 16 (rho >> 2) + 8 u + 4 t + (rho & 3), so that lane group g = lane >> 4 is left with the
// scores of keys 16 g .. 16 g + 15, whose values of one dim are one 16-byte load, and weights go to the second product
// without leaving their lane.  Dims of K and Q are taken as 64 c + 16 g + [0, 16) by lane group g: one 16-byte load, two steps.
#include <algorithm>

#include "int8_rows.h"

namespace k8s {
namespace q8 {

constexpr int D = 128;
constexpr float kLog2e = 1.4426950408889634f;

struct Item {  // (a list may begin at any word of a step's buffer)
  int x, y, z, w;
};
struct AttnArgs {
  const uint16_t* q;
  long ldq;
  const uint8_t *k, *v;
  const float *ks, *vs;
  const int* bt;       // [S][bt_stride] block ids
  int bt_stride, NB;
  int bt_keys;         // what a row of the table has pages for (a context behind that, a page outside the pool: clamped, never read)
  const int *ctx, *q_start;
  int S, nq, nkv, G, BS;
  float scale_log2;
  uint16_t* out;
  long ldo;
  // replies: a list of (row, part | -1, end key, q row | (tokens - 1) << 24), parts of part_size keys
  const Item* items;
  int n_items;
  const int* d_items;  // {items, keys a part} on the device, of n_items that the list has room for; or null
  float *part_o, *part_ml;
  int n_parts, part_size;
  // chunks: tiles of rows and runs of 64-key pages
  const int *tile_seq, *tile_tok0, *tile_len, *tile_kv0, *tile_kv1, *tile_slot;
  int n_tiles;
  const int *m_tok0, *m_len, *m_slot0, *m_np;
  int n_merge, slot_rows;
  int own, parts;  // tokens of a tile that the kernel finds by itself and runs that its keys are cut into; 0: the lists above
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
// A chunk's keys and values make room for the next chunk's as soon as they are used, so that a wave always has 8 to 16 KB on the way.
// They are read non-temporally: a page is read once a step (96 replies over 1500 to 6000 keys take 3 % less).
__device__ __forceinline__ u32x4 once(const uint8_t* p) { return __builtin_nontemporal_load(reinterpret_cast<const u32x4*>(p)); }
__device__ __forceinline__ void walk(State& st, const AttnArgs& a, const int* bt, int kvh, int k0, int k1, int kmin, int lim, int lane) {
  const int r = lane & 15, g = lane >> 4, n = (k1 - k0 + 63) >> 6;
  if (n <= 0) return;
  const uint8_t* const kb = a.k + ((size_t)kvh * a.BS + 16 * (r >> 2) + (r & 3)) * D + 16 * g;
  const uint8_t* const vb = a.v + ((size_t)kvh * D + r) * a.BS + 16 * g;
  const float *const ksb = a.ks + kvh * a.BS + 16 * g, *const vsb = a.vs + kvh * a.BS + 16 * g;
  // block ids of 64 chunks, a lane each
  auto ids_from = [&](int c) { return min(max(bt[(k0 + 64 * min(c + lane, n - 1)) / a.BS], 0), a.NB - 1); };
  int ids = ids_from(0), off = k0 % a.BS;
  u32x4 kf[4][2], vf[8];
  f32x4 ks[4], vs[4];
  auto ask_k = [&](size_t at) {
#pragma unroll
    for (int t = 0; t < 4; ++t) {
#pragma unroll
      for (int c = 0; c < 2; ++c) kf[t][c] = once(kb + (at + 4 * t) * D + 64 * c);
      ks[t] = *reinterpret_cast<const f32x4*>(ksb + at + 4 * t);
    }
  };
  auto ask_v = [&](size_t at, int off) {
    const uint8_t* const p = vb + (at - off) * D + off;
#pragma unroll
    for (int d = 0; d < 8; ++d) vf[d] = once(p + 16 * d * a.BS);
  };
  auto ask_vs = [&](size_t at) {
#pragma unroll
    for (int t = 0; t < 4; ++t) vs[t] = *reinterpret_cast<const f32x4*>(vsb + at + 4 * t);
  };
  const size_t step = (size_t)a.nkv * a.BS;  // keys of all heads in a block
  {
    const size_t at = __builtin_amdgcn_readlane(ids, 0) * step + off;
    ask_k(at);
    ask_vs(at);
    ask_v(at, off);
  }
  for (int c = 0; c < n; ++c) {
    const int kb0 = k0 + 64 * c;
    if (c + 1 < n) {
      off += 64;
      if (off >= a.BS) off = 0;
      if (((c + 1) & 63) == 0) ids = ids_from(c + 1);
    }
    const size_t at = __builtin_amdgcn_readlane(ids, min(c + 1, n - 1) & 63) * step + off;  // (the last chunk asks for itself again)
    f32x4 sc[4];
#pragma unroll
    for (int t = 0; t < 4; ++t) {
      f32x4 acc = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16x8(kf[t][e][0], kf[t][e][1]), st.qf[2 * e], acc, 0, 0, 0);
        acc = __builtin_amdgcn_mfma_f32_16x16x32_bf16(to_bf16x8(kf[t][e][2], kf[t][e][3]), st.qf[2 * e + 1], acc, 0, 0, 0);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i) sc[t][i] = acc[i] * (ks[t][i] * a.scale_log2);
    }
    __builtin_amdgcn_sched_barrier(0);
    ask_k(at);
    if (kb0 + 64 > kmin) {  // keys that a row does not see: no weight, whatever stands there (a scale may be a NaN)
#pragma unroll
      for (int t = 0; t < 4; ++t)
#pragma unroll
        for (int i = 0; i < 4; ++i)
          if (kb0 + 16 * g + 4 * t + i >= lim) sc[t][i] = -INFINITY, vs[t][i] = 0.f;
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
        pf[t >> 1][4 * (t & 1) + i] = (__bf16)(e * vs[t][i]);
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
    ask_vs(at);
#pragma unroll
    for (int d = 0; d < 8; ++d) {
      st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[0], to_bf16x8(vf[d][0], vf[d][1]), st.o[d], 0, 0, 0);
      st.o[d] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(pf[1], to_bf16x8(vf[d][2], vf[d][3]), st.o[d], 0, 0, 0);
    }
    __builtin_amdgcn_sched_barrier(0);
    ask_v(at, off);
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
  const int n_items = a.d_items ? min(__builtin_amdgcn_readfirstlane(a.d_items[0]), a.n_items) : a.n_items;
  const int part_size = a.d_items ? __builtin_amdgcn_readfirstlane(a.d_items[1]) : a.part_size;
  const int total = n_items * a.nkv;
  for (int w = blockIdx.x; w < total; w += gridDim.x) {
    const int it = w / a.nkv, kvh = w - it * a.nkv;
    const Item item = a.items[it];
    const int seq = item.x, k1 = min(item.z, a.bt_keys), qrow = item.w & 0xFFFFFF, nt = (item.w >> 24) + 1;
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
      } else if (a.n_parts > 1 && part < a.n_parts) {  // (else there is no room for it)
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

// The parts of a row: 32 lanes have four dims each, the groups of 32 every G-th part; they meet in LDS.  Parts are added in an
// order that only their count decides.
template <int G>
__device__ __forceinline__ void join_parts(const float* po, const float* pml, size_t at, size_t step, int np, uint16_t* out) {
  __shared__ f32x4 so[G][32];
  __shared__ float sl[G];
  const int c = threadIdx.x & 31, g = threadIdx.x >> 5;
  float M = -INFINITY, L = 0.f;
  f32x4 O = {0.f, 0.f, 0.f, 0.f};
  {
    for (int p = c; p < np; p += 32) M = fmaxf(M, pml[(at + p * step) * 2]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) M = fmaxf(M, __shfl_xor(M, o, 64));
#pragma unroll 4
    for (int p = g; p < np; p += G) {
      const float m = pml[(at + p * step) * 2], l = pml[(at + p * step) * 2 + 1];
      const f32x4 v = *reinterpret_cast<const f32x4*>(po + (at + p * step) * D + 4 * c);
      const float f = m == -INFINITY ? 0.f : __builtin_amdgcn_exp2f(m - M);
      L = fmaf(l, f, L);
#pragma unroll
      for (int e = 0; e < 4; ++e) O[e] = fmaf(v[e], f, O[e]);
    }
  }
  so[g][c] = O;
  if (c == 0) sl[g] = L;
  __syncthreads();
  if (g) return;
#pragma unroll
  for (int k = 1; k < G; ++k) {
    L += sl[k];
    O += so[k][c];
  }
  const float inv = L == 0.f ? 0.f : 1.f / L;
#pragma unroll
  for (int e = 0; e < 4; ++e) out[4 * c + e] = f2bf(O[e] * inv);
}

// rows of more than one part: grid (nq, S)
__global__ void __launch_bounds__(256) reply_merge_kernel(AttnArgs a) {
  const int head = blockIdx.x, seq = blockIdx.y;
  const int part_size = a.d_items ? a.d_items[1] : a.part_size;
  const int np = min(a.n_parts, (a.ctx[seq] + part_size - 1) / part_size);
  if (np <= 1) return;
  join_parts<8>(a.part_o, a.part_ml, ((size_t)seq * a.nq + head) * a.n_parts, 1, np, a.out + a.q_start[seq] * a.ldo + head * D);
}

// ------------------------------------------------------------------ chunks
// A workgroup holds up to 256 rows (token, q head) of one kv head, 32 a wave, and walks pages of 64 keys.  Keys and values are made
// bf16 once for all waves on their way into LDS: 16 of each a thread, asked for a page ahead.
// v_mfma_f32_32x32x16_bf16, S^T = K Q^T: row rho of the 32-key half kt is key 32 kt + 16 (reg >> 3) + 8 hi + (reg & 7) with
// reg = (rho & 3) + 4 (rho >> 3), hi = (rho >> 2) & 1, so that a lane has one row's keys 16 s + 8 hi .. + 7 in registers
// 8 s .. 8 s + 7: the second operand of O^T += V^T P^T as they are.
// LDS (three pages of each, so that a turn's first fragments are read in front of its barrier): a key's 256 bytes with 16-byte
// piece c at c ^ (key & 15), a dim's 128 bytes with piece c at c ^ ((dim >> 1) & 7): no bank conflicts in either direction.
// A turn has page i's softmax beside the products of its neighbours, so that the vector and the matrix units work at once: scales,
// maximum and the weights of the first 32 keys beside V(i - 1), the other weights beside the first half of K(i + 1), whose
// scores take the registers that the weights have left, the staging beside its second half.  A fixed order of instructions holds it
// together: left to the compiler, the products come first and the weights behind them.
// us of four threads' chunks of up to 2048 tokens over 4000, 32 + 2 x 8 heads: page after page 585, in turns 576, in this order
// 507, with a turn's first reads in front of its barrier 495 to 509 by card (865 to 890 TFLOP/s); a prompt of 8192 567 to 585 (940 to 970).  What bounds it is the
// vector unit beside the matrix unit: a turn's 250 vector instructions and 32 exponentials a wave take as long as its 32 products,
// two waves a SIMD leave some 30 % of both to waits, and tiles of 60 to 94 pages fill 256 units unevenly.
constexpr int kRows = 256, kPitch = 272;
constexpr int AHEAD = 3;  // products that a fragment is read in front of its own
struct ChunkLds {
  uint8_t k[3][64 * 256], v[3][D * 128];
  float s[4][2][64];  // keys' scales (with the softmax's, in powers of two), values'
};
template <int N>
using ic = std::integral_constant<int, N>;
template <int N, int J = 0, typename F>
__device__ __forceinline__ void each(F&& f) {
  if constexpr (J < N) {
    f(ic<J>{});
    each<N, J + 1>(f);
  }
}
__device__ __forceinline__ void lds_bar() {
  asm volatile("s_waitcnt lgkmcnt(0)\n\ts_barrier" ::: "memory");
}
// Tile number t of all sequences' (of `own` tokens each, a sequence's last tokens first: those have the most keys): every lane counts
// a sequence's.  No tokens where there are fewer tiles, since the launch has as many as T rows of S sequences can have.
struct Found {
  int seq, tok0, len;
};
__device__ __forceinline__ Found find_tile(const AttnArgs& a, int t) {
  const int lane = threadIdx.x & 63;
  for (int s0 = 0; s0 < a.S; s0 += 64) {
    const int s = min(s0 + lane, a.S - 1), first = a.q_start[s], last = a.q_start[s + 1];
    const int n = s0 + lane < a.S ? (max(last - first, 0) + a.own - 1) / a.own : 0;
    int sum = n;  // of this sequence's and those before it
#pragma unroll
    for (int o = 1; o < 64; o *= 2) {
      const int below = __shfl_up(sum, o, 64);
      if (lane >= o) sum += below;
    }
    const unsigned long long behind = __ballot(sum > t);
    if (behind) {
      const int l = __builtin_ctzll(behind), i = __builtin_amdgcn_readlane(sum, l) - 1 - t, end = __builtin_amdgcn_readlane(last, l);
      const int tok0 = __builtin_amdgcn_readlane(first, l) + i * a.own;
      return {s0 + l, tok0, min(a.own, end - tok0)};
    }
    t -= __builtin_amdgcn_readlane(sum, 63);
  }
  return {0, 0, 0};
}
__global__ void __launch_bounds__(512, 1) chunk_kernel(AttnArgs a) {
  __shared__ __attribute__((aligned(1024))) union {
    ChunkLds p;
    uint8_t o[8 * 32 * kPitch];
  } sm;
  const int kvh = blockIdx.x % a.nkv, tile = blockIdx.x / a.nkv;
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int r = lane & 31, hi = lane >> 5;
  int seq, tok0, len;
  if (a.own) {
    const Found f = find_tile(a, tile / a.parts);
    if (f.len == 0) return;
    seq = f.seq, tok0 = f.tok0, len = f.len;
  } else {
    seq = a.tile_seq[tile], tok0 = a.tile_tok0[tile], len = a.tile_len[tile];
  }
  const int rows = min(len * a.G, kRows);
  const int qs = a.q_start[seq], base = a.ctx[seq] - (a.q_start[seq + 1] - qs) + (tok0 - qs);
  const int* const bt = a.bt + (size_t)seq * a.bt_stride;
  const int grow = 32 * w + r;
  const bool valid = grow < rows;
  const int end = min(base + len, a.bt_keys);               // keys of the whole tile
  const int all = (end + 63) >> 6;
  int p0, p1, slot = -1;
  if (a.own) {
    p0 = max(all, 0) * (tile % a.parts) / a.parts, p1 = max(all, 0) * (tile % a.parts + 1) / a.parts;
    if (a.parts > 1) slot = tile;
  } else {
    p0 = a.tile_kv0[tile], p1 = min(a.tile_kv1[tile], all), slot = a.tile_slot[tile];
  }
  const int np = p1 - p0;
  // this lane's row sees keys below `limit`, every row of the wave those below `lo`
  const int limit = min(valid ? base + grow / a.G + 1 : 0, end), lo = 32 * w + 31 < rows ? base + 32 * w / a.G + 1 : 0;

  bf16x8 qf[8];
  {
    const int at = min(grow, rows - 1), tt = at / a.G;
    const uint16_t* const q = a.q + (long)(tok0 + tt) * a.ldq + (kvh * a.G + at - tt * a.G) * D + 8 * hi;
#pragma unroll
    for (int s = 0; s < 8; ++s) {
      u16x8 z = {0, 0, 0, 0, 0, 0, 0, 0};
      if (valid) z = *reinterpret_cast<const u16x8*>(q + 16 * s);
      qf[s] = __builtin_bit_cast(bf16x8, z);
    }
  }
  f32x16 o[4] = {};
  float m = 0.f, l = 0.f;

  // staging: 16 dims of key tid >> 3, 16 keys of dim tid >> 2, a key's scales
  const int key = tid >> 3, kc = tid & 7, dim = tid >> 2, vc = tid & 3;
  const int step = a.nkv * a.BS;                            // keys of all heads in a block
  const uint8_t* const kb = a.k + ((size_t)kvh * a.BS + key) * D + 16 * kc;
  const uint8_t* const vb = a.v + ((size_t)kvh * D + dim) * a.BS + 16 * vc;
  const float *const ksb = a.ks + kvh * a.BS + lane, *const vsb = a.vs + kvh * a.BS + lane;
  // block ids of 64 pages, a lane each, and where the page that is asked for next lies (the last one for those behind the end)
  auto ids_from = [&](int i) { return min(max(bt[64 * (p0 + min(i + lane, np - 1)) / a.BS], 0), a.NB - 1); };
  int ids = 0, at_k = -1, off_k = 0, blk_k[3], offs[3];
  u32x4 kx, vx;
  float ksx = 0.f, vsx = 0.f;
  auto ask_k = [&](int i) {
    if (i < np) {
      off_k += 64;
      if (off_k >= a.BS) off_k = 0;
      at_k = i;
    }
    blk_k[0] = blk_k[1], blk_k[1] = blk_k[2], offs[0] = offs[1], offs[1] = offs[2];
    blk_k[2] = __builtin_amdgcn_readlane(ids, at_k & 63), offs[2] = off_k;
    const size_t first = (size_t)blk_k[2] * step + off_k;
    kx = *reinterpret_cast<const u32x4*>(kb + first * D);
    ksx = ksb[first];
    vsx = vsb[first];
  };
  auto ask_v = [&] { vx = *reinterpret_cast<const u32x4*>(vb + (size_t)blk_k[0] * step * D + offs[0]); };  // of the page two behind
  auto keep_k = [&](int i, int slot) {
    uint8_t* const kr = sm.p.k[slot] + key * 256;
    *reinterpret_cast<bf16x8*>(kr + 16 * ((2 * kc) ^ (key & 15))) = to_bf16x8(kx[0], kx[1]);
    *reinterpret_cast<bf16x8*>(kr + 16 * ((2 * kc + 1) ^ (key & 15))) = to_bf16x8(kx[2], kx[3]);
    // a key behind the context is nothing, whatever its scales say; a value that is no number makes its key's score none, so
    // that the weights' factor is always a number (and a hidden key's product zero).  All waves write the same.
    const bool in = 64 * (p0 + i) + lane < end, number = fabsf(vsx) < INFINITY;
    sm.p.s[i & 3][0][lane] = in ? (number ? ksx * a.scale_log2 : __uint_as_float(0x7fc00000u)) : 0.f;
    sm.p.s[i & 3][1][lane] = in && number ? vsx : 0.f;
  };
  auto keep_v = [&](int slot) {
    uint8_t* const vr = sm.p.v[slot] + dim * 128;
    *reinterpret_cast<bf16x8*>(vr + 16 * ((2 * vc) ^ ((dim >> 1) & 7))) = to_bf16x8(vx[0], vx[1]);
    *reinterpret_cast<bf16x8*>(vr + 16 * ((2 * vc + 1) ^ ((dim >> 1) & 7))) = to_bf16x8(vx[2], vx[3]);
  };
  const int kreg = (r & 3) + 4 * (r >> 3), krow = 16 * (kreg >> 3) + 8 * ((r >> 2) & 1) + (kreg & 7);
  const int ko = krow * 256 + 16 * (hi ^ (krow & 15)), vo = r * 128 + 16 * (hi ^ ((r >> 1) & 7));
  f32x16 sc[2];
  bf16x8 pf[2][2] = {};
  // Product j of a turn: 0-15 V(i - 1), in its place `vp`, by the weights of its page, 16-31 K(i + 1), in `kp`, by Q.  Fragments are
  // read AHEAD products ahead.
  auto fragment = [&](auto J, int vp, int kp) {
    constexpr int j = decltype(J)::value;
    if constexpr (j < 16)
      return *reinterpret_cast<const bf16x8*>(sm.p.v[vp] + 4096 * (j & 3) + (vo ^ (32 * (j >> 2))));
    else
      return *reinterpret_cast<const bf16x8*>(sm.p.k[kp] + 8192 * ((j - 16) >> 3) + (ko ^ (32 * (j & 7))));
  };
  auto product = [&](auto J, const bf16x8& f) {
    constexpr int j = decltype(J)::value;
    if constexpr (j < 16) {
      o[j & 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, pf[j >> 3][(j >> 2) & 1], o[j & 3], 0, 0, 0);
    } else {
      if constexpr ((j & 7) == 0) sc[(j - 16) >> 3] = f32x16{};
      sc[(j - 16) >> 3] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(f, qf[j & 7], sc[(j - 16) >> 3], 0, 0, 0);
    }
  };
  if (np > 0) {
    ids = ids_from(0);
    off_k = 64 * p0 % a.BS - 64;
    ask_k(0);
    keep_k(0, 0);
    ask_k(1);
    keep_k(1, 1);
    ask_k(2);
    ask_v();
    keep_k(2, 2);
    keep_v(0);
    ask_k(3);
    ask_v();
    for (int i = tid; i < D * 8; i += 512) *reinterpret_cast<u32x4*>(sm.p.v[2] + 16 * i) = u32x4{0, 0, 0, 0};  // (page -1's weights are zeros)
    lds_bar();
    int s0 = 0, s1 = 1, s2 = 2;  // i, i + 1 and i + 2 by three
    // A wave without rows stages its share and nothing else: the others have its time.  (us of eight threads' 12 tokens over 7332 keys,
    // 16 + 2 x 16 heads, 133 -> 99; five threads' 24 over 7398, 32 + 2 x 8, 46 -> 37.)
    if (32 * w >= rows) {
      for (int i = 0; i < np; ++i) {
        lds_bar();
        keep_k(i + 3, s0);
        ask_k(i + 4);
        keep_v(s1);
        ask_v();
        if (((i + 5) & 63) == 0 && i + 5 < np) ids = ids_from(i + 5);
        const int s3 = s0;
        s0 = s1, s1 = s2, s2 = s3;
      }
    } else {
      each<16>([&](auto J) { product(ic<decltype(J)::value + 16>{}, fragment(ic<decltype(J)::value + 16>{}, 0, 0)); });
      auto four = [](const float* f, int g) { return *reinterpret_cast<const f32x4*>(f + 16 * (g >> 1) + 4 * (g & 1)); };  // of a lane's scores 4g ..
      auto hide = [&](int i) {  // keys that the row does not see
        const int k0 = 64 * (p0 + i) + 8 * hi;
  #pragma unroll
        for (int e = 0; e < 32; ++e)
          if (k0 + 16 * (e >> 3) + (e & 7) >= limit) sc[e >> 4][e & 15] = -INFINITY;
      };
      auto largest = [&] {
        float c0 = -INFINITY, c1 = -INFINITY;
  #pragma unroll
        for (int e = 0; e < 16; ++e) {
          c0 = fmaxf(c0, sc[0][e]);
          c1 = fmaxf(c1, sc[1][e]);
        }
        return fmaxf(c0, c1);
      };
      auto of_row = [](float top) {  // the two halves of a row
        const auto pr = __builtin_amdgcn_permlane32_swap(__float_as_uint(top), __float_as_uint(top), false, false);
        return fmaxf(__uint_as_float(pr[0]), __uint_as_float(pr[1]));
      };
      {
        // where the row's weights begin: the largest score of the first page (a row without a key there has none at all)
        const f32x16 raw[2] = {sc[0], sc[1]};
  #pragma unroll
        for (int g = 0; g < 8; ++g) {
          const f32x4 f = four(sm.p.s[0][0] + 8 * hi, g);
  #pragma unroll
          for (int e = 0; e < 4; ++e) sc[g >> 2][4 * (g & 3) + e] *= f[e];
        }
        hide(0);
        const float top = of_row(largest());
        m = top == -INFINITY ? 0.f : top;
        sc[0] = raw[0], sc[1] = raw[1];
      }
      bf16x8 fr[4];
      f32x4 fs[4];
      // scales of four keys: of keys 4q .. of a lane, wanted by step q (q < 8), of values 4(q - 8) .., wanted by step 2 q - 8; read
      // three steps in front
      auto scale = [&](auto Q, int i) {
        constexpr int q = decltype(Q)::value;
        fs[q & 3] = four(sm.p.s[i & 3][q >> 3] + 8 * hi, q & 7);
      };
      each<3>([&](auto J) {
        scale(J, 0);
        fr[J] = fragment(J, 2, 1);
      });
      for (int i = 0; i < np; ++i) {
        lds_bar();  // K(i + 2) and V(i) are there, every wave is done with K(i) and V(i - 2)
        uint32_t pn[16];
        float c[2] = {-INFINITY, -INFINITY}, sum[4] = {0.f, 0.f, 0.f, 0.f}, up = 0.f;
        each<32>([&](auto Jc) {
          constexpr int j = decltype(Jc)::value;
          if constexpr (j + AHEAD < 32)
            fr[(j + AHEAD) & 3] = fragment(ic<j + AHEAD>{}, s2, s1);
          else
            fr[(j + AHEAD) & 3] = fragment(ic<j + AHEAD - 32>{}, s0, s2);  // the next turn's
          if constexpr (j < 5)
            scale(ic<j + 3>{}, i);
          else if constexpr (j < 20 && (j & 1))
            scale(ic<(j + 11) / 2>{}, i);
          else if constexpr (j >= 29)
            scale(ic<j - 29>{}, i + 1);
          product(Jc, fr[j & 3]);
          if constexpr (j < 8) {  // four scores of the lane, above what the row's weights stand on
  #pragma unroll
            for (int e = 0; e < 4; ++e) {
              float x = fmaf(sc[j >> 2][4 * (j & 3) + e], fs[j & 3][e], -m);
              asm volatile("" : "+v"(x));  // (not made again from the sum and the scale, which would stay in registers for it)
              sc[j >> 2][4 * (j & 3) + e] = x;
              c[e & 1] = fmaxf(c[e & 1], x);
            }
          } else if constexpr (j < 24) {  // two weights
            if constexpr (j == 8) {
              float top = fmaxf(c[0], c[1]);
              if (64 * (p0 + i) + 64 > lo) {
                hide(i);
                top = largest();
              }
              top = of_row(top);
              // where a row grows by more than 8, its weights stand on its new maximum from here on: weights up to 2^8
              if (__ballot(top > 8.f)) {
                up = top > 8.f ? top : 0.f;
                m += up;
  #pragma unroll
                for (int e = 0; e < 32; ++e) sc[e >> 4][e & 15] -= up;
              }
            }
            constexpr int t = j - 8, kt = t >> 3, e = 2 * (t & 7);
            const float x0 = __builtin_amdgcn_exp2f(sc[kt][e]), x1 = __builtin_amdgcn_exp2f(sc[kt][e + 1]);
            sum[2 * (t & 1)] += x0;
            sum[2 * (t & 1) + 1] += x1;
            typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
            uint32_t two = __builtin_bit_cast(uint32_t, bf16x2{(__bf16)(x0 * fs[(t >> 1) & 3][e & 3]), (__bf16)(x1 * fs[(t >> 1) & 3][(e & 3) + 1])});
            // (wanted in the next turn only: computed here all the same, beside the products)
            asm volatile("" : "+v"(two), "+v"(sum[2 * (t & 1)]), "+v"(sum[2 * (t & 1) + 1]));
            pn[t] = two;
          } else if constexpr (j == 24) {
            keep_k(i + 3, s0);
          } else if constexpr (j == 27) {
            ask_k(i + 4);
          } else if constexpr (j == 28) {
            keep_v(s1);
          } else if constexpr (j == 30) {
            ask_v();
          }
          __builtin_amdgcn_sched_barrier(0);
        });
        if (((i + 5) & 63) == 0 && i + 5 < np) ids = ids_from(i + 5);
        if (__ballot(up != 0.f)) {
          const float alpha = __builtin_amdgcn_exp2f(-up);
          l *= alpha;
  #pragma unroll
          for (int d = 0; d < 4; ++d)
  #pragma unroll
            for (int e = 0; e < 16; ++e) o[d][e] *= alpha;
        }
        l += (sum[0] + sum[1]) + (sum[2] + sum[3]);
  #pragma unroll
        for (int kt = 0; kt < 2; ++kt)
  #pragma unroll
          for (int s = 0; s < 2; ++s) {
            const uint32_t* const t = pn + 8 * kt + 4 * s;
            pf[kt][s] = __builtin_bit_cast(bf16x8, u32x4{t[0], t[1], t[2], t[3]});
          }
        const int s3 = s0;
        s0 = s1, s1 = s2, s2 = s3;
      }
      each<16>([&](auto J) {  // (V(np - 1) is at s2)
        constexpr int j = decltype(J)::value;
        product(J, fr[j & 3]);
        if constexpr (j + AHEAD < 16) fr[(j + AHEAD) & 3] = fragment(ic<j + AHEAD>{}, s2, 0);
      });
    }
  }
  l += __shfl_xor(l, 32, 64);
  if (slot >= 0) {
    if (!valid) return;
    const size_t at = ((size_t)slot * a.nkv + kvh) * a.slot_rows + grow;
#pragma unroll
    for (int d = 0; d < 4; ++d)
#pragma unroll
      for (int e = 0; e < 16; e += 4)
        *reinterpret_cast<f32x4*>(a.part_o + at * D + 32 * d + 2 * e + 4 * hi) = f32x4{o[d][e], o[d][e + 1], o[d][e + 2], o[d][e + 3]};
    if (hi == 0) {
      a.part_ml[2 * at] = l == 0.f ? -INFINITY : m;  // (a row without a key in this run)
      a.part_ml[2 * at + 1] = l;
    }
    return;
  }
  // rows leave through LDS, so that 16 lanes store one whole
  const float inv = l == 0.f ? 0.f : 1.f / l;
  lds_bar();
  uint8_t* const ow = sm.o + w * (32 * kPitch);
#pragma unroll
  for (int d = 0; d < 4; ++d)
#pragma unroll
    for (int e = 0; e < 16; e += 4)
      *reinterpret_cast<u16x4*>(ow + r * kPitch + 2 * (32 * d + 2 * e + 4 * hi)) =
          u16x4{f2bf(o[d][e] * inv), f2bf(o[d][e + 1] * inv), f2bf(o[d][e + 2] * inv), f2bf(o[d][e + 3] * inv)};
  wave_lds_fence();
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    const int rr = 4 * j + (lane >> 4), gr = 32 * w + rr, c = lane & 15;
    if (gr >= rows) continue;
    uint16_t* const dst = a.out + (long)(tok0 + gr / a.G) * a.ldo + (kvh * a.G + gr % a.G) * D + 8 * c;
    const u16x8 v = *reinterpret_cast<const u16x8*>(ow + rr * kPitch + 16 * c);
    if (((uintptr_t)dst & 15) == 0) {
      *reinterpret_cast<u16x8*>(dst) = v;
    } else {
#pragma unroll
      for (int e = 0; e < 8; ++e) dst[e] = v[e];
    }
  }
}

// rows of split tiles: grid (split tiles * nkv, rows)
__global__ void __launch_bounds__(64) chunk_merge_kernel(AttnArgs a) {
  const int kvh = blockIdx.x % a.nkv, mi = blockIdx.x / a.nkv, row = blockIdx.y;
  int tok0, len, slot0, np;
  if (a.own) {
    const Found f = find_tile(a, mi);
    tok0 = f.tok0, len = f.len, slot0 = mi * a.parts, np = a.parts;
  } else {
    tok0 = a.m_tok0[mi], len = a.m_len[mi], slot0 = a.m_slot0[mi], np = a.m_np[mi];
  }
  if (row >= len * a.G) return;
  join_parts<2>(a.part_o, a.part_ml, ((size_t)slot0 * a.nkv + kvh) * a.slot_rows + row, (size_t)a.nkv * a.slot_rows, np,
                a.out + (long)(tok0 + row / a.G) * a.ldo + (kvh * a.G + row % a.G) * D);
}

}  // namespace q8
}  // namespace k8s

K8S_API int k8s_int8_attn_reply(const void* q, long ldq, const void* k, const void* v, const float* ks, const float* vs, int NB, const int* bt,
                                int bt_stride, int bt_cols, const int* ctx, const int* q_start, int S, int nq, int nkv, int BS, float scale, void* out,
                                long ldo, float* part_o, float* part_ml, int n_parts, int part_size, const void* items, int n_items,
                                const int* d_items, int grid, void* stream) {
  using namespace k8s::q8;
  if (S <= 0) return 0;
  if (nkv <= 0 || nq % nkv || nq / nkv > 16 || BS <= 0 || (BS & 63) || grid <= 0 || NB <= 0) return (int)hipErrorInvalidValue;
  if (n_parts > 1 && (!part_o || !part_ml || part_size <= 0 || (part_size & 63))) return (int)hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const uint16_t*)q, a.ldq = ldq, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs, a.bt = bt;
  a.bt_stride = bt_stride, a.bt_keys = (int)std::min((long)bt_cols * BS, 0x7fffffc0L);
  a.NB = NB, a.ctx = ctx, a.q_start = q_start, a.S = S, a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.BS = BS;
  a.scale_log2 = scale * kLog2e, a.out = (uint16_t*)out, a.ldo = ldo, a.part_o = part_o, a.part_ml = part_ml, a.n_parts = n_parts;
  a.part_size = part_size, a.items = (const Item*)items, a.n_items = n_items, a.d_items = d_items;
  hipStream_t st = (hipStream_t)stream;
  hipLaunchKernelGGL(reply_kernel, dim3(grid), dim3(64), 0, st, a);
  if (n_parts > 1) hipLaunchKernelGGL(reply_merge_kernel, dim3(nq, S), dim3(256), 0, st, a);
  return (int)hipGetLastError();
}

// Tiles of up to `rows` (token, q head) rows; split tiles leave parts of slot_rows rows a slot and kv head.  With own > 0 the lists are not
// read: n_tiles is the most tiles of `own` tokens that the rows can make, and each one's keys are cut into `parts` runs.
K8S_API int k8s_int8_attn_chunk(const void* q, long ldq, const void* k, const void* v, const float* ks, const float* vs, int NB, const int* bt,
                                int bt_stride, int bt_cols, const int* ctx, const int* q_start, int S, int nq, int nkv, int BS, float scale, void* out, long ldo,
                                const int* tile_seq, const int* tile_tok0, const int* tile_len, const int* tile_kv0, const int* tile_kv1,
                                const int* tile_slot, int n_tiles, int rows, const int* m_tok0, const int* m_len, const int* m_slot0,
                                const int* m_np, int n_merge, float* part_o, float* part_ml, int slot_rows, int own, int parts, void* stream) {
  using namespace k8s::q8;
  if (n_tiles <= 0) return 0;
  if (nkv <= 0 || nq % nkv || BS <= 0 || (BS & 63) || NB <= 0 || rows <= 0 || rows > kRows || rows > slot_rows) return (int)hipErrorInvalidValue;
  if (own < 0 || (own > 0 && (parts <= 0 || S <= 0 || (long)own * (nq / nkv) > rows))) return (int)hipErrorInvalidValue;
  const int runs = own > 0 ? parts : 1, merged = own > 0 ? (parts > 1 ? n_tiles : 0) : n_merge;
  if (merged > 0 && (!part_o || !part_ml)) return (int)hipErrorInvalidValue;
  AttnArgs a{};
  a.q = (const uint16_t*)q, a.ldq = ldq, a.k = (const uint8_t*)k, a.v = (const uint8_t*)v, a.ks = ks, a.vs = vs, a.bt = bt;
  a.bt_stride = bt_stride, a.bt_keys = (int)std::min((long)bt_cols * BS, 0x7fffffc0L);
  a.NB = NB, a.ctx = ctx, a.q_start = q_start, a.S = S, a.nq = nq, a.nkv = nkv, a.G = nq / nkv, a.BS = BS;
  a.scale_log2 = scale * kLog2e, a.out = (uint16_t*)out, a.ldo = ldo, a.part_o = part_o, a.part_ml = part_ml, a.own = own, a.parts = runs;
  a.tile_seq = tile_seq, a.tile_tok0 = tile_tok0, a.tile_len = tile_len, a.tile_kv0 = tile_kv0, a.tile_kv1 = tile_kv1, a.tile_slot = tile_slot;
  a.n_tiles = n_tiles, a.m_tok0 = m_tok0, a.m_len = m_len, a.m_slot0 = m_slot0, a.m_np = m_np;
  a.n_merge = n_merge, a.slot_rows = slot_rows;
  hipStream_t st = (hipStream_t)stream;
  const long blocks = (long)n_tiles * runs * nkv;
  if (blocks > 0x7fffffffL) return (int)hipErrorInvalidValue;
  hipLaunchKernelGGL(chunk_kernel, dim3((unsigned)blocks), dim3(512), 0, st, a);
  if (merged > 0) hipLaunchKernelGGL(chunk_merge_kernel, dim3(merged * nkv, rows), dim3(64), 0, st, a);
  return (int)hipGetLastError();
}
