// Attention of one token per row over a paged KV cache, for sm_100a.
//
//   out[r,h,:] = sum_j w_j V[j,:] / sum_j w_j,   w_j = exp(scale q[r,h,:] . K[j,:])
//
// over the keys j that row r sees: j < len, and with a window only the first
// `sinks` and the last `window` of them. The keys of a row are numbered
// 0..n-1 in order and cut into splits of `chunk` keys; one CTA takes a split
// for all query heads of a KV head (so K and V are read once), keeps a running
// maximum m, sum l and weighted sum of V, and the last CTA of a (row, KV head)
// to finish joins the splits:
//   m = max m_s,  out = sum_s 2^(m_s - m) acc_s / sum_s 2^(m_s - m) l_s.
// Exponents are base 2 with log2(e) folded into q. All statistics are fp32.
#include <cuda.h>

#include <cmath>

#include "mma_sync.cuh"
#include "paged.cuh"

namespace tllm {

// tma.cu
int make_map(CUtensorMap *m, const void *base, int dtype, int rank, const long *dims,
             const long *strides_bytes, const int *box, bool swizzle128);

namespace {

constexpr int kMaxSplits = 256;
constexpr float kLog2e = 1.4426950408889634f;

struct AttnParams {
  PagedView kv;
  const float *q;        // row r, head h at q + r * q_sr + h * q_sh
  const int *row_seq;    // or null: row r reads sequence r
  const int *row_len;
  float *out;
  uint16_t *out_act;     // or operand-format output, planes out_plane apart
  size_t out_plane;
  int out_planes;
  long q_sr, q_sh, o_sr, o_sh;
  float *part_acc;       // (rows, n_y, max_splits, G, D)
  float *part_ml;        // (rows, n_y, max_splits, G, 2)
  int *counters;         // (rows, n_y)
  int *err;
  int rows, row0, group, n_gsub, g_tile, n_y;   // heads per KV head, sub-groups, heads per CTA
  int chunk, max_splits, tile;
  int window, sinks;
  float qscale;          // sm_scale * log2(e)
};

// The keys of one row and this CTA's share of them.
struct RowSpan {
  int seq, len;
  int s, a;              // keys [0, s) and [a, len) are visible
  int n_splits, begin, end;   // on the axis of the kernel's keys
};

// Splits of the planned size over n keys; longer ones where the host's bound
// on the length was too small.
__device__ __forceinline__ void split_row(const AttnParams &p, RowSpan &x, int split, int n) {
  int chunk = p.chunk;
  if ((long)chunk * p.max_splits < n) {
    chunk = (n + p.max_splits - 1) / p.max_splits;
    chunk = (chunk + p.tile - 1) / p.tile * p.tile;
  }
  x.n_splits = n > 0 ? (n + chunk - 1) / chunk : 1;
  x.begin = split * chunk;
  x.end = min(x.begin + chunk, n);
}

__device__ __forceinline__ RowSpan row_keys(const AttnParams &p, int row, int split) {
  RowSpan x;
  x.seq = p.row_seq ? p.row_seq[row] : row;
  x.len = p.row_len[row];
  const int cap = p.kv.table_cols * p.kv.page_size;
  if (x.len > cap) {
    x.len = cap;
    if (threadIdx.x == 0 && split == 0) atomicOr(p.err, DEV_ERR_LEN_CLAMPED);
  }
  if (x.seq < 0 || x.seq >= p.kv.n_seq) {
    x.len = 0;
    if (threadIdx.x == 0 && split == 0) atomicOr(p.err, DEV_ERR_PAGE);
  }
  if (x.len < 0) x.len = 0;
  x.s = p.window > 0 ? min(p.sinks, x.len) : 0;
  x.a = p.window > 0 ? max(x.len - p.window, x.s) : 0;
  return x;
}

__device__ __forceinline__ void store_out(const AttnParams &p, size_t idx, float v) {
  if (p.out_act)
    store_act(p.out_act, p.out_plane, idx, v, p.out_planes);
  else
    p.out[idx] = v;
}

// Joins the NW warps' (acc, m, l) of this split, which lie in shared memory as
// w_acc[NW][G][D], w_m[NW][G], w_l[NW][G], and, with several splits, the
// splits of this (row, y) in the CTA that finishes last. Called by all threads
// after a barrier; reuses the shared memory.
template <int NW, int THREADS>
__device__ void finish_split(const AttnParams &p, const RowSpan &x, int row, int y,
                             int head0, int G, int D, int split, float *smem,
                             int *s_flag) {
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const float *w_acc = smem;
  const float *w_m = smem + NW * G * D;
  const float *w_l = w_m + NW * G;
  const bool single = x.n_splits == 1;
  const size_t slot = ((size_t)row * p.n_y + y) * p.max_splits + split;
  for (int i = tid; i < G * D; i += THREADS) {
    const int g = i / D;
    float mx = -INFINITY;
#pragma unroll
    for (int w = 0; w < NW; ++w) mx = fmaxf(mx, w_m[w * G + g]);
    float num = 0.f, den = 0.f;
#pragma unroll
    for (int w = 0; w < NW; ++w) {
      const float m = w_m[w * G + g];
      // (a warp without a visible key has m = -inf and sums of zero)
      const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);
      num = fmaf(w_acc[(w * G + g) * D + (i - g * D)], f, num);
      den = fmaf(w_l[w * G + g], f, den);
    }
    if (single) {
      store_out(p, (size_t)row * p.o_sr + (size_t)(head0 + g) * p.o_sh + (i - g * D),
                den == 0.f ? 0.f : num / den);
    } else {
      p.part_acc[slot * p.g_tile * D + i] = num;
      if (i == g * D) {
        p.part_ml[(slot * p.g_tile + g) * 2] = mx;
        p.part_ml[(slot * p.g_tile + g) * 2 + 1] = den;
      }
    }
  }
  if (single) return;

  __syncthreads();
  if (tid == 0) {
    int *ctr = p.counters + (size_t)row * p.n_y + y;
    __threadfence();   // (of all writes that the barrier has ordered before)
    *s_flag = atomicAdd(ctr, 1) == x.n_splits - 1;
    if (*s_flag) *ctr = 0;   // all other CTAs of this (row, y) took theirs
    __threadfence();
  }
  __syncthreads();
  if (!*s_flag) return;

  // The statistics (one split per lane) and the first kJoin values of this
  // thread's first output are on the way together; later ones come in batches
  // whose size does not depend on the number of splits.
  constexpr int kJoin = 8;
  const size_t base = ((size_t)row * p.n_y + y) * p.max_splits;
  const float *acc = p.part_acc + base * p.g_tile * D;
  const size_t step = (size_t)p.g_tile * D;
  float v[kJoin];
  auto load = [&](int s0, int i) {
#pragma unroll
    for (int k = 0; k < kJoin; ++k)
      v[k] = __ldcg(acc + (size_t)min(s0 + k, x.n_splits - 1) * step + i);
  };
  if (tid < G * D) load(0, tid);
  float *sw = smem;   // [G][kMaxSplits] weights of the splits
  const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml) + base * p.g_tile;
  for (int g = warp; g < G; g += THREADS / 32) {
    auto stats = [&](int s) {
      return s < x.n_splits ? __ldcg(ml + (size_t)s * p.g_tile + g)
                            : make_float2(-INFINITY, 0.f);
    };
    const float2 own = stats(lane);
    float mx = own.x, den = 0.f;
    for (int s = lane + 32; s < x.n_splits; s += 32) mx = fmaxf(mx, stats(s).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
    auto weigh = [&](int s, float2 m) {
      const float f = m.x == -INFINITY ? 0.f : fast_exp2(m.x - mx);
      if (s < x.n_splits) sw[g * kMaxSplits + s] = f;
      den = fmaf(m.y, f, den);
    };
    weigh(lane, own);
    for (int s = lane + 32; s < x.n_splits; s += 32) weigh(s, stats(s));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(~0u, den, o);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    __syncwarp();
    for (int s = lane; s < x.n_splits; s += 32) sw[g * kMaxSplits + s] *= inv;
  }
  __syncthreads();
  for (int i = tid; i < G * D; i += THREADS) {
    const int g = i / D;
    float o = 0.f;
    for (int s0 = 0; s0 < x.n_splits; s0 += kJoin) {
      if (i != tid || s0 > 0) load(s0, i);
#pragma unroll
      for (int k = 0; k < kJoin; ++k)
        if (s0 + k < x.n_splits) o = fmaf(sw[g * kMaxSplits + s0 + k], v[k], o);
    }
    store_out(p, (size_t)row * p.o_sr + (size_t)(head0 + g) * p.o_sh + (i - g * D), o);
  }
}

// --------------------------------------------------------------------------
// Every page size, layout, cache type and head_dim: CUDA cores, loads straight
// from the pages. LPR lanes (8, 16 or 32) share a key, each holding NV 16-byte
// units of it; a warp takes U * 32 / LPR keys at a time with all their K and V
// loads in flight and their pages looked up one step ahead. The U x G partial
// products of a lane are summed over the LPR lanes by halving: a lane passes
// on half of its sums and keeps the other half in every step, so that 16 sums
// over 32 lanes cost 16 shuffles, not 80, and end in one lane each, which keeps
// the running maximum and sum of its head. Each group of LPR lanes has its own
// over its keys; they are joined at the end.
//
// Bound by instruction issue where several heads share the keys: 16 rows of
// 24/8/128 fp32 with 1024 to 8192 keys take 139 us (0.67 of HBM's bandwidth; 65 % of
// the issue slots of SMs that are active for 85 % of the time; 3 heads run as 4),
// 64 rows of the same over bf16 pages of 20 slots 417 (0.45), 64 of 12/4/96 176 (0.40);
// with one head per KV head by HBM: 32 rows of 32/32/64 fp32 96.5 (0.90).
// --------------------------------------------------------------------------
constexpr int kGenWarps = 8;

template <typename T> struct Unit;
template <> struct Unit<float> {
  static constexpr int N = 4;
  __device__ static void unpack(const uint4 &v, float (&f)[4]) {
    f[0] = __uint_as_float(v.x); f[1] = __uint_as_float(v.y);
    f[2] = __uint_as_float(v.z); f[3] = __uint_as_float(v.w);
  }
};
template <> struct Unit<__nv_bfloat16> {
  static constexpr int N = 8;
  __device__ static void unpack(const uint4 &v, float (&f)[8]) {
    f[0] = bf16lo(v.x); f[1] = bf16hi(v.x); f[2] = bf16lo(v.y); f[3] = bf16hi(v.y);
    f[4] = bf16lo(v.z); f[5] = bf16hi(v.z); f[6] = bf16lo(v.w); f[7] = bf16hi(v.w);
  }
};

// Keys of a group of lanes whose loads are in flight together, as far as the
// registers go.
__host__ __device__ constexpr int units_deep(int NV) { return NV > 1 ? 2 : 4; }

template <typename T, int G, int NV, int LPR>
__global__ void __launch_bounds__(kGenWarps * 32)
    paged_rows_kernel(const AttnParams p) {
  griddep_launch();
  griddep_wait();
  using UT = Unit<T>;
  constexpr int E = UT::N;
  constexpr int U = units_deep(NV), N = U * G;
  constexpr int R = N > LPR ? N / LPR : 1;   // sums that a lane ends up with
  constexpr int rpw = 32 / LPR;              // groups of lanes
  static_assert(U <= LPR, "a lane's sums are of one key");
  extern __shared__ __align__(16) float smem_f[];
  __shared__ int s_flag;
  const int row = p.row0 + blockIdx.z, y = blockIdx.y, split = blockIdx.x;
  RowSpan x = row_keys(p, row, split);
  split_row(p, x, split, x.s + x.len - x.a);   // the visible keys, in order
  if (split >= x.n_splits) return;
  const int kvh = y / p.n_gsub;
  const int gofs = (y - kvh * p.n_gsub) * p.g_tile;
  const int Gn = min(p.g_tile, p.group - gofs);   // heads of this CTA
  const int head0 = kvh * p.group + gofs;
  const int D = p.kv.head_dim;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = D / E;
  const int rl = lane / LPR, cl = lane % LPR;
  const T *kp = static_cast<const T *>(p.kv.k);
  const T *vp = static_cast<const T *>(p.kv.v);
  const int *table = p.kv.table + (size_t)x.seq * p.kv.table_stride;

  float q[G][NV * E], acc[G][NV * E];
#pragma unroll
  for (int g = 0; g < G; ++g) {
#pragma unroll
    for (int v = 0; v < NV; ++v) {
      const int c = cl + v * LPR;
#pragma unroll
      for (int e = 0; e < E; e += 4) {
        float4 t = make_float4(0.f, 0.f, 0.f, 0.f);
        if (g < Gn && c < units)
          t = *reinterpret_cast<const float4 *>(
              p.q + (size_t)row * p.q_sr + (size_t)(head0 + g) * p.q_sh + c * E + e);
        q[g][v * E + e] = t.x * p.qscale;
        q[g][v * E + e + 1] = t.y * p.qscale;
        q[g][v * E + e + 2] = t.z * p.qscale;
        q[g][v * E + e + 3] = t.w * p.qscale;
      }
    }
#pragma unroll
    for (int e = 0; e < NV * E; ++e) acc[g][e] = 0.f;
  }
  // Sum n = u * G + g (key u, head g) ends in the lane of each group that has
  // lane bit o_k set where n has bit half_k, o_k = LPR / 2, LPR / 4, .. and
  // half_k = N / 2, N / 4, ..; with R > 1 a lane has R neighbours.
  int n0 = 0;
#pragma unroll
  for (int o = LPR / 2, half = N / 2; o > 0 && half >= R && half > 0; o >>= 1, half >>= 1)
    if (cl & o) n0 += half;
  const int my_u = n0 / G;
  auto holder = [&](int n) {   // lane of sum n in this lane's group
    int at = rl * LPR;
#pragma unroll
    for (int o = LPR / 2, half = N / 2; o > 0 && half >= R && half > 0; o >>= 1, half >>= 1)
      if (n & half) at += o;
    return at;
  };
  float m[R], l[R];   // of heads n0 % G + i; l of this lane's keys only
#pragma unroll
  for (int i = 0; i < R; ++i) {
    m[i] = -INFINITY;
    l[i] = 0.f;
  }

  const int step = kGenWarps * U * rpw;
  bool bad = false;
  // page of key i (-1: none, or out of range); looked up one step ahead
  auto lookup = [&](int i) {
    if (i >= x.end) return -1;
    const int page = table[p.kv.column(i < x.s ? i : i - x.s + x.a)];
    if (page >= 0 && page < p.kv.n_pages) return page;
    bad = true;
    return -1;
  };
  int next[U];
  const int first = x.begin + warp * U * rpw;
#pragma unroll
  for (int u = 0; u < U; ++u) next[u] = lookup(first + u * rpw + rl);
  for (int i0 = first; i0 < x.end; i0 += step) {
    uint4 kr[U][NV], vr[U][NV];
    bool mine = false;   // whether the row sees this lane's key
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rpw + rl;
      const int pos = i < x.s ? i : i - x.s + x.a;
      const bool ok = next[u] >= 0;
      if (u == my_u) mine = ok;
      const size_t at =
          ok ? p.kv.offset(next[u], kvh, pos - p.kv.column(pos) * p.kv.page_size) : 0;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = cl + v * LPR;
        kr[u][v] = vr[u][v] = make_uint4(0, 0, 0, 0);
        if (ok && c < units) {
          kr[u][v] = ld_stream(kp + at + c * E);
          vr[u][v] = ld_stream(vp + at + c * E);
        }
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) next[u] = lookup(i0 + step + u * rpw + rl);
    float sc[N];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int g = 0; g < G; ++g) sc[u * G + g] = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float f[E];
        UT::unpack(kr[u][v], f);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < E; ++e)
            sc[u * G + g] = fmaf(q[g][v * E + e], f[e], sc[u * G + g]);
      }
    }
#pragma unroll
    for (int o = LPR / 2, half = N / 2; o > 0; o >>= 1, half >>= 1) {
      if (half >= R && half > 0) {
        const bool upper = cl & o;
#pragma unroll
        for (int i = 0; i < half; ++i) {
          const float give = upper ? sc[i] : sc[i + half];
          const float keep = upper ? sc[i + half] : sc[i];
          sc[i] = keep + __shfl_xor_sync(~0u, give, o);
        }
      } else {
#pragma unroll
        for (int i = 0; i < R; ++i) sc[i] += __shfl_xor_sync(~0u, sc[i], o);
      }
    }
    float alpha[R];
    bool moved = false;
#pragma unroll
    for (int i = 0; i < R; ++i) {
      if (!mine) sc[i] = -INFINITY;
      // maximum over the group's keys: the lanes that differ in the bits of u
      float mn = fmaxf(m[i], sc[i]);
#pragma unroll
      for (int o = LPR / 2, k = U; k > 1; o >>= 1, k >>= 1)
        mn = fmaxf(mn, __shfl_xor_sync(~0u, mn, o));
      const float base = mn == -INFINITY ? 0.f : mn;
      alpha[i] = fast_exp2(m[i] - base);   // 0 while m is -inf
      moved |= mn != m[i];
      m[i] = mn;
      sc[i] = fast_exp2(sc[i] - base);
      l[i] = fmaf(l[i], alpha[i], sc[i]);
    }
    if (__any_sync(~0u, moved)) {
#pragma unroll
      for (int g = 0; g < G; ++g) {
        const float f = __shfl_sync(~0u, alpha[g & (R - 1)], holder(g));
#pragma unroll
        for (int e = 0; e < NV * E; ++e) acc[g][e] *= f;
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u) {
      float w[G];
#pragma unroll
      for (int g = 0; g < G; ++g)
        w[g] = __shfl_sync(~0u, sc[(u * G + g) & (R - 1)], holder(u * G + g));
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float f[E];
        UT::unpack(vr[u][v], f);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < E; ++e)
            acc[g][v * E + e] = fmaf(w[g], f[e], acc[g][v * E + e]);
      }
    }
  }
  if (bad) atomicOr(p.err, DEV_ERR_PAGE);

  // every lane's view of all heads: maximum, and the sum over the group's keys
  float mg[G], lg[G];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int o = LPR / 2, k = U; k > 1; o >>= 1, k >>= 1)
      l[i] += __shfl_xor_sync(~0u, l[i], o);
#pragma unroll
  for (int g = 0; g < G; ++g) {
    mg[g] = __shfl_sync(~0u, m[g & (R - 1)], holder(g));
    lg[g] = __shfl_sync(~0u, l[g & (R - 1)], holder(g));
  }
  // join the groups of lanes of this warp
#pragma unroll
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float mo = __shfl_xor_sync(~0u, mg[g], o);
      const float mn = fmaxf(mg[g], mo);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f0 = fast_exp2(mg[g] - base), f1 = fast_exp2(mo - base);
      mg[g] = mn;
      lg[g] = lg[g] * f0 + __shfl_xor_sync(~0u, lg[g], o) * f1;
#pragma unroll
      for (int e = 0; e < NV * E; ++e)
        acc[g][e] = acc[g][e] * f0 + __shfl_xor_sync(~0u, acc[g][e], o) * f1;
    }
  float *w_acc = smem_f;
  float *w_m = smem_f + kGenWarps * Gn * D;
  float *w_l = w_m + kGenWarps * Gn;
  if (rl == 0) {
#pragma unroll
    for (int g = 0; g < G; ++g) {
      if (g >= Gn) continue;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = cl + v * LPR;
        if (c < units)
#pragma unroll
          for (int e = 0; e < E; ++e)
            w_acc[(warp * Gn + g) * D + c * E + e] = acc[g][v * E + e];
      }
      if (cl == 0) {
        w_m[warp * Gn + g] = mg[g];
        w_l[warp * Gn + g] = lg[g];
      }
    }
  }
  __syncthreads();
  finish_split<kGenWarps, kGenWarps * 32>(p, x, row, y, head0, Gn, D, split, smem_f,
                                          &s_flag);
}

// --------------------------------------------------------------------------
// bf16 pages of 8, 16, 32, .. slots, head_dim 64 or 128: TMA and tensor cores.
//
// A producer warp streams KT-key tiles of K and V (128-byte swizzle) from the
// pages into a ring of kStages shared-memory stages; each of four consumer
// warps owns KB blocks of 16 keys of every tile and computes with mma.sync
// m16n8k16, keys as the 16 rows and query heads as the 8 columns:
//   S^T (16 keys x 8 heads) = K_w Q^T,   O^T (D x 8 heads) += V_w^T P^T.
// q and p are fp32 and go in as three bf16 terms each (8 + 8 + 8 bits, exact),
// so the products are exact and sums are fp32, as in the plain formula: two
// terms leave 2.5e-6 of each value, which the result then shows. A tile's
// O^T is added to the running one by ordinary fp32 additions: the tensor
// core's own additions round towards zero, and a chain of them over a long
// row loses 1e-5 (measured over 20011 keys). The work is bound by HBM: a tile is
// 32 KB, 1400 cycles of an SM's share of 6.4 TB/s. Measured in a graph: 64 rows of
// 24/8/128 with 1024 to 8192 keys 191 us (6.35 TB/s), one of 131071 keys 90 (5.95),
// 8 of 1024 to 8192 keys 33 (4.55), 48 of 15/5/64 over 1028 keys of a window 17.5
// (3.4: the first tile and the last write take as long as the stream).
//
// The tiles run over the row's pages: with a window, the pages of the first
// tokens and then those from the window's first page on (all pages where the
// two meet); keys between are masked.
// --------------------------------------------------------------------------
constexpr int kStages = 3;
constexpr int kRowBlock = 512;   // rows that share one axis (and one grid row)
constexpr int kMaxPerSm = 2;     // CTAs that the shared memory lets an SM hold
constexpr int kSegs = 2;         // segments announced to the consumers
constexpr int kSegTiles = 2;     // tiles that a CTA reads in the time of a segment's end
constexpr int kMinTiles = 2;     // least tiles of a share
constexpr int kJobWaits = 1024;  // waits of the joining warp
constexpr int kJoinTiles = 4;    // tiles that a CTA reads in the time of a join

template <int D>
struct Tile {
  static constexpr int KT = D == 128 ? 64 : 128;   // keys
  static constexpr int SUB = D / 64;               // 128-byte columns
  static constexpr int SUB_BYTES = KT * 128;
  static constexpr int BYTES = SUB * SUB_BYTES;    // K or V of a tile: 16 KB
  static constexpr int NCW = 4;                    // consumer warps
  static constexpr int KB = KT / NCW / 16;         // 16-key blocks of a warp
  static constexpr int THREADS = (NCW + 2) * 32;   // a producer warp and a joining one
  static constexpr size_t SMEM = 2 * (size_t)kStages * BYTES + 2 * (kStages + kSegs + 1) * 8;
};

// 4-D tiled TMA load, completion on bar.
__device__ __forceinline__ void tma_load_4d(uint32_t dst, const void *map, uint64_t *bar,
                                            int c0, int c1, int c2, int c3) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes "
      "[%0], [%1, {%3, %4, %5, %6}], [%2];" ::"r"(dst), "l"(map), "r"(smem_u32(bar)), "r"(c0),
      "r"(c1), "r"(c2), "r"(c3)
      : "memory");
}
__device__ __forceinline__ void arrive(uint64_t *bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// Transpose of the 8 x 8 bf16 matrix in the accumulator fragment layout.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
  uint32_t r;
  asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(r) : "r"(x));
  return r;
}
// (x0, x1) as three bf16 pairs of their sign whose sum is x (cut off, not
// rounded, so 8 + 8 + 8 bits hold all 24). The lower terms of an x != 0 are
// kept from zero by 2e-38, far below any product that counts: an infinite k
// or v then gives x * inf, and not the NaN of 0 * inf.
__device__ __forceinline__ void split3(float x0, float x1, uint32_t (&t)[3]) {
  const float e0 = copysignf(x0 == 0.f ? 0.f : 2e-38f, x0);
  const float e1 = copysignf(x1 == 0.f ? 0.f : 2e-38f, x1);
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    t[i] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    x0 = (x0 - bf16lo(t[i])) + e0;
    x1 = (x1 - bf16hi(t[i])) + e1;
  }
}
// The same for weights, which are not negative (one that is 0 where V is
// infinite gives infinity instead of NaN).
__device__ __forceinline__ void split3_weight(float x0, float x1, uint32_t (&t)[3]) {
#pragma unroll
  for (int i = 0; i < 3; ++i) {
    t[i] = __byte_perm(__float_as_uint(x0), __float_as_uint(x1), 0x7632);
    x0 = (x0 - bf16lo(t[i])) + 2e-38f;
    x1 = (x1 - bf16hi(t[i])) + 2e-38f;
  }
}

// The pages of a row as one axis: sink pages, then the window's. n counts its
// slots up to the row's end.
struct PageSpan {
  int sink_pages, first;   // pages [0, sink_pages) and [first, ..)
  int n;
  __device__ __forceinline__ int column(int vp) const {
    return vp < sink_pages ? vp : vp - sink_pages + first;
  }
};
__device__ __forceinline__ PageSpan page_span(const AttnParams &p, int len, int *s, int *a) {
  const int P = p.kv.page_size;
  *s = p.window > 0 ? min(p.sinks, len) : 0;
  *a = p.window > 0 ? max(len - p.window, *s) : 0;
  PageSpan g;
  g.first = p.kv.column(*a);
  g.sink_pages = p.kv.column(*s + P - 1);
  if (g.sink_pages >= g.first) g.sink_pages = g.first = 0;
  g.n = g.sink_pages * P + len - g.first * P;
  return g;
}

// The tiles of all (row, head group) pairs, in that order, are one axis, with
// kSegTiles idle places after each pair for the time that its end takes (32 rows
// of 100 to 2048 keys, 32 heads of 64: 87.7 us without them, 56.6 with one place,
// 53.6 with two, 54.2 with three). It is cut into equal
// shares, one for each CTA. The part of a pair that lies in one share is a
// segment: a share holds the end of one pair, some whole ones and the start of
// another. (Short intervals at the end of the shares, for the CTAs
// that are done first, balance the SMs' bandwidth, but every further segment
// costs its CTA about 2 us and its pair's join 0.15 us: 64 x 24/8/128 took 200
// us with two of 7 tiles, 203 with four of 3 and 192 without; one row of 131071
// keys 93.5, 116 and 96, and 90 without them since.)
struct Segment {
  int row, y;      // row of this block of rows, head group; row < 0: no more
  int t0, t1;      // tiles of the pair
  int first, parts;   // the shares that hold the pair: parts == 1: it is whole
};

__device__ __forceinline__ void bar_consumers(int threads) {
  asm volatile("bar.sync 1, %0;" ::"r"(threads) : "memory");
}
// The same, and whether any of the threads says so.
__device__ __forceinline__ bool bar_any(int threads, bool say) {
  uint32_t r;
  asm volatile(
      "{\n\t.reg .pred p, q;\n\t"
      "setp.ne.u32 p, %2, 0;\n\t"
      "bar.red.or.pred q, 1, %1, p;\n\t"
      "selp.u32 %0, 1, 0, q;\n\t}"
      : "=r"(r)
      : "r"(threads), "r"((uint32_t)say)
      : "memory");
  return r != 0;
}

// Slot of the partials for a segment: a share may hold the end of one pair and
// the start of another.
__device__ __forceinline__ size_t part_slot(size_t share, bool starts) {
  return share * 2 + starts;
}

// Waits for a phase of bar, but not after a failure in this CTA; false if the
// (bounded) wait ran out or there is one.
__device__ __forceinline__ bool wait_phase(uint64_t *bar, uint32_t phase, volatile int *fail) {
  for (uint32_t i = 0; i < 1u << 22; ++i) {
    if (mbar_try_wait(bar, phase)) return true;
    if (*fail) return false;
  }
  return false;
}

// Maximum and 1 / sum over the n parts of one pair, for head h; by one warp.
__device__ __forceinline__ void part_stats(const AttnParams &p, size_t base, int n, int h,
                                           float *top_out, float *inv_out) {
  const int lane = threadIdx.x & 31;
  const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml);
  float mx = -INFINITY, den = 0.f;   // of this lane's parts
#pragma unroll 4
  for (int i = lane; i < n; i += 32) {
    const float2 v = __ldcg(ml + part_slot(base + i, i == 0) * p.g_tile + h);
    const float top = fmaxf(mx, v.x), zero = top == -INFINITY ? 0.f : top;
    den = den * fast_exp2(mx - zero) + v.y * fast_exp2(v.x - zero);
    mx = top;
  }
  float top = mx;
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) top = fmaxf(top, __shfl_xor_sync(~0u, top, d));
  if (mx != -INFINITY) den *= fast_exp2(mx - top);
#pragma unroll
  for (int d = 16; d > 0; d >>= 1) den += __shfl_xor_sync(~0u, den, d);
  *top_out = top;
  *inv_out = den == 0.f ? 0.f : 1.f / den;
}
__device__ __forceinline__ float part_weight(float m, float top, float inv) {
  return m == -INFINITY ? 0.f : fast_exp2(m - top) * inv;
}

// The parts of one pair joined by the consumer warps at the end of their CTA;
// part i lies in share base + i. As many parts as fit the ring, which is free
// by then, are copied there at once (64 of 3 x 128 values: one round trip to
// L2, beside that of the statistics) and summed in order. The code is short on
// purpose: it runs once per CTA, from a cold instruction cache. (Not inlined:
// its registers would take away from those of the tile loop.)
template <int D, int THREADS>
__device__ __noinline__ void join_parts(const AttnParams &p, size_t base, int n, int G,
                                        float4 *ring, float *s_top, float *s_inv,
                                        size_t out_row) {
  constexpr int kWeights = 1024;                              // of 16 bytes, for weights
  constexpr int kUnits = 2 * kStages * Tile<D>::BYTES / 16 - kWeights;   // and for values
  constexpr int kMost = 16 * D / 4 / THREADS;                 // columns of a thread
  const int tid = threadIdx.x, warp = tid >> 5;
  const int cols = G * (D / 4), batch = min(kUnits / cols, 4 * kWeights / G);
  const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml);
  const float4 *acc = reinterpret_cast<const float4 *>(p.part_acc);
  const size_t step = (size_t)p.g_tile * (D / 4);
  float *s_w = reinterpret_cast<float *>(ring + kUnits);
  float4 r[kMost];
#pragma unroll
  for (int j = 0; j < kMost; ++j) r[j] = make_float4(0.f, 0.f, 0.f, 0.f);
  for (int i0 = 0; i0 < n; i0 += batch) {
    const int m = min(batch, n - i0);
    for (int k = warp; k < m; k += THREADS / 32) {   // (a warp per part)
      const float4 *from = acc + part_slot(base + i0 + k, i0 + k == 0) * step;
      const uint32_t to = smem_u32(ring + k * cols);
#pragma unroll 1
      for (int c = tid & 31; c < cols; c += 32)
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + c * 16),
                     "l"(from + c)
                     : "memory");
    }
    if (i0 == 0) {
      for (int h = warp; h < G; h += THREADS / 32) {
        float top, inv;
        part_stats(p, base, n, h, &top, &inv);
        if ((tid & 31) == 0) {
          s_top[h] = top;
          s_inv[h] = inv;
        }
      }
      bar_consumers(THREADS);
    }
    for (int i = tid; i < m * G; i += THREADS) {
      const int part = i / G, h = i - part * G;
      const float x = __ldcg(&ml[part_slot(base + i0 + part, i0 + part == 0) * p.g_tile + h].x);
      s_w[i] = part_weight(x, s_top[h], s_inv[h]);
    }
    asm volatile("cp.async.wait_all;" ::: "memory");
    bar_consumers(THREADS);
#pragma unroll
    for (int j = 0; j < kMost; ++j) {
      const int col = tid + j * THREADS;
      if (col >= cols) break;
      const int h = col / (D / 4);
#pragma unroll 4
      for (int k = 0; k < m; ++k) {
        const float4 v = ring[k * cols + col];
        const float f = s_w[k * G + h];
        r[j].x = fmaf(f, v.x, r[j].x);
        r[j].y = fmaf(f, v.y, r[j].y);
        r[j].z = fmaf(f, v.z, r[j].z);
        r[j].w = fmaf(f, v.w, r[j].w);
      }
    }
    bar_consumers(THREADS);
  }
#pragma unroll
  for (int j = 0; j < kMost; ++j) {
    const int col = tid + j * THREADS;
    if (col >= cols) break;
    const int h = col / (D / 4);
    const size_t at = out_row + (size_t)h * p.o_sh + (col - h * (D / 4)) * 4;
    store_out(p, at, r[j].x);
    store_out(p, at + 1, r[j].y);
    store_out(p, at + 2, r[j].z);
    store_out(p, at + 3, r[j].w);
  }
}

// A segment that ended before its CTA's last one, for the joining warp.
struct Job {
  size_t base, out_row;   // the pair's first share, its output
  int first, parts, G;    // parts == 0: no more
};

// The same sums by one warp, while the others go on with the next segment.
template <int D>
__device__ __noinline__ void join_by_warp(const AttnParams &p, const Job &job) {
  const int lane = threadIdx.x & 31;
  const float2 *ml = reinterpret_cast<const float2 *>(p.part_ml);
  const float4 *acc = reinterpret_cast<const float4 *>(p.part_acc);
  for (int h = 0; h < job.G; ++h) {
    float top, inv;
    part_stats(p, job.base, job.parts, h, &top, &inv);
    if (lane >= D / 4) continue;
    float4 r = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 8
    for (int i = 0; i < job.parts; ++i) {
      const size_t at = part_slot(job.base + i, i == 0) * p.g_tile + h;
      const float4 v = __ldcg(acc + at * (D / 4) + lane);
      const float f = part_weight(__ldcg(ml + at).x, top, inv);
      r.x = fmaf(f, v.x, r.x);
      r.y = fmaf(f, v.y, r.y);
      r.z = fmaf(f, v.z, r.z);
      r.w = fmaf(f, v.w, r.w);
    }
    const size_t at = job.out_row + (size_t)h * p.o_sh + lane * 4;
    store_out(p, at, r.x);
    store_out(p, at + 1, r.y);
    store_out(p, at + 2, r.z);
    store_out(p, at + 3, r.w);
  }
}

template <int D, int QB>
__global__ void __launch_bounds__(Tile<D>::THREADS, QB == 1 || D == 64 ? 2 : 1)
    paged_mma_kernel(const __grid_constant__ AttnParams p, const __grid_constant__ CUtensorMap mk,
                     const __grid_constant__ CUtensorMap mv, const int slots_first) {
  griddep_launch();
  using T = Tile<D>;
  constexpr int KT = T::KT, NCW = T::NCW, KB = T::KB;
  extern __shared__ __align__(1024) uint8_t smem[];   // stages of (K, V)
  uint64_t *full = reinterpret_cast<uint64_t *>(smem + 2 * kStages * T::BYTES);
  uint64_t *empty = full + kStages;
  uint64_t *seg_full = empty + kStages, *seg_empty = seg_full + kSegs;
  uint64_t *job_full = seg_empty + kSegs, *job_empty = job_full + 1;
  __shared__ uint32_t s_bad[kStages];                 // bad pages of a stage's tile
  __shared__ Segment s_seg[kSegs];
  __shared__ Job s_job;
  __shared__ long s_cum[kRowBlock + 1], s_warp[NCW + 2];   // (512 x 2^24 places)
  __shared__ int s_len[kRowBlock], s_most[NCW + 2], s_last;
  __shared__ volatile int s_fail;
  __shared__ float s_m[NCW][16], s_l[NCW][16];
  const int row0 = blockIdx.y * kRowBlock, nrows = min(kRowBlock, p.rows - row0);
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  if (smem_u32(smem) & 1023) {
    griddep_wait();
    if (tid == 0) atomicOr(p.err, DEV_ERR_SMEM_ALIGN);
    return;
  }
  if (tid == 0) {
    for (int s = 0; s < kStages; ++s) {
      mbar_init(&full[s], 1);
      mbar_init(&empty[s], NCW);
    }
    for (int s = 0; s < kSegs; ++s) {
      mbar_init(&seg_full[s], 1);
      mbar_init(&seg_empty[s], NCW);
    }
    mbar_init(job_full, 1);
    mbar_init(job_empty, 1);
    fence_mbar_init();
    s_fail = 0;
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mk) : "memory");
    asm volatile("prefetch.tensormap [%0];" ::"l"(&mv) : "memory");
  }
  griddep_wait();

  // ---- places of every row's pairs, summed up (a row without keys has a tile,
  // empty)
  const int per = (nrows + T::THREADS - 1) / T::THREADS;
  int sum = 0, most = 0;   // (a warp's 96 rows: below 2^31)
  for (int i = tid * per; i < min(nrows, (tid + 1) * per); ++i) {
    int len = p.row_len[row0 + i];
    const int cap = p.kv.table_cols * p.kv.page_size;
    if (len > cap) {
      len = cap;
      if (blockIdx.x == 0) atomicOr(p.err, DEV_ERR_LEN_CLAMPED);
    }
    const int seq = p.row_seq ? p.row_seq[row0 + i] : row0 + i;
    if (seq < 0 || seq >= p.kv.n_seq) {
      len = 0;
      if (blockIdx.x == 0) atomicOr(p.err, DEV_ERR_PAGE);
    }
    if (len < 0) len = 0;
    int xs, xa;
    const int places = max(1, (page_span(p, len, &xs, &xa).n + KT - 1) / KT) + kSegTiles;
    s_len[i] = len;
    s_cum[i] = places;
    sum += places;
    most = max(most, places);
  }
  int scan = sum;
#pragma unroll
  for (int o = 1; o < 32; o <<= 1) {
    const int v = __shfl_up_sync(~0u, scan, o);
    if (lane >= o) scan += v;
    most = max(most, __shfl_xor_sync(~0u, most, o));
  }
  if (lane == 31) {
    s_warp[warp] = scan;
    s_most[warp] = most;
  }
  __syncthreads();
  long before = scan - sum, total = 0;
#pragma unroll
  for (int w = 0; w < NCW + 2; ++w) {
    if (w < warp) before += s_warp[w];
    total += s_warp[w];
    most = max(most, s_most[w]);
  }
  for (int i = tid * per; i < min(nrows, (tid + 1) * per); ++i) {
    const long places = s_cum[i];
    s_cum[i] = before;
    before += places;
  }
  if (tid == 0) s_cum[nrows] = total;
  __syncthreads();

  // ---- shares. Where every pair can have a CTA of its own and sharing would
  // save less than kJoinTiles, pairs stay whole: joining costs about as much.
  const int ncta = gridDim.x;
  const long work = total * p.n_y;
  long share = (work + ncta - 1) / ncta;
  if (share < kMinTiles + kSegTiles) share = kMinTiles + kSegTiles;
  const bool whole_pairs = (long)nrows * p.n_y <= ncta && most <= share + kJoinTiles;
  const size_t base = (size_t)blockIdx.y * ncta;   // of the shares
  const int P = p.kv.page_size, box = min(P, KT);   // slots of one load

  if (warp == NCW) {
    // ---- producer: lane (kv, sub, page of the tile) issues its loads
    const int pt = KT / box;
    const int j = lane % pt, sub = lane / pt % T::SUB, is_v = lane / pt / T::SUB;
    const bool mine = is_v < 2;
    const uint32_t dst0 = smem_u32(smem) + (is_v ? T::BYTES : 0) + sub * T::SUB_BYTES +
                          j * box * 128;
    int it = 0, segs = 0;   // tiles issued, segments announced
    bool failed = false;
    auto announce = [&](const Segment &g) {
      const int s = segs % kSegs;
      if (segs >= kSegs && !wait_phase(&seg_empty[s], (segs / kSegs - 1) & 1, &s_fail))
        failed = true;
      failed = __any_sync(~0u, failed);
      if (failed) return;
      if (lane == 0) {
        s_seg[s] = g;
        arrive(&seg_full[s]);
      }
      ++segs;
    };
    // announces and loads one segment
    auto stream = [&](const Segment &g) {
      announce(g);
      if (failed) return;
      int xs, xa;
      const PageSpan ps = page_span(p, s_len[g.row], &xs, &xa);
      const int seq = p.row_seq ? p.row_seq[row0 + g.row] : row0 + g.row;
      const int *table = p.kv.table + (size_t)seq * p.kv.table_stride;
      const int kvh = g.y / p.n_gsub;
      // page of tile t for this lane: -1 past the end, -2 out of range
      auto entry = [&](int t) {
        const int u = t * KT + j * box;
        if (t >= g.t1 || u >= ps.n) return -1;
        const int page = table[ps.column(p.kv.column(u))];
        return page >= 0 && page < p.kv.n_pages ? page : -2;
      };
      int next0 = entry(g.t0), next1 = entry(g.t0 + 1);
      for (int t = g.t0; t < g.t1; ++t, ++it) {
        const int s = it % kStages, page = next0;
        next0 = next1;
        next1 = entry(t + 2);
        const uint32_t good = __ballot_sync(~0u, mine && page >= 0);
        const uint32_t bad = __ballot_sync(~0u, lane < pt && page == -2);
        if (it >= kStages && !wait_phase(&empty[s], (it / kStages - 1) & 1, &s_fail))
          failed = true;
        failed = __any_sync(~0u, failed);
        if (failed) return;
        if (lane == 0) {
          s_bad[s] = bad;
          mbar_expect_tx(&full[s], __popc(good) * box * 128);
          if (bad) atomicOr(p.err, DEV_ERR_PAGE);
        }
        __syncwarp();
        if (mine && page >= 0) {
          const int u = t * KT + j * box;
          const int slot = u - p.kv.column(u) * P;
          tma_load_4d(dst0 + s * 2 * T::BYTES, is_v ? &mv : &mk, &full[s], sub * 64,
                      slots_first ? kvh : slot, slots_first ? slot : kvh, page);
        }
      }
    };
    auto tiles_of = [&](int row) { return (int)(s_cum[row + 1] - s_cum[row]) - kSegTiles; };
    Segment g;
    if (whole_pairs) {
      if (blockIdx.x < nrows * p.n_y) {
        g.row = blockIdx.x / p.n_y;
        g.y = blockIdx.x - g.row * p.n_y;
        g.t0 = 0;
        g.t1 = tiles_of(g.row);
        g.parts = 1;
        stream(g);
      }
    } else {
      long w = blockIdx.x * share;
      const long w1 = min(w + share, work);
      int lo = 0, hi = nrows;   // s_cum[lo] * n_y <= w < s_cum[hi] * n_y
      while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (s_cum[mid] * p.n_y <= w) lo = mid; else hi = mid;
      }
      g.row = lo;
      int nt = tiles_of(lo);
      const long rem = w - s_cum[lo] * p.n_y;
      g.y = (int)(rem / (nt + kSegTiles));
      g.t0 = (int)(rem - (long)g.y * (nt + kSegTiles));
      while (w < w1 && !failed) {
        const long begin = w - g.t0;   // of the pair
        if (g.t0 < nt) {
          g.t1 = (int)min((long)nt, g.t0 + w1 - w);
          g.first = (int)(begin / share);
          g.parts = (int)((begin + nt - 1) / share) - g.first + 1;
          stream(g);
        }
        w = begin + nt + kSegTiles;
        g.t0 = 0;
        if (++g.y == p.n_y) {
          g.y = 0;
          ++g.row;
          if (g.row < nrows) nt = tiles_of(g.row);
        }
      }
    }
    Segment none;
    none.row = -1;
    if (!failed) announce(none);
    if (failed) {
      // let the copies in flight land (bounded) before the CTA exits
      if (lane == 0) {
        atomicOr(p.err, DEV_ERR_WAIT_TIMEOUT);
        s_fail = 1;
        for (int t = max(0, it - kStages); t < it; ++t)
          mbar_wait_bounded(&full[t % kStages], (t / kStages) & 1, 1u << 12);
      }
      __syncwarp();
    }
    return;
  }

  auto last_part = [&](int first, int parts) {   // one thread's: takes a ticket
    int *ticket = p.counters + base + first;
    __threadfence();   // (of all writes that a barrier has ordered before)
    const bool last = atomicAdd(ticket, 1) == parts - 1;
    if (last) *ticket = 0;
    __threadfence();
    return last;
  };
  if (warp == NCW + 1) {
    // ---- joining warp (its wait lasts as long as the CTA's first segment, whose
    // own waits are bounded)
    for (int jobs = 0;; ++jobs) {
      bool told = false;
      for (int n = 0; n < kJobWaits && !told && !s_fail; ++n)
        told = __all_sync(~0u, wait_phase(job_full, jobs & 1, &s_fail));
      if (!told) {
        if (lane == 0 && !s_fail) atomicOr(p.err, DEV_ERR_WAIT_TIMEOUT);
        s_fail = 1;
        return;
      }
      const Job job = s_job;
      __syncwarp();
      if (lane == 0) arrive(job_empty);
      if (job.parts == 0) return;
      bool last = false;
      if (lane == 0) last = last_part(job.first, job.parts);
      last = __any_sync(~0u, last);
      __syncwarp();
      if (last) join_by_warp<D>(p, job);
    }
  }

  // ---- consumers. Fragments: rows (keys, or dims of O^T) r0 and r0 + 8,
  // columns (heads) cq and cq + 1 of every block of 8. A wait that runs out
  // sets s_fail and an error bit; the CTA then goes through its segment
  // without waiting, so that barriers stay in step, and ends.
  const int r0 = lane >> 2, cq = (lane & 3) * 2;
  // ldmatrix rows: K as the A operand, V^T by the transposing load
  const int key0 = warp * KB * 16;   // this warp's first key of a tile
  const int a_key = key0 + ((lane >> 3) & 1) * 8 + (lane & 7), a_dim = (lane >> 4) * 8;
  const int t_key = key0 + (lane >> 4) * 8 + (lane & 7), t_dim = ((lane >> 3) & 1) * 8;
  // the next segment announced; false on a failure (for all warps or none)
  int segs = 0;
  auto next_segment = [&](Segment *g) {
    const int s = segs % kSegs;
    const bool told = wait_phase(&seg_full[s], (segs / kSegs) & 1, &s_fail);
    if (!told) {
      if (!s_fail) atomicOr(p.err, DEV_ERR_WAIT_TIMEOUT);
      s_fail = 1;
    }
    if (bar_any(NCW * 32, !told)) return false;
    *g = s_seg[s];
    ++segs;
    return true;
  };
  struct Heads { int head0, G; };
  auto heads_of = [&](const Segment &g) {
    const int kvh = g.y / p.n_gsub, gofs = (g.y - kvh * p.n_gsub) * p.g_tile;
    return Heads{kvh * p.group + gofs, min(p.g_tile, p.group - gofs)};
  };
  float2 qv[QB][D / 16][2];   // q of the segment that comes next
  auto load_q = [&](const Segment &g) {
    const Heads hd = heads_of(g);
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      const float *q = p.q + (size_t)(row0 + g.row) * p.q_sr +
                       (size_t)(hd.head0 + qb * 8 + r0) * p.q_sh + cq;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk)
#pragma unroll
        for (int f = 0; f < 2; ++f)
          qv[qb][kk][f] = qb * 8 + r0 < hd.G
                              ? *reinterpret_cast<const float2 *>(q + kk * 16 + 8 * f)
                              : make_float2(0.f, 0.f);
    }
  };
  int it = 0, jobs = 0;
  // whether the joining warp has the last job (until then s_job is not ours)
  auto job_taken = [&]() {
    if (jobs == 0 || wait_phase(job_empty, (jobs - 1) & 1, &s_fail)) return true;
    if (!s_fail) atomicOr(p.err, DEV_ERR_WAIT_TIMEOUT);
    s_fail = 1;
    return false;
  };
  Segment g;
  if (!next_segment(&g)) return;
  if (QB == 1 && g.row >= 0) load_q(g);
  while (g.row >= 0) {
    if (QB > 1) load_q(g);
    const int row = row0 + g.row;
    int xs, xa;
    const PageSpan ps = page_span(p, s_len[g.row], &xs, &xa);
    const int head0 = heads_of(g).head0, G = heads_of(g).G;
    const int sink_keys = ps.sink_pages * P;
    float o[QB][D / 16][4], m_r[QB][2], l_r[QB][2];
    uint32_t qf[QB][D / 16][2][3];
#pragma unroll
    for (int qb = 0; qb < QB; ++qb) {
      m_r[qb][0] = m_r[qb][1] = -INFINITY;
      l_r[qb][0] = l_r[qb][1] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
#pragma unroll
        for (int e = 0; e < 4; ++e) o[qb][kk][e] = 0.f;
#pragma unroll
        for (int f = 0; f < 2; ++f)
          split3(qv[qb][kk][f].x * p.qscale, qv[qb][kk][f].y * p.qscale, qf[qb][kk][f]);
      }
    }

    for (int t = g.t0; t < g.t1; ++t, ++it) {
      const int s = it % kStages;
      const bool ok = wait_phase(&full[s], (it / kStages) & 1, &s_fail);
      if (!__all_sync(~0u, ok)) {
        if (lane == 0 && !s_fail) atomicOr(p.err, DEV_ERR_WAIT_TIMEOUT);
        s_fail = 1;
        continue;
      }
      const uint32_t kt = smem_u32(smem) + s * 2 * T::BYTES;
      const uint32_t vt = kt + T::BYTES;
      const int u0 = t * KT + key0;
      const uint32_t bad = s_bad[s];
      // whether the row sees key u0 + i
      auto sees = [&](int i) {
        const int u = u0 + i;
        if (u >= ps.n || (bad && (bad >> ((key0 + i) / box) & 1))) return false;
        const int pos = u < sink_keys ? u : u - sink_keys + ps.first * P;
        return pos < xs || pos >= xa;
      };
      const int pos0 = u0 < sink_keys ? 0 : u0 - sink_keys + ps.first * P;
      const bool whole = !bad && u0 + KB * 16 <= ps.n && pos0 >= xa;

      float sc[QB][KB][3][4];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb)
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int i = 0; i < 3; ++i)
#pragma unroll
            for (int e = 0; e < 4; ++e) sc[qb][kb][i][e] = 0.f;
#pragma unroll
      for (int kk = 0; kk < D / 16; ++kk) {
        const int dim = kk * 16 + a_dim;
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t ka[4];
          ldsm_x4(kt + (dim >> 6) * T::SUB_BYTES + (a_key + kb * 16) * 128 +
                      ((((dim & 63) >> 3) ^ (a_key & 7)) << 4),
                  ka[0], ka[1], ka[2], ka[3]);
#pragma unroll
          for (int qb = 0; qb < QB; ++qb)
#pragma unroll
            for (int i = 0; i < 3; ++i)   // (independent sums)
              mma_bf16(sc[qb][kb][i], ka, qf[qb][kk][0][i], qf[qb][kk][1][i]);
        }
      }
      uint32_t pb[QB][KB][2][3];
#pragma unroll
      for (int qb = 0; qb < QB; ++qb) {
        float w[KB][4];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 4; ++e)
            w[kb][e] = sc[qb][kb][0][e] + (sc[qb][kb][1][e] + sc[qb][kb][2][e]);
        if (!whole) {
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            if (!sees(kb * 16 + r0)) w[kb][0] = w[kb][1] = -INFINITY;
            if (!sees(kb * 16 + r0 + 8)) w[kb][2] = w[kb][3] = -INFINITY;
          }
        }
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          float mx = fmaxf(w[0][c], w[0][c + 2]);
#pragma unroll
          for (int kb = 1; kb < KB; ++kb) mx = fmaxf(mx, fmaxf(w[kb][c], w[kb][c + 2]));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 4));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 8));
          mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, 16));
          const float mn = fmaxf(m_r[qb][c], mx);
          const float base = mn == -INFINITY ? 0.f : mn;
          if (mn != m_r[qb][c]) {
            const float alpha = fast_exp2(m_r[qb][c] - base);   // 0 while m is -inf
            l_r[qb][c] *= alpha;
#pragma unroll
            for (int mb = 0; mb < D / 16; ++mb) {
              o[qb][mb][c] *= alpha;
              o[qb][mb][c + 2] *= alpha;
            }
            m_r[qb][c] = mn;
          }
#pragma unroll
          for (int kb = 0; kb < KB; ++kb) {
            w[kb][c] = fast_exp2(w[kb][c] - base);
            w[kb][c + 2] = fast_exp2(w[kb][c + 2] - base);
            l_r[qb][c] += w[kb][c] + w[kb][c + 2];
          }
        }
#pragma unroll
        for (int kb = 0; kb < KB; ++kb) {
          uint32_t t0[3], t1[3];
          split3_weight(w[kb][0], w[kb][1], t0);   // key r0
          split3_weight(w[kb][2], w[kb][3], t1);   // key r0 + 8
#pragma unroll
          for (int i = 0; i < 3; ++i) {
            pb[qb][kb][0][i] = transpose8(t0[i]);
            pb[qb][kb][1][i] = transpose8(t1[i]);
          }
        }
      }
      if (!whole) {
        // V of keys that the row does not see may be anything, NaN too, and
        // 0 * NaN is no 0: clear it
        for (int i = lane; i < KB * 16 * T::SUB * 8; i += 32) {
          const int key = i / (T::SUB * 8), c = i % (T::SUB * 8);
          if (!sees(key))
            asm volatile("st.shared.v4.u32 [%0], {%1, %1, %1, %1};" ::"r"(
                             vt + (c >> 3) * T::SUB_BYTES + (key0 + key) * 128 +
                             ((c & 7) << 4)),
                         "r"(0)
                         : "memory");
        }
        __syncwarp();
      }
#pragma unroll
      for (int mb = 0; mb < D / 16; ++mb) {
        const int dim = mb * 16 + t_dim;
        uint32_t va[KB][4];
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
          ldsm_x4_t(vt + (dim >> 6) * T::SUB_BYTES + (t_key + kb * 16) * 128 +
                        ((((dim & 63) >> 3) ^ (t_key & 7)) << 4),
                    va[kb][0], va[kb][1], va[kb][2], va[kb][3]);
#pragma unroll
        for (int qb = 0; qb < QB; ++qb) {
          float d[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
          for (int i = 2; i >= 0; --i)
#pragma unroll
            for (int kb = 0; kb < KB; ++kb)
              mma_bf16(d, va[kb], pb[qb][kb][0][i], pb[qb][kb][1][i]);
#pragma unroll
          for (int e = 0; e < 4; ++e) o[qb][mb][e] += d[e];
        }
      }
      if (t + 1 < g.t1) {   // (the segment's last stage is held for the join)
        if (!whole) fence_proxy_async();   // generic writes before the next TMA
        __syncwarp();
        if (lane == 0) arrive(&empty[s]);
      }
    }

    // ---- join the warps through the last stage's 32 KB, which the producer
    // gets back afterwards; it loads the next segment's tiles meanwhile, and
    // its q is on the way
    const int held = (it - 1) % kStages;
    Segment next;
    if (!next_segment(&next)) return;   // (a barrier: all have read the stage)
    if (QB == 1 && next.row >= 0) load_q(next);   // (two blocks take too many registers)
    float *w_acc = reinterpret_cast<float *>(smem + held * 2 * T::BYTES);   // [NCW][G][D]
#pragma unroll
    for (int qb = 0; qb < QB; ++qb)
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        float l = l_r[qb][c];
#pragma unroll
        for (int d = 4; d < 32; d <<= 1) l += __shfl_xor_sync(~0u, l, d);
        const int h = qb * 8 + cq + c;
        if (h >= G) continue;
#pragma unroll
        for (int mb = 0; mb < D / 16; ++mb) {
          w_acc[(warp * G + h) * D + mb * 16 + r0] = o[qb][mb][c];
          w_acc[(warp * G + h) * D + mb * 16 + r0 + 8] = o[qb][mb][c + 2];
        }
        if (r0 == 0) {
          s_m[warp][h] = m_r[qb][c];
          s_l[warp][h] = l;
        }
      }
    bar_consumers(NCW * 32);
    const bool part = g.parts > 1;
    const size_t out_row = (size_t)row * p.o_sr + (size_t)head0 * p.o_sh;
    const size_t mine = part_slot(base + blockIdx.x, g.t0 == 0) * p.g_tile;
    for (int i = tid; i < G * D; i += NCW * 32) {
      const int h = i / D;
      float mx = -INFINITY;
#pragma unroll
      for (int w = 0; w < NCW; ++w) mx = fmaxf(mx, s_m[w][h]);
      float num = 0.f, den = 0.f;
#pragma unroll
      for (int w = 0; w < NCW; ++w) {
        const float m = s_m[w][h];
        // (a warp without a visible key has m = -inf and sums of zero)
        const float f = m == -INFINITY ? 0.f : fast_exp2(m - mx);
        num = fmaf(w_acc[w * G * D + i], f, num);
        den = fmaf(s_l[w][h], f, den);
      }
      if (!part) {
        store_out(p, out_row + (size_t)h * p.o_sh + (i - h * D), den == 0.f ? 0.f : num / den);
      } else {
        p.part_acc[mine * D + i] = num;
        if (i == h * D) {
          p.part_ml[(mine + h) * 2] = mx;
          p.part_ml[(mine + h) * 2 + 1] = den;
        }
      }
    }
    if (part) {
      // the CTA that finishes a pair's last part joins them all: the joining
      // warp, or at the end of the share all consumers
      bar_consumers(NCW * 32);
      if (next.row >= 0) {
        if (tid == 0 && job_taken()) {
          s_job = Job{base + g.first, out_row, g.first, g.parts, G};
          arrive(job_full);
        }
        ++jobs;
      } else {
        if (tid == 0) s_last = last_part(g.first, g.parts);
        bar_consumers(NCW * 32);
        if (s_last)
          join_parts<D, NCW * 32>(p, base + g.first, g.parts, G,
                                  reinterpret_cast<float4 *>(smem), s_m[0], s_l[0], out_row);
      }
    }
    if (next.row >= 0) {
      fence_proxy_async();
      __syncwarp();
      if (lane == 0) {
        arrive(&empty[held]);
        arrive(&seg_empty[(segs - 2) % kSegs]);
      }
    }
    g = next;
  }
  if (tid == 0 && job_taken()) {
    s_job.parts = 0;
    arrive(job_full);
  }
}

// --------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------
using MmaKern = void (*)(const AttnParams, const CUtensorMap, const CUtensorMap, const int);

// The kernel for D and heads per CTA, and its CTAs per SM (looked up once per
// device).
template <int D, int QB>
int mma_setup(MmaKern *kern, int *per_sm) {
  static int occupancy[64] = {};
  int dev = 0;
  TLLM_CUDA(cudaGetDevice(&dev));
  TLLM_CHECK_ARG(dev >= 0 && dev < 64, "device index %d out of range", dev);
  *kern = paged_mma_kernel<D, QB>;
  if (!occupancy[dev]) {
    TLLM_CUDA(cudaFuncSetAttribute(*kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)Tile<D>::SMEM));
    int n = 0;
    TLLM_CUDA(cudaOccupancyMaxActiveBlocksPerMultiprocessor(&n, *kern, Tile<D>::THREADS,
                                                            Tile<D>::SMEM));
    TLLM_CHECK_ARG(n > 0, "the kernel does not fit the device");
    occupancy[dev] = n;
  }
  *per_sm = occupancy[dev];
  return TLLM_OK;
}

// Tensor map of K or V pages with boxes of 64 values x `rows` slots of one
// head and page; the axes are in the order of their strides.
int page_map(CUtensorMap *m, const void *base, const tllm_paged_kv *kv, int rows,
             bool slots_first) {
  const long slot = kv->slot_stride * 2;
  const long head = kv->n_kv_head > 1 ? kv->head_stride * 2 : slot * kv->page_size;
  const long page = kv->n_pages > 1 ? kv->page_stride * 2
                                    : (slot > head ? slot : head) * kv->page_size;
  const long dims[4] = {kv->head_dim, slots_first ? kv->n_kv_head : kv->page_size,
                        slots_first ? kv->page_size : kv->n_kv_head, kv->n_pages};
  const long strides[3] = {slots_first ? head : slot, slots_first ? slot : head, page};
  const int box[4] = {64, slots_first ? 1 : rows, slots_first ? rows : 1, 1};
  return make_map(m, base, TLLM_BF16, 4, dims, strides, box, true);
}

// The tensor-core kernel takes bf16 pages of a power of two >= 8 slots (a TMA
// box of 8 rows is one swizzle atom, and pages divide tiles or tiles pages),
// head_dim 64 or 128, and distinct heads and pages (strides > 0).
bool mma_takes(const tllm_paged_kv *kv, const PagedView &w) {
  return kv->kv_dtype == TLLM_BF16 && (kv->head_dim == 64 || kv->head_dim == 128) &&
         w.page_shift >= 3 && kv->n_pages > 0 && (kv->n_kv_head == 1 || kv->head_stride > 0) &&
         (kv->n_pages == 1 || kv->page_stride > 0);
}

template <typename T, int G, int NV, int LPR>
int launch_rows(const AttnParams &p, dim3 grid, cudaStream_t st) {
  const int D = p.kv.head_dim;
  size_t smem = (size_t)kGenWarps * G * (D + 2) * sizeof(float);
  const size_t sw = (size_t)G * kMaxSplits * sizeof(float);
  if (sw > smem) smem = sw;
  auto kern = paged_rows_kernel<T, G, NV, LPR>;
  if (smem > 48 * 1024)
    TLLM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)smem));
  TLLM_CUDA(launch_pdl(kern, grid, dim3(kGenWarps * 32), smem, st, p));
  return TLLM_OK;
}

template <typename T, int NV, int LPR>
int launch_rows_g(const AttnParams &p, dim3 grid, cudaStream_t st) {
  if (p.g_tile == 1) return launch_rows<T, 1, NV, LPR>(p, grid, st);
  if (p.g_tile == 2) return launch_rows<T, 2, NV, LPR>(p, grid, st);
  if (p.g_tile <= 4) return launch_rows<T, 4, NV, LPR>(p, grid, st);
  if constexpr (NV * Unit<T>::N <= 8) return launch_rows<T, 8, NV, LPR>(p, grid, st);
  set_error("group tile %d not built", p.g_tile);
  return TLLM_ERR_UNSUPPORTED;
}

template <typename T>
int launch_rows_t(const AttnParams &p, int lpr, int nv, dim3 grid, cudaStream_t st) {
  if (lpr == 8) return launch_rows_g<T, 1, 8>(p, grid, st);
  if (lpr == 16) return launch_rows_g<T, 1, 16>(p, grid, st);
  if (nv == 1) return launch_rows_g<T, 1, 32>(p, grid, st);
  if (nv == 2) return launch_rows_g<T, 2, 32>(p, grid, st);
  if constexpr (Unit<T>::N == 4) return launch_rows_g<T, 4, 32>(p, grid, st);
  set_error("head_dim %d not built", p.kv.head_dim);
  return TLLM_ERR_UNSUPPORTED;
}

// A split of fewer keys costs more than it saves. With 64, 128 and 256: 6 rows of
// 12 heads of 64 fp32 with 17 to 1003 keys 12.9, 10.2 and 14.0 us; one row of
// 24/8/128 fp32 with 3000 keys 19.3, 14.8, 18.8; 4 rows of 9/3/64 fp32 with 100 to
// 2000 keys 8.4, 9.2, 10.5; 16 rows of 6/2/96 bf16 with 100 to 4000 keys 23.3, 23.2,
// 16.9. Larger calls take longer splits anyway.
constexpr int kMinKeys = 128;

constexpr size_t kMaxScratch = 512u << 20;   // of the splits, whatever the rows

// Keys per split, a multiple of `tile`, for `pairs` (row, head group) pairs
// of at most max_keys keys and about `keys` in all rows.
int plan_chunk(int tile, long rows, int n_y, long keys, long max_keys, long slots) {
  const long tiles = (max_keys + tile - 1) / tile;
  long c = (keys * n_y / tile + slots - 1) / slots;   // one CTA per slot
  if (rows * n_y >= slots || c > 32) c = c < 32 ? 32 : c;
  if (c * tile < kMinKeys) c = (kMinKeys + tile - 1) / tile;
  const long least = (tiles + kMaxSplits - 1) / kMaxSplits;
  if (c < least) c = least;
  if (c > tiles) c = tiles > 0 ? tiles : 1;
  return (int)(c * tile);
}

}  // namespace

int paged_view(const tllm_paged_kv *kv, PagedView *w) {
  TLLM_CHECK_ARG(kv, "kv is NULL");
  TLLM_CHECK_ARG(kv->kv_dtype == TLLM_F32 || kv->kv_dtype == TLLM_BF16,
                 "kv_dtype must be F32 or BF16");
  TLLM_CHECK_ARG(kv->n_pages >= 0 && kv->page_size >= 1 && kv->n_kv_head >= 1 &&
                     kv->head_dim >= 1 && kv->n_seq >= 0 && kv->table_cols >= 0,
                 "invalid paged cache: %d pages of %d slots, %d heads of %d, table %d x %d",
                 kv->n_pages, kv->page_size, kv->n_kv_head, kv->head_dim, kv->n_seq,
                 kv->table_cols);
  TLLM_CHECK_ARG((long)kv->table_cols * kv->page_size < (1L << 30),
                 "table_cols * page_size must be below 2^30");
  TLLM_CHECK_ARG(kv->page_stride >= 0 && kv->head_stride >= 0 && kv->slot_stride >= kv->head_dim &&
                     (kv->table_stride >= kv->table_cols || kv->n_seq <= 1),
                 "invalid strides of a paged cache");
  TLLM_CHECK_ARG((kv->k_pages && kv->v_pages) || kv->n_pages == 0, "NULL page pointer");
  TLLM_CHECK_ARG(kv->table || kv->n_seq == 0 || kv->table_cols == 0, "NULL page table");
  w->k = kv->k_pages;
  w->v = kv->v_pages;
  w->table = kv->table;
  w->page_stride = kv->page_stride;
  w->head_stride = kv->head_stride;
  w->slot_stride = kv->slot_stride;
  w->table_stride = kv->table_stride;
  w->n_pages = kv->n_pages;
  w->page_size = kv->page_size;
  w->page_shift = -1;
  for (int i = 0; i < 31; ++i)
    if (kv->page_size == 1 << i) w->page_shift = i;
  w->n_kv = kv->n_kv_head;
  w->head_dim = kv->head_dim;
  w->n_seq = kv->n_seq;
  w->table_cols = kv->table_cols;
  return TLLM_OK;
}

}  // namespace tllm

using namespace tllm;

extern "C" int tllm_paged_attention_workspace(int rows, int n_head, int n_kv_head,
                                              int head_dim, size_t *partial_bytes,
                                              size_t *counter_bytes) {
  TLLM_CHECK_ARG(partial_bytes && counter_bytes, "NULL output pointer");
  TLLM_CHECK_ARG(rows >= 0 && n_head > 0 && n_kv_head > 0 && head_dim > 0, "invalid shape");
  TLLM_CHECK_ARG(n_head % n_kv_head == 0, "n_head (%d) must be divisible by n_kv_head (%d)",
                 n_head, n_kv_head);
  // One token per row and split (heads of a KV head padded to a tile of 1, 2, 4
  // or 8): splits that fill the GPU a few times over, at least 8 within 512 MB
  // (64000 heads of 128 in all rows; so many fill it by themselves). Or two parts
  // of up to 16 heads per share of the tensor-core kernel.
  long splits = 8192 / ((long)(rows > 0 ? rows : 1) * n_kv_head);
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits < 8) splits = 8;
  const size_t row = (head_dim + 2) * sizeof(float);
  const size_t blocks = (size_t)(rows + kRowBlock - 1) / kRowBlock;
  const size_t ctas = (size_t)kMaxPerSm * sm_count();
  const int group = n_head / n_kv_head;
  const size_t all = (size_t)rows * n_head * 2 * splits * row;
  const size_t a = all < kMaxScratch ? all : kMaxScratch;
  const size_t b = blocks * ctas * 2 * (group < 16 ? group : 16) * row;
  *partial_bytes = a > b ? a : b;
  const size_t c = (size_t)rows * n_head;
  const size_t d = blocks * ctas;
  *counter_bytes = (c > d ? c : d) * sizeof(int32_t);
  return TLLM_OK;
}

extern "C" int tllm_paged_attention(const tllm_paged_kv *kv, const tllm_paged_attn *a,
                                    tllm_stream_t stream) {
  TLLM_INJECT("launch");
  AttnParams p;
  int rc = paged_view(kv, &p.kv);
  if (rc) return rc;
  TLLM_CHECK_ARG(a, "args is NULL");
  const float *q = a->q;
  void *out = a->out, *partial = a->partial;
  const int32_t *row_seq = a->row_seq, *row_len = a->row_len;
  int32_t *counters = a->counters;
  const size_t partial_bytes = a->partial_bytes, counter_bytes = a->counter_bytes;
  const long q_row_stride = a->q_row_stride, q_head_stride = a->q_head_stride;
  const long out_plane_rows = a->out_plane_rows, out_row_stride = a->out_row_stride;
  const long out_head_stride = a->out_head_stride, keys_hint = a->keys_hint;
  const int out_dtype = a->out_dtype, rows = a->rows, n_head = a->n_head;
  const int max_len = a->max_len, window = a->window, sinks = a->sinks;
  float sm_scale = a->sm_scale;
  const int D = kv->head_dim, n_kv = kv->n_kv_head, P = kv->page_size;
  TLLM_CHECK_ARG(rows >= 0 && n_head > 0, "invalid rows %d / n_head %d", rows, n_head);
  TLLM_CHECK_ARG(n_head % n_kv == 0, "n_head (%d) must be divisible by n_kv_head (%d)",
                 n_head, n_kv);
  TLLM_CHECK_ARG(out_dtype == TLLM_F32 || out_dtype == TLLM_SPLIT || out_dtype == TLLM_BF16,
                 "out_dtype must be F32, SPLIT or BF16");
  TLLM_CHECK_ARG(out_dtype == TLLM_F32 || out_plane_rows >= rows,
                 "out_plane_rows (%ld) < rows (%d)", out_plane_rows, rows);
  TLLM_CHECK_ARG(window >= 0 && sinks >= 0, "window (%d) and sinks (%d) must be >= 0",
                 window, sinks);
  TLLM_CHECK_ARG(window > 0 || sinks == 0, "sinks (%d) need a window", sinks);
  TLLM_CHECK_ARG(max_len >= 0 && keys_hint >= 0, "max_len and keys_hint must be >= 0");
  if (rows == 0) return TLLM_OK;
  TLLM_CHECK_ARG(q && out && row_len, "NULL tensor pointer");
  TLLM_CHECK_ARG(row_seq || rows <= kv->n_seq,
                 "%d rows for a table of %d sequences (pass row_seq)", rows, kv->n_seq);
  const int esz = dtype_size(kv->kv_dtype), vec = 16 / esz;
  TLLM_CHECK_ARG(D % vec == 0 && D <= 512,
                 "head_dim %d: rows must be whole 16-byte units of at most 512 values", D);
  TLLM_CHECK_ARG((((uintptr_t)kv->k_pages | (uintptr_t)kv->v_pages) & 15) == 0 &&
                     kv->page_stride % vec == 0 && kv->head_stride % vec == 0 &&
                     kv->slot_stride % vec == 0,
                 "pages must be 16-byte aligned, with strides of whole 16 bytes");
  TLLM_CHECK_ARG(((uintptr_t)q & 15) == 0 && q_row_stride % 4 == 0 && q_head_stride % 4 == 0,
                 "q must be 16-byte aligned, with strides of whole 16 bytes");
  TLLM_CHECK_ARG(out_row_stride >= 0 && out_head_stride >= 0, "negative output stride");
  TLLM_CHECK_ARG(((uintptr_t)out & (out_dtype == TLLM_F32 ? 3 : 1)) == 0, "out misaligned");

  const int group = n_head / n_kv;
  const bool mma = mma_takes(kv, p.kv);
  const int units = D / vec;
  int lpr = 8;
  while (lpr < units && lpr < 32) lpr <<= 1;
  int nv = (units + lpr - 1) / lpr;
  if (nv == 3) nv = 4;
  const int g_max = mma ? 16 : nv * vec <= 8 ? 8 : 4;
  const int n_gsub = (group + g_max - 1) / g_max;
  const int g_even = (group + n_gsub - 1) / n_gsub;
  const int g_tile = mma ? g_even : g_even <= 2 ? g_even : g_even <= 4 ? 4 : 8;
  const int n_y = n_kv * n_gsub;
  const int tile = mma ? (D == 128 ? Tile<128>::KT : Tile<64>::KT)
                       : kGenWarps * units_deep(nv) * (32 / lpr);
  TLLM_CHECK_ARG(n_y <= 65535, "%d head groups", n_y);

  const long cap = (long)kv->table_cols * kv->page_size;
  long most = max_len > 0 && max_len < cap ? max_len : cap;
  long keys = keys_hint > 0 && keys_hint < most * rows ? keys_hint : most * rows;
  if (window > 0) {
    const long seen = (long)window + sinks;
    if (most > seen) most = seen;
    if (keys > seen * rows) keys = seen * rows;
  }
  if (mma && window > 0) {
    // whole pages, and tiles that start before the window
    most += 2 * (P > tile ? P : tile);
    if (most > cap) most = cap;
  }
  // tensor-core kernel: CTAs that share a block of rows, as many as are
  // resident at once and have work; others: splits of a row
  int chunk = 0;
  long splits = 1, ctas = 1;
  const long blocks = (rows + kRowBlock - 1) / kRowBlock;
  TLLM_CHECK_ARG(blocks <= 65535, "%d rows", rows);
  MmaKern kern = nullptr;
  size_t one, count;
  if (mma) {
    const long pairs = (long)(rows < kRowBlock ? rows : kRowBlock) * n_y;
    const long tiles = pairs * ((most + tile - 1) / tile);
    ctas = (tiles + kMinTiles - 1) / kMinTiles;
    if (ctas < pairs) ctas = pairs;
    if (ctas > (long)kMaxPerSm * sm_count()) ctas = (long)kMaxPerSm * sm_count();
    one = (size_t)blocks * 2 * g_tile * (D + 2) * sizeof(float);
    if (ctas > 1 && one * ctas > partial_bytes) ctas = partial_bytes / one;
    if (ctas < 1) ctas = 1;
    count = ctas > 1 ? blocks * ctas : 0;   // (one CTA takes all pairs whole)
  } else {
    chunk = plan_chunk(tile, rows, n_y, keys, most, 4L * sm_count());
    splits = most > 0 ? (most + chunk - 1) / chunk : 1;
    one = (size_t)rows * n_y * g_tile * (D + 2) * sizeof(float);
    if (splits > 1 && one * splits > partial_bytes) {
      splits = partial_bytes / one;
      if (splits < 1) splits = 1;
      const long per = (most + splits - 1) / splits;
      chunk = (int)((per + tile - 1) / tile * tile);
    }
    count = splits > 1 ? (size_t)rows * n_y : 0;
  }
  if (count > 0) {
    TLLM_CHECK_ARG(partial && counters, "several splits need the partial and counter buffers");
    TLLM_CHECK_ARG(((uintptr_t)partial & 15) == 0, "partial misaligned");
    TLLM_CHECK_ARG(counter_bytes >= count * sizeof(int32_t),
                   "counters hold %zu bytes, %zu needed", counter_bytes,
                   count * sizeof(int32_t));
  }

  if (mma) {
    int per_sm = 0;
    if (D == 64)
      rc = g_tile <= 8 ? mma_setup<64, 1>(&kern, &per_sm) : mma_setup<64, 2>(&kern, &per_sm);
    else
      rc = g_tile <= 8 ? mma_setup<128, 1>(&kern, &per_sm) : mma_setup<128, 2>(&kern, &per_sm);
    if (rc) return rc;
    if (ctas > (long)per_sm * sm_count()) ctas = (long)per_sm * sm_count();
  }

  if (sm_scale <= 0.f) sm_scale = 1.0f / sqrtf((float)D);
  p.q = q;
  p.row_seq = row_seq;
  p.row_len = row_len;
  const bool act = out_dtype != TLLM_F32;
  p.out = act ? nullptr : static_cast<float *>(out);
  p.out_act = act ? static_cast<uint16_t *>(out) : nullptr;
  p.out_plane = act ? (size_t)out_plane_rows * out_row_stride : 0;
  p.out_planes = out_dtype == TLLM_SPLIT ? 2 : 1;
  p.q_sr = q_row_stride;
  p.q_sh = q_head_stride;
  p.o_sr = out_row_stride;
  p.o_sh = out_head_stride;
  p.part_acc = static_cast<float *>(partial);
  const size_t slots = mma ? (size_t)blocks * ctas * 2 : (size_t)rows * n_y * splits;
  p.part_ml = p.part_acc ? p.part_acc + slots * g_tile * D : nullptr;
  p.counters = counters;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
  p.rows = rows;
  p.row0 = 0;
  p.group = group;
  p.n_gsub = n_gsub;
  p.g_tile = g_tile;
  p.n_y = n_y;
  p.chunk = chunk;
  p.max_splits = (int)splits;
  p.tile = tile;
  p.window = window;
  p.sinks = sinks;
  p.qscale = sm_scale * kLog2e;
  cudaStream_t st = resolve(stream);
  if (mma) {
    const bool slots_first = n_kv > 1 && kv->head_stride < kv->slot_stride;
    CUtensorMap mk, mv;
    rc = page_map(&mk, kv->k_pages, kv, P < tile ? P : tile, slots_first);
    if (!rc) rc = page_map(&mv, kv->v_pages, kv, P < tile ? P : tile, slots_first);
    if (rc) return rc;
    TLLM_CUDA(launch_pdl(kern, dim3((unsigned)ctas, (unsigned)blocks),
                         dim3(D == 64 ? Tile<64>::THREADS : Tile<128>::THREADS),
                         D == 64 ? Tile<64>::SMEM : Tile<128>::SMEM, st, p, mk, mv,
                         (int)slots_first));
    return TLLM_OK;
  }
  for (p.row0 = 0; p.row0 < rows; p.row0 += 65535) {   // (a grid's third axis)
    const dim3 grid((unsigned)splits, n_y, rows - p.row0 < 65535 ? rows - p.row0 : 65535);
    rc = kv->kv_dtype == TLLM_BF16 ? launch_rows_t<__nv_bfloat16>(p, lpr, nv, grid, st)
                                   : launch_rows_t<float>(p, lpr, nv, grid, st);
    if (rc) return rc;
  }
  return TLLM_OK;
}
