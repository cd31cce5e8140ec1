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
  int group, n_gsub, g_tile, n_y;   // heads per KV head, sub-groups, heads per CTA
  int chunk, max_splits, tile;
  int window, sinks;
  float qscale;          // sm_scale * log2(e)
};

// The keys of one row and this CTA's share of them.
struct RowSpan {
  int seq, len;
  int s, a;              // keys [0, s) and [a, len) are visible
  int n;                 // s + len - a
  int n_splits, begin, end;
};

__device__ __forceinline__ RowSpan row_span(const AttnParams &p, int row, int split) {
  RowSpan x;
  x.seq = p.row_seq ? p.row_seq[row] : row;
  x.len = p.row_len[row];
  const long cap = (long)p.kv.table_cols * p.kv.page_size;
  if (x.len > cap) {
    x.len = (int)cap;
    if (threadIdx.x == 0 && split == 0) atomicOr(p.err, DEV_ERR_LEN_CLAMPED);
  }
  if (x.seq < 0 || x.seq >= p.kv.n_seq) {
    x.len = 0;
    if (threadIdx.x == 0 && split == 0) atomicOr(p.err, DEV_ERR_PAGE);
  }
  if (x.len < 0) x.len = 0;
  x.s = p.window > 0 ? min(p.sinks, x.len) : 0;
  x.a = p.window > 0 ? max(x.len - p.window, x.s) : 0;
  x.n = x.s + x.len - x.a;
  // splits of the planned size; longer ones where the host's bound on the
  // length was too small
  int chunk = p.chunk;
  if ((long)chunk * p.max_splits < x.n) {
    chunk = (x.n + p.max_splits - 1) / p.max_splits;
    chunk = (chunk + p.tile - 1) / p.tile * p.tile;
  }
  x.n_splits = x.n > 0 ? (x.n + chunk - 1) / chunk : 1;
  x.begin = split * chunk;
  x.end = min(x.begin + chunk, x.n);
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

  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int *ctr = p.counters + (size_t)row * p.n_y + y;
    const int ticket = atomicAdd(ctr, 1);
    *s_flag = ticket == x.n_splits - 1;
    if (*s_flag) *ctr = 0;   // all other CTAs of this (row, y) took theirs
  }
  __syncthreads();
  if (!*s_flag) return;
  __threadfence();

  const size_t base = ((size_t)row * p.n_y + y) * p.max_splits;
  float *sw = smem;   // [G][max_splits] weights of the splits
  for (int g = warp; g < G; g += THREADS / 32) {
    float mx = -INFINITY;
    for (int s = lane; s < x.n_splits; s += 32)
      mx = fmaxf(mx, __ldcg(&p.part_ml[((base + s) * p.g_tile + g) * 2]));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(~0u, mx, o));
    float den = 0.f;
    for (int s = lane; s < x.n_splits; s += 32) {
      const float2 ml = __ldcg(reinterpret_cast<const float2 *>(
          &p.part_ml[((base + s) * p.g_tile + g) * 2]));
      const float f = ml.x == -INFINITY ? 0.f : fast_exp2(ml.x - mx);
      sw[g * kMaxSplits + s] = f;
      den = fmaf(ml.y, f, den);
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) den += __shfl_xor_sync(~0u, den, o);
    const float inv = den == 0.f ? 0.f : 1.f / den;
    for (int s = lane; s < x.n_splits; s += 32) sw[g * kMaxSplits + s] *= inv;
  }
  __syncthreads();
  for (int i = tid; i < G * D; i += THREADS) {
    const int g = i / D;
    float o = 0.f;
#pragma unroll 4
    for (int s = 0; s < x.n_splits; ++s)
      o = fmaf(sw[g * kMaxSplits + s], __ldcg(&p.part_acc[(base + s) * p.g_tile * D + i]), o);
    store_out(p, (size_t)row * p.o_sr + (size_t)(head0 + g) * p.o_sh + (i - g * D), o);
  }
}

// --------------------------------------------------------------------------
// Every page size, layout, cache type and head_dim: CUDA cores, loads straight
// from the pages. LPR lanes (a power of two) share a key, each holding NV
// 16-byte units of it; a warp takes KPW = U * 32 / LPR keys at a time with all
// their K and V loads in flight. Each group of LPR lanes keeps its own running
// maximum and sums over its keys, joined at the end.
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

template <typename T, int G, int NV>
__global__ void __launch_bounds__(kGenWarps * 32)
    paged_rows_kernel(const AttnParams p, const int LPR) {
  griddep_launch();
  griddep_wait();
  using UT = Unit<T>;
  constexpr int E = UT::N;
  constexpr int U = NV == 1 ? 4 : 2;
  extern __shared__ __align__(16) float smem_f[];
  __shared__ int s_flag;
  const int row = blockIdx.z, y = blockIdx.y, split = blockIdx.x;
  const RowSpan x = row_span(p, row, split);
  if (split >= x.n_splits) return;
  const int kvh = y / p.n_gsub;
  const int gofs = (y - kvh * p.n_gsub) * p.g_tile;
  const int Gn = min(p.g_tile, p.group - gofs);   // heads of this CTA
  const int head0 = kvh * p.group + gofs;
  const int D = p.kv.head_dim;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int units = D / E;
  const int rl = lane / LPR, cl = lane % LPR, rpw = 32 / LPR;
  const T *kp = static_cast<const T *>(p.kv.k);
  const T *vp = static_cast<const T *>(p.kv.v);
  const int *table = p.kv.table + (size_t)x.seq * p.kv.table_stride;

  float q[G][NV * E], acc[G][NV * E], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY;
    l[g] = 0.f;
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

  const int step = kGenWarps * U * rpw;
  bool bad = false;
  for (int i0 = x.begin + warp * U * rpw; i0 < x.end; i0 += step) {
    uint4 kr[U][NV], vr[U][NV];
    bool ok[U];
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const int i = i0 + u * rpw + rl;
      ok[u] = i < x.end;
      int page = 0, slot = 0;
      if (ok[u]) {
        const int pos = i < x.s ? i : i - x.s + x.a;
        const int col = p.kv.column(pos);
        slot = pos - col * p.kv.page_size;
        page = table[col];
        if (page < 0 || page >= p.kv.n_pages) {
          ok[u] = false;
          bad = true;
        }
      }
      const size_t at = ok[u] ? p.kv.offset(page, kvh, slot) : 0;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        const int c = cl + v * LPR;
        kr[u][v] = vr[u][v] = make_uint4(0, 0, 0, 0);
        if (ok[u] && c < units) {
          kr[u][v] = ld_stream(kp + at + c * E);
          vr[u][v] = ld_stream(vp + at + c * E);
        }
      }
    }
    float sc[U][G];
#pragma unroll
    for (int u = 0; u < U; ++u) {
#pragma unroll
      for (int g = 0; g < G; ++g) sc[u][g] = 0.f;
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float f[E];
        UT::unpack(kr[u][v], f);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < E; ++e) sc[u][g] = fmaf(q[g][v * E + e], f[e], sc[u][g]);
      }
    }
    for (int o = 1; o < LPR; o <<= 1)
#pragma unroll
      for (int u = 0; u < U; ++u)
#pragma unroll
        for (int g = 0; g < G; ++g) sc[u][g] += __shfl_xor_sync(~0u, sc[u][g], o);
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float mn = m[g];
#pragma unroll
      for (int u = 0; u < U; ++u) {
        if (!ok[u]) sc[u][g] = -INFINITY;
        mn = fmaxf(mn, sc[u][g]);
      }
      const float base = mn == -INFINITY ? 0.f : mn;
      const float alpha = fast_exp2(m[g] - base);   // 0 while m is -inf
      m[g] = mn;
      l[g] *= alpha;
#pragma unroll
      for (int e = 0; e < NV * E; ++e) acc[g][e] *= alpha;
#pragma unroll
      for (int u = 0; u < U; ++u) {
        sc[u][g] = fast_exp2(sc[u][g] - base);
        l[g] += sc[u][g];
      }
    }
#pragma unroll
    for (int u = 0; u < U; ++u)
#pragma unroll
      for (int v = 0; v < NV; ++v) {
        float f[E];
        UT::unpack(vr[u][v], f);
#pragma unroll
        for (int g = 0; g < G; ++g)
#pragma unroll
          for (int e = 0; e < E; ++e)
            acc[g][v * E + e] = fmaf(sc[u][g], f[e], acc[g][v * E + e]);
      }
  }
  if (bad) atomicOr(p.err, DEV_ERR_PAGE);

  // join the groups of lanes of this warp
  for (int o = LPR; o < 32; o <<= 1)
#pragma unroll
    for (int g = 0; g < G; ++g) {
      const float mo = __shfl_xor_sync(~0u, m[g], o);
      const float mn = fmaxf(m[g], mo);
      const float base = mn == -INFINITY ? 0.f : mn;
      const float f0 = fast_exp2(m[g] - base), f1 = fast_exp2(mo - base);
      m[g] = mn;
      l[g] = l[g] * f0 + __shfl_xor_sync(~0u, l[g], o) * f1;
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
        w_m[warp * Gn + g] = m[g];
        w_l[warp * Gn + g] = l[g];
      }
    }
  }
  __syncthreads();
  finish_split<kGenWarps, kGenWarps * 32>(p, x, row, y, head0, Gn, D, split, smem_f,
                                          &s_flag);
}

// --------------------------------------------------------------------------
// Host side
// --------------------------------------------------------------------------
template <typename T, int G, int NV>
int launch_rows(const AttnParams &p, int lpr, dim3 grid, cudaStream_t st) {
  const int D = p.kv.head_dim;
  size_t smem = (size_t)kGenWarps * G * (D + 2) * sizeof(float);
  const size_t sw = (size_t)G * kMaxSplits * sizeof(float);
  if (sw > smem) smem = sw;
  auto kern = paged_rows_kernel<T, G, NV>;
  if (smem > 48 * 1024)
    TLLM_CUDA(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                   (int)smem));
  TLLM_CUDA(launch_pdl(kern, grid, dim3(kGenWarps * 32), smem, st, p, lpr));
  return TLLM_OK;
}

template <typename T, int NV>
int launch_rows_g(const AttnParams &p, int lpr, dim3 grid, cudaStream_t st) {
  if (p.g_tile == 1) return launch_rows<T, 1, NV>(p, lpr, grid, st);
  if (p.g_tile == 2) return launch_rows<T, 2, NV>(p, lpr, grid, st);
  if (p.g_tile <= 4) return launch_rows<T, 4, NV>(p, lpr, grid, st);
  if constexpr (NV * Unit<T>::N <= 8) return launch_rows<T, 8, NV>(p, lpr, grid, st);
  set_error("group tile %d not built", p.g_tile);
  return TLLM_ERR_UNSUPPORTED;
}

template <typename T>
int launch_rows_t(const AttnParams &p, int lpr, int nv, dim3 grid, cudaStream_t st) {
  if (nv == 1) return launch_rows_g<T, 1>(p, lpr, grid, st);
  if (nv == 2) return launch_rows_g<T, 2>(p, lpr, grid, st);
  if constexpr (Unit<T>::N == 4) return launch_rows_g<T, 4>(p, lpr, grid, st);
  set_error("head_dim %d not built", p.kv.head_dim);
  return TLLM_ERR_UNSUPPORTED;
}

// Keys per split, a multiple of `tile`, for `pairs` (row, head group) pairs
// of at most max_keys keys and about `keys` in all rows.
int plan_chunk(int tile, long rows, int n_y, long keys, long max_keys, long slots) {
  const long tiles = (max_keys + tile - 1) / tile;
  long c = (keys * n_y / tile + slots - 1) / slots;   // one CTA per slot
  if (rows * n_y >= slots || c > 32) c = c < 32 ? 32 : c;
  if (c < 2) c = 2;
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
  // splits per row that fill the GPU a few times over, and at least 8
  long splits = 8192 / ((long)(rows > 0 ? rows : 1) * n_kv_head);
  if (splits > kMaxSplits) splits = kMaxSplits;
  if (splits < 8) splits = 8;
  // (heads of a KV head may be padded to the next tile of 1, 2, 4 or 8)
  *partial_bytes = (size_t)rows * n_head * 2 * splits * (head_dim + 2) * sizeof(float);
  *counter_bytes = (size_t)rows * n_head * sizeof(int32_t);
  return TLLM_OK;
}

extern "C" int tllm_paged_attention(
    const tllm_paged_kv *kv, const float *q, long q_row_stride, long q_head_stride,
    const int32_t *row_seq, const int32_t *row_len, void *out, int out_dtype,
    long out_plane_rows, long out_row_stride, long out_head_stride, int rows,
    int n_head, int max_len, long keys_hint, int window, int sinks, float sm_scale,
    void *partial, size_t partial_bytes, int32_t *counters, size_t counter_bytes,
    tllm_stream_t stream) {
  TLLM_INJECT("launch");
  AttnParams p;
  int rc = paged_view(kv, &p.kv);
  if (rc) return rc;
  const int D = kv->head_dim, n_kv = kv->n_kv_head;
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
  const int units = D / vec;
  int lpr = 1;
  while (lpr < units && lpr < 32) lpr <<= 1;
  int nv = (units + lpr - 1) / lpr;
  if (nv == 3) nv = 4;
  const int g_max = nv * vec <= 8 ? 8 : 4;
  const int n_gsub = (group + g_max - 1) / g_max;
  const int g_even = (group + n_gsub - 1) / n_gsub;
  const int g_tile = g_even <= 2 ? g_even : g_even <= 4 ? 4 : 8;
  const int n_y = n_kv * n_gsub;
  const int tile = kGenWarps * (nv == 1 ? 4 : 2) * (32 / lpr);
  TLLM_CHECK_ARG(n_y <= 65535 && rows <= 65535, "grid too large: %d rows, %d head groups",
                 rows, n_y);

  const long cap = (long)kv->table_cols * kv->page_size;
  long most = max_len > 0 && max_len < cap ? max_len : cap;
  long keys = keys_hint > 0 && keys_hint < most * rows ? keys_hint : most * rows;
  if (window > 0) {
    const long seen = (long)window + sinks;
    if (most > seen) most = seen;
    if (keys > seen * rows) keys = seen * rows;
  }
  int chunk = plan_chunk(tile, rows, n_y, keys, most, 4L * sm_count());
  long splits = most > 0 ? (most + chunk - 1) / chunk : 1;
  const size_t one = (size_t)rows * n_y * g_tile * (D + 2) * sizeof(float);
  if (splits > 1 && one * splits > partial_bytes) {
    splits = partial_bytes / one;
    if (splits < 1) splits = 1;
    const long per = (most + splits - 1) / splits;
    chunk = (int)((per + tile - 1) / tile * tile);
  }
  if (splits > 1) {
    TLLM_CHECK_ARG(partial && counters, "several splits need the partial and counter buffers");
    TLLM_CHECK_ARG(((uintptr_t)partial & 15) == 0, "partial misaligned");
    TLLM_CHECK_ARG(counter_bytes >= (size_t)rows * n_y * sizeof(int32_t),
                   "counters hold %zu bytes, %zu needed", counter_bytes,
                   (size_t)rows * n_y * sizeof(int32_t));
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
  p.part_ml = p.part_acc ? p.part_acc + (size_t)rows * n_y * splits * g_tile * D : nullptr;
  p.counters = counters;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
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
  const dim3 grid((unsigned)splits, n_y, rows);
  cudaStream_t st = resolve(stream);
  return kv->kv_dtype == TLLM_BF16
             ? launch_rows_t<__nv_bfloat16>(p, lpr, nv, grid, st)
             : launch_rows_t<float>(p, lpr, nv, grid, st);
}
