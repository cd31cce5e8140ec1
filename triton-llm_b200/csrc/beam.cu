// Beam search on the device, for sm_100a: the selection over beams and
// vocabulary (tllm_beam_select) and the reordering of the beams' page tables
// (tllm_beam_reorder).
//
// Selection: candidate (b, t) of a group scores s_b + (x_bt - L_b) with
// L_b = max + log sum exp(x_bt - max). Within a beam the order is that of its
// logits, so a CTA that reads a chunk of one row needs to keep only the
// chunk's max, its sum of exponentials and its k largest logits; the last CTA
// of a group to finish joins them.
#include <cmath>

#include "mma_sync.cuh"
#include "paged.cuh"

namespace tllm {
namespace {

constexpr int kMaxK = 64;
constexpr int kMaxBeams = 32;
constexpr int kBeamWarps = 8;
constexpr int kPerLane = 16;
constexpr int kChunk = kBeamWarps * 32 * kPerLane;   // logits of one CTA
constexpr float kLog2e = 1.4426950408889634f;
constexpr int kMaxRows = 65535;
// the groups' tickets lie at the front of the workspace whatever its shape, so
// that one made for a larger call stays valid for a smaller one
constexpr size_t kCounterBytes = (size_t)(kMaxRows + 1) * sizeof(int);

// Order-preserving code of (value, index): larger value first, then the lower
// index. -0 and +0 are equal. Never 0.
__device__ __forceinline__ uint64_t rank_key(float v, uint32_t index) {
  uint32_t u = __float_as_uint(v + 0.f);
  u = (u >> 31) ? ~u : (u | 0x80000000u);
  return ((uint64_t)u << 32) | (uint32_t)~index;
}
__device__ __forceinline__ float key_value(uint64_t key) {
  uint32_t u = (uint32_t)(key >> 32);
  u = (u >> 31) ? (u & 0x7fffffffu) : ~u;
  return __uint_as_float(u);
}
__device__ __forceinline__ uint32_t key_index(uint64_t key) { return ~(uint32_t)key; }

__device__ __forceinline__ uint64_t warp_max(uint64_t v) {
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) {
    const uint64_t w = __shfl_xor_sync(~0u, v, o);
    v = w > v ? w : v;
  }
  return v;
}

struct BeamParams {
  const float *logits;
  long ld;
  const float *scores;
  const int *done;
  int pad, groups, beams, vocab, k, chunks;
  float *out_scores;
  int *out_parents, *out_tokens;
  int *counters;        // (groups)
  float2 *stats;        // (rows, chunks): max, sum
  uint64_t *lists;      // (rows, chunks, k)
};

// The k largest of n keys in shared memory, in order, into out[0..k); called
// by one warp. n >= k. Destroys keys.
__device__ void warp_select(uint64_t *keys, int n, int k, uint64_t *out) {
  const int lane = threadIdx.x & 31;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    int at = -1;
    for (int i = lane; i < n; i += 32)
      if (keys[i] > best) {
        best = keys[i];
        at = i;
      }
    const uint64_t top = warp_max(best);
    if (lane == 0) out[j] = top;
    if (at >= 0 && best == top) keys[at] = 0;
    __syncwarp();
  }
}

__global__ void __launch_bounds__(kBeamWarps * 32) beam_select_kernel(const BeamParams p) {
  griddep_launch();
  griddep_wait();
  extern __shared__ __align__(16) uint64_t smem_k[];
  __shared__ float s_m[kBeamWarps], s_s[kBeamWarps];
  __shared__ int s_last;
  __shared__ float s_base[kMaxBeams], s_lse[kMaxBeams];
  const int chunk = blockIdx.x, row = blockIdx.y, group = row / p.beams;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = p.k;

  if (!(p.done && p.done[row])) {
    const float *x = p.logits + (size_t)row * p.ld;
    const int first = chunk * kChunk + warp * 32 * kPerLane + lane;
    float v[kPerLane];
    bool nan = false;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      const int t = first + i * 32;
      v[i] = t < p.vocab ? __ldcs(x + t) : -INFINITY;
      nan |= v[i] != v[i];
    }
    float m = -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) m = fmaxf(m, v[i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(~0u, m, o));
    if (__any_sync(~0u, nan)) m = NAN;
    float s = 0.f;
    if (m != -INFINITY)
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) s += fast_exp2((v[i] - m) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) {
      s_m[warp] = m;
      s_s[warp] = s;
    }
    // this warp's k largest
    uint32_t taken = 0;
    for (int j = 0; j < k; ++j) {
      uint64_t best = 0;
      int at = -1;
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) {
        const int t = first + i * 32;
        const uint64_t key = rank_key(v[i], (uint32_t)t);
        if (t < p.vocab && !(taken >> i & 1) && key > best) {
          best = key;
          at = i;
        }
      }
      const uint64_t top = warp_max(best);
      if (at >= 0 && best == top) taken |= 1u << at;
      if (lane == 0) smem_k[warp * k + j] = top;
    }
    __syncthreads();
    if (warp == 0) {
      warp_select(smem_k, kBeamWarps * k, k,
                  p.lists + ((size_t)row * p.chunks + chunk) * k);
      if (lane == 0) {
        float mm = -INFINITY, ss = 0.f;
        bool bad = false;
        for (int w = 0; w < kBeamWarps; ++w) {
          bad |= s_m[w] != s_m[w];
          mm = fmaxf(mm, s_m[w]);
        }
        for (int w = 0; w < kBeamWarps; ++w)
          if (s_m[w] != -INFINITY) ss += s_s[w] * fast_exp2((s_m[w] - mm) * kLog2e);
        p.stats[(size_t)row * p.chunks + chunk] = make_float2(bad ? NAN : mm, ss);
      }
    }
  }
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int *ctr = p.counters + group;
    s_last = atomicAdd(ctr, 1) == p.chunks * p.beams - 1;
    if (s_last) *ctr = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();

  // ---- the last CTA of the group: rows' logsumexp, then the k best
  for (int b = warp; b < p.beams; b += kBeamWarps) {
    const int r = group * p.beams + b;
    float mm = -INFINITY, ss = 0.f;
    if (!(p.done && p.done[r])) {
      bool bad = false;
      for (int c = lane; c < p.chunks; c += 32) {
        const float m = __ldcg(&p.stats[(size_t)r * p.chunks + c]).x;
        bad |= m != m;
        mm = fmaxf(mm, m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
      if (__any_sync(~0u, bad)) mm = NAN;
      for (int c = lane; c < p.chunks; c += 32) {
        const float2 st = __ldcg(&p.stats[(size_t)r * p.chunks + c]);
        if (st.x != -INFINITY) ss += st.y * expf(st.x - mm);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    }
    if (lane == 0) {
      s_base[b] = p.scores[r];
      s_lse[b] = mm + logf(ss);
    }
  }
  __syncthreads();
  const int per = p.chunks * k, n = p.beams * per;
  uint64_t mine[1];
  (void)mine;
  // candidates are visited k times; each round takes the best one left,
  // which is the best below the last one taken (keys are distinct)
  uint64_t last = ~0ull;
  uint64_t *s_best = smem_k;
  for (int j = 0; j < k; ++j) {
    uint64_t best = 0;
    for (int i = tid; i < n; i += kBeamWarps * 32) {
      const int b = i / per, c = i - b * per;
      const int r = group * p.beams + b;
      const float base = s_base[b];
      float score;
      uint32_t token;
      if (p.done && p.done[r]) {
        if (c >= k) continue;
        // the pad token first, then others at -inf in order
        token = c == 0 ? p.pad : (c - 1 < p.pad ? c - 1 : c);
        score = c == 0 ? base : -INFINITY;
      } else {
        const float lse = s_lse[b];
        const bool dead = !(fabsf(lse) < INFINITY) || !(fabsf(base) < INFINITY);
        if (dead) {
          if (c >= k) continue;
          token = c;
          score = -INFINITY;
        } else {
          const uint64_t key = __ldcg(&p.lists[(size_t)r * per + c]);
          if (key == 0) continue;
          token = key_index(key);
          score = base + (key_value(key) - lse);
        }
      }
      if (!(score == score)) score = -INFINITY;
      const uint64_t key = rank_key(score, (uint32_t)b * p.vocab + token);
      if (key < last && key > best) best = key;
    }
    best = warp_max(best);
    __syncthreads();
    if (lane == 0) s_best[warp] = best;
    __syncthreads();
    best = 0;
#pragma unroll
    for (int w = 0; w < kBeamWarps; ++w) best = s_best[w] > best ? s_best[w] : best;
    last = best;
    if (tid == 0) {
      const uint32_t index = key_index(best);
      p.out_scores[(size_t)group * k + j] = key_value(best);
      p.out_parents[(size_t)group * k + j] = index / p.vocab;
      p.out_tokens[(size_t)group * k + j] = index % p.vocab;
    }
  }
}

// --------------------------------------------------------------------------
// Reordering: one CTA per group, one thread per table column.
// --------------------------------------------------------------------------
struct ReorderParams {
  const int *parents, *lens, *table_in;
  int *table_out;
  int beams, cols, page_size;
  int *copy_src, *copy_dst, *copy_fill;
  int *err;
};

__global__ void beam_reorder_kernel(const ReorderParams p) {
  griddep_launch();
  griddep_wait();
  __shared__ int s_parent[kMaxBeams], s_target[kMaxBeams], s_ok;
  const int g = blockIdx.x, W = p.beams, tid = threadIdx.x;
  const size_t row0 = (size_t)g * W;
  const int len = p.lens[row0];
  const int c = len / p.page_size, f = len - c * p.page_size;
  if (tid < 32) {
    const int up = tid < W ? p.parents[row0 + tid] : 0;
    const bool good = up >= 0 && up < W && len >= 0 && (f > 0 ? c < p.cols : c <= p.cols);
    const bool ok = __all_sync(~0u, good);
    // first children keep their parent's page, in order the others take those
    // of the beams without a child
    uint32_t parents_seen = 0;   // beams that have a child
    for (int i = 0; i < W; ++i) parents_seen |= 1u << (__shfl_sync(~0u, up, i) & 31);
    bool first = tid < W;
    for (int i = 0; i < W; ++i) {
      const int other = __shfl_sync(~0u, up, i);
      if (i < tid && other == up) first = false;
    }
    const uint32_t extra = __ballot_sync(~0u, tid < W && !first);
    const uint32_t all = W == 32 ? ~0u : (1u << W) - 1;
    const uint32_t ends = all & ~parents_seen;
    int target = up;
    if (tid < W && !first) {
      const int nth = __popc(extra & ((1u << tid) - 1));
      target = __fns(ends, 0, nth + 1);
    }
    if (tid < W) {
      s_parent[tid] = ok ? up : tid;
      s_target[tid] = ok ? target : tid;
      int src = -1, dst = -1;
      if (ok && f > 0) {
        src = p.table_in[(row0 + up) * p.cols + c];
        dst = p.table_in[(row0 + target) * p.cols + c];
      }
      p.copy_src[row0 + tid] = src;
      p.copy_dst[row0 + tid] = dst;
      p.copy_fill[row0 + tid] = ok && f > 0 ? f : 0;
    }
    if (tid == 0) {
      s_ok = ok;
      if (!ok) atomicOr(p.err, DEV_ERR_PAGE);
    }
  }
  __syncthreads();
  const bool ok = s_ok;
  for (int j = tid; j < p.cols; j += blockDim.x) {
    if (p.table_out == p.table_in && (!ok || j > c || (j == c && f == 0))) continue;
    int v[kMaxBeams];
    for (int i = 0; i < W; ++i) {
      const int from = !ok ? i : j < c ? s_parent[i] : j == c && f > 0 ? s_target[i] : i;
      v[i] = p.table_in[(row0 + from) * p.cols + j];
    }
    for (int i = 0; i < W; ++i) p.table_out[(row0 + i) * p.cols + j] = v[i];
  }
}

size_t align256(size_t n) { return (n + 255) / 256 * 256; }

}  // namespace
}  // namespace tllm

using namespace tllm;

extern "C" int tllm_beam_workspace(int groups, int beams, int vocab, int k, size_t *bytes) {
  TLLM_CHECK_ARG(bytes, "NULL output pointer");
  TLLM_CHECK_ARG(groups >= 0 && beams >= 1 && beams <= kMaxBeams,
                 "groups (%d) must be >= 0 and beams (%d) in [1, %d]", groups, beams, kMaxBeams);
  TLLM_CHECK_ARG(vocab >= 1 && vocab < (1 << 27), "vocab (%d) must be in [1, 2^27)", vocab);
  TLLM_CHECK_ARG(k >= 1 && k <= kMaxK && k <= vocab, "k (%d) must be in [1, %d] and <= vocab (%d)",
                 k, kMaxK, vocab);
  const size_t rows = (size_t)groups * beams, chunks = (vocab + kChunk - 1) / kChunk;
  *bytes = kCounterBytes + align256(rows * chunks * sizeof(float2)) +
           rows * chunks * k * sizeof(uint64_t);
  return TLLM_OK;
}

extern "C" int tllm_beam_select(const float *logits, long ld, const float *scores,
                                const int32_t *done, int pad_token, int groups, int beams,
                                int vocab, int k, float *out_scores, int32_t *out_parents,
                                int32_t *out_tokens, void *workspace,
                                size_t workspace_bytes, tllm_stream_t stream) {
  TLLM_INJECT("launch");
  size_t need = 0;
  int rc = tllm_beam_workspace(groups, beams, vocab, k, &need);
  if (rc) return rc;
  TLLM_CHECK_ARG(ld == 0 || ld >= vocab, "row stride %ld < vocab = %d", ld, vocab);
  TLLM_CHECK_ARG(!done || (pad_token >= 0 && pad_token < vocab),
                 "pad_token (%d) outside the vocabulary (%d)", pad_token, vocab);
  TLLM_CHECK_ARG((long)groups * beams <= kMaxRows, "more than %d rows", kMaxRows);
  if (groups == 0) return TLLM_OK;
  TLLM_CHECK_ARG(logits && scores && out_scores && out_parents && out_tokens, "NULL pointer");
  TLLM_CHECK_ARG(workspace && workspace_bytes >= need && ((uintptr_t)workspace & 255) == 0,
                 "workspace of %zu bytes, %zu needed (256-byte aligned)", workspace_bytes, need);
  BeamParams p;
  p.logits = logits;
  p.ld = ld > 0 ? ld : vocab;
  p.scores = scores;
  p.done = done;
  p.pad = pad_token;
  p.groups = groups;
  p.beams = beams;
  p.vocab = vocab;
  p.k = k;
  p.chunks = (vocab + kChunk - 1) / kChunk;
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  char *w = static_cast<char *>(workspace);
  p.counters = reinterpret_cast<int *>(w);
  w += kCounterBytes;
  p.stats = reinterpret_cast<float2 *>(w);
  w += align256((size_t)groups * beams * p.chunks * sizeof(float2));
  p.lists = reinterpret_cast<uint64_t *>(w);
  const size_t smem = (size_t)kBeamWarps * k * sizeof(uint64_t);
  TLLM_CUDA(launch_pdl(beam_select_kernel, dim3(p.chunks, groups * beams),
                       dim3(kBeamWarps * 32), smem, resolve(stream), p));
  return TLLM_OK;
}

extern "C" int tllm_beam_reorder(const int32_t *parents, const int32_t *lens,
                                 const int32_t *table_in, int32_t *table_out, int groups,
                                 int beams, int table_cols, int page_size,
                                 int32_t *copy_src, int32_t *copy_dst, int32_t *copy_fill,
                                 tllm_stream_t stream) {
  TLLM_INJECT("launch");
  TLLM_CHECK_ARG(groups >= 0 && beams >= 1 && beams <= kMaxBeams,
                 "groups (%d) must be >= 0 and beams (%d) in [1, %d]", groups, beams, kMaxBeams);
  TLLM_CHECK_ARG(table_cols >= 0 && page_size >= 1, "invalid table: %d columns of %d slots",
                 table_cols, page_size);
  if (groups == 0) return TLLM_OK;
  TLLM_CHECK_ARG(parents && lens && copy_src && copy_dst && copy_fill &&
                     (table_cols == 0 || (table_in && table_out)),
                 "NULL pointer");
  ReorderParams p;
  p.parents = parents;
  p.lens = lens;
  p.table_in = table_in;
  p.table_out = table_out;
  p.beams = beams;
  p.cols = table_cols;
  p.page_size = page_size;
  p.copy_src = copy_src;
  p.copy_dst = copy_dst;
  p.copy_fill = copy_fill;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
  const int threads = table_cols >= 256 ? 256 : (table_cols + 31) / 32 * 32 > 32
                                                    ? (table_cols + 31) / 32 * 32
                                                    : 32;
  TLLM_CUDA(launch_pdl(beam_reorder_kernel, dim3(groups), dim3(threads), 0,
                       resolve(stream), p));
  return TLLM_OK;
}
