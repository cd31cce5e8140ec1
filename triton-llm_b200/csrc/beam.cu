// Beam search on the device, for sm_100a: the selection over beams and
// vocabulary (tllm_beam_select) and the reordering of the beams' page tables
// (tllm_beam_reorder).
//
// Selection: candidate (b, t) of a group scores s_b + (x_bt - L_b) with
// L_b = max + log sum exp(x_bt - max). Within a beam the order is that of its
// logits, so a CTA that reads a chunk of one row needs to keep only the
// chunk's max, its sum of exponentials and its k largest logits; the last CTA
// of a group to finish joins them. Each logit is read once.
//
// The k largest of a CTA's values: the k-th largest of any set of at least k
// of them is a bound that the k largest reach. With the threads' own maxima as
// that set the bound leaves few values over, which go to shared memory and are
// ranked by counting. Values carry their index in a 64-bit code, so all are
// distinct and ties are in order.
#include <cmath>

#include "mma_sync.cuh"
#include "paged.cuh"

namespace tllm {
namespace {

constexpr int kMaxK = 64;
constexpr int kMaxBeams = 32;
constexpr int kBeamWarps = 8;
constexpr int kBeamThreads = kBeamWarps * 32;
constexpr int kPerLane = 16;                          // logits of a thread
constexpr int kChunk = kBeamThreads * kPerLane;       // logits of a CTA
constexpr int kBatch = 8;                             // listed candidates of a thread
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

// A bound that at least k keys of the CTA reach, from every thread's largest
// key `best`: the k-th largest of a warp's 32 (the best of the eight warps'),
// or for k > 32 the least of the warps' ceil(k / 8)-th largest.
__device__ __forceinline__ uint64_t key_bound(uint64_t best, int k, uint64_t *s_warp) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  // bitonic sort of the warp's keys, largest first
#pragma unroll
  for (int size = 2; size <= 32; size <<= 1)
#pragma unroll
    for (int d = size >> 1; d > 0; d >>= 1) {
      const uint64_t other = __shfl_xor_sync(~0u, best, d);
      const bool larger = ((lane & d) == 0) == ((lane & size) == 0);
      best = (other > best) == larger ? other : best;
    }
  const int nth = k <= 32 ? k : (k + kBeamWarps - 1) / kBeamWarps;
  best = __shfl_sync(~0u, best, nth - 1);
  if (lane == 0) s_warp[warp] = best;
  __syncthreads();
  uint64_t bound = s_warp[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w)
    bound = (s_warp[w] > bound) == (k <= 32) ? s_warp[w] : bound;
  return bound;
}

__device__ __forceinline__ void keep(uint64_t key, uint64_t *list, int *n) {
  list[atomicAdd(n, 1)] = key;
}

// Calls put(rank, key) for the k largest of the n keys of a list in shared
// memory; all threads, after a barrier.
template <typename F>
__device__ __forceinline__ void rank_keys(const uint64_t *list, int n, int k, F put) {
  for (int i = threadIdx.x; i < n; i += kBeamThreads) {
    const uint64_t key = list[i];
    int rank = 0;
    for (int j = 0; j < n; ++j) rank += list[j] > key;
    if (rank < k) put(rank, key);
  }
}

template <bool kVec>
__global__ void __launch_bounds__(kBeamThreads) beam_select_kernel(const BeamParams p) {
  griddep_launch();
  griddep_wait();
  extern __shared__ __align__(16) uint64_t s_list[];
  __shared__ uint64_t s_warp[kBeamWarps], s_top[kMaxK];
  __shared__ float s_m[kBeamWarps], s_s[kBeamWarps];
  __shared__ int s_n, s_last;
  __shared__ float s_base[kMaxBeams], s_lse[kMaxBeams];
  const int chunk = blockIdx.x, row = blockIdx.y, group = row / p.beams;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = p.k;
  if (tid == 0) s_n = 0;

  if (!(p.done && p.done[row])) {
    const float *x = p.logits + (size_t)row * p.ld;
    const int t0 = chunk * kChunk;
    // value i of this thread: token t0 + index(i), ascending in i
    auto index = [&](int i) {
      return kVec ? (i >> 2) * 4 * kBeamThreads + 4 * tid + (i & 3) : i * kBeamThreads + tid;
    };
    const int left = p.vocab - t0;
    float v[kPerLane];
    bool nan = false;
    if constexpr (kVec) {
#pragma unroll
      for (int i = 0; i < kPerLane; i += 4) {
        const int at = index(i);
        float4 f = make_float4(-INFINITY, -INFINITY, -INFINITY, -INFINITY);
        if (at + 3 < left) {
          f = __ldcs(reinterpret_cast<const float4 *>(x + t0 + at));
        } else {
          if (at < left) f.x = x[t0 + at];
          if (at + 1 < left) f.y = x[t0 + at + 1];
          if (at + 2 < left) f.z = x[t0 + at + 2];
        }
        v[i] = f.x;
        v[i + 1] = f.y;
        v[i + 2] = f.z;
        v[i + 3] = f.w;
      }
    } else {
#pragma unroll
      for (int i = 0; i < kPerLane; ++i)
        v[i] = index(i) < left ? __ldcs(x + t0 + index(i)) : -INFINITY;
    }
    float m = -INFINITY;
    int at = 0;      // the first largest
#pragma unroll
    for (int i = 0; i < kPerLane; ++i) {
      nan |= v[i] != v[i];
      if (v[i] > m) {
        m = v[i];
        at = index(i);
      }
    }
    if (m == -INFINITY) at = index(0);
    const uint64_t best = at < left ? rank_key(m, (uint32_t)(t0 + at)) : 0;
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
    const uint64_t bound = key_bound(best, k, s_warp);
    const float least = bound ? key_value(bound) : -INFINITY;
#pragma unroll
    for (int i = 0; i < kPerLane; ++i)
      if (v[i] >= least && index(i) < left) {
        const uint64_t key = rank_key(v[i], (uint32_t)(t0 + index(i)));
        if (key >= bound) keep(key, s_list, &s_n);
      }
    __syncthreads();
    uint64_t *list = p.lists + ((size_t)row * p.chunks + chunk) * k;
    const int n = s_n;
    rank_keys(s_list, n, k, [&](int rank, uint64_t key) { list[rank] = key; });
    for (int i = n + tid; i < k; i += kBeamThreads) list[i] = 0;   // a short last chunk
    if (tid == 0) {
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
  __threadfence();
  __syncthreads();
  if (tid == 0) {
    int *ctr = p.counters + group;
    s_last = atomicAdd(ctr, 1) == p.chunks * p.beams - 1;
    if (s_last) *ctr = 0;
    s_n = 0;
  }
  __syncthreads();
  if (!s_last) return;
  __threadfence();

  // ---- the last CTA of the group: the rows' logsumexp, then the k best
  for (int b = warp; b < p.beams; b += kBeamWarps) {
    const int r = group * p.beams + b;
    float mm = -INFINITY, ss = 0.f;
    if (!(p.done && p.done[r])) {
      const float2 *stats = p.stats + (size_t)r * p.chunks;
      const float2 own = lane < p.chunks ? __ldcg(stats + lane) : make_float2(-INFINITY, 0.f);
      bool bad = own.x != own.x;
      mm = own.x;
      for (int c = lane + 32; c < p.chunks; c += 32) {
        const float m = __ldcg(stats + c).x;
        bad |= m != m;
        mm = fmaxf(mm, m);
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
      if (__any_sync(~0u, bad)) mm = NAN;
      if (own.x != -INFINITY) ss = own.y * expf(own.x - mm);
      for (int c = lane + 32; c < p.chunks; c += 32) {
        const float2 st = __ldcg(stats + c);
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
  // candidates in batches of kBatch per thread beside the best of those before
  const int per = p.chunks * k, n = p.beams * per;
  int kept = 0;
  for (int i0 = 0; i0 < n; i0 += kBatch * kBeamThreads) {
    uint64_t key[kBatch], best = tid < kept ? s_top[tid] : 0;
    const uint64_t old = best;
    // (the loads of a batch are in flight together)
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kBeamThreads + tid;
      key[j] = i < n ? __ldcg(&p.lists[(size_t)group * n + i]) : 0;
    }
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kBeamThreads + tid;
      uint64_t made = 0;
      if (i < n) {
        const int b = i / per, c = i - b * per;
        const float base = s_base[b], lse = s_lse[b];
        float score = -INFINITY;
        uint32_t token = c;
        bool is = true;
        if (p.done && p.done[group * p.beams + b]) {
          // the pad token, then others at -inf in order
          is = c < k;
          token = c == 0 ? p.pad : (c - 1 < p.pad ? c - 1 : c);
          if (c == 0) score = base;
        } else if (!(fabsf(lse) < INFINITY) || !(fabsf(base) < INFINITY)) {
          is = c < k;   // the beam has no finite candidate
        } else {
          is = key[j] != 0;
          token = key_index(key[j]);
          score = base + (key_value(key[j]) - lse);
        }
        if (!(score == score)) score = -INFINITY;
        if (is) made = rank_key(score, (uint32_t)b * p.vocab + token);
      }
      key[j] = made;
      best = made > best ? made : best;
    }
    const uint64_t bound = key_bound(best, k, s_warp);
    if (old && old >= bound) keep(old, s_list, &s_n);
#pragma unroll
    for (int j = 0; j < kBatch; ++j)
      if (key[j] && key[j] >= bound) keep(key[j], s_list, &s_n);
    __syncthreads();
    const int found = s_n;
    rank_keys(s_list, found, k, [&](int rank, uint64_t code) { s_top[rank] = code; });
    kept = min(found, k);
    __syncthreads();
    if (tid == 0) s_n = 0;
    __syncthreads();
  }
  if (tid < k) {
    const uint32_t at = key_index(s_top[tid]);
    p.out_scores[(size_t)group * k + tid] = key_value(s_top[tid]);
    p.out_parents[(size_t)group * k + tid] = at / p.vocab;
    p.out_tokens[(size_t)group * k + tid] = at % p.vocab;
  }
}

// Keys that can reach the bound in the first pass (up to k threads of a warp
// have a maximum that does, for k <= 32) and in a batch of the second.
int list_size(int k) {
  const int first = k <= 32 && k * kBeamWarps * kPerLane < kChunk ? k * kBeamWarps * kPerLane
                                                                   : kChunk;
  const int batch = kBatch * kBeamThreads + kMaxK;
  return first > batch ? first : batch;
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
  const size_t smem = list_size(k) * sizeof(uint64_t);
  const bool vec = ((uintptr_t)logits & 15) == 0 && p.ld % 4 == 0;
  TLLM_CUDA(launch_pdl(vec ? beam_select_kernel<true> : beam_select_kernel<false>,
                       dim3(p.chunks, groups * beams), dim3(kBeamThreads), smem,
                       resolve(stream), p));
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
