// Beam search on the device, for sm_100a: the selection over beams and
// vocabulary (tllm_beam_select) and the reordering of the beams' page tables
// (tllm_beam_reorder).
//
// Selection: candidate (b, t) of a group scores
//   s_b + ((x_bt - m_b) - log sum_t exp(x_bt - m_b)),   m_b = max_t x_bt,
// where every logit is taken less the maximum before it is scaled, multiplied or
// rounded: m_b itself may be of any size (a mask of the type's lowest value,
// 1000 with its steps of 2^-14). Within a beam the order is that of its
// logits, so a CTA that reads a part of one row needs to keep only the part's
// max, its sum of exponentials and its k largest logits; the last CTA of a
// group to finish joins them. Each logit is read once.
//
// Values carry their index in a 64-bit code, so all are distinct and ties are
// in order. Unequal logits may round to equal scores (a beam at -1000 collapses
// logits 6e-5 apart), so the group's order is by score, beam and then the same
// code of logit and token: by score alone, the lower token would win among the
// listed ones and the larger logit at the end of a part's list.
//
// A thread reads its share of the part with the next 16 values on the
// way, keeps the maximum and the sum, and remembers its two best steps (of 16
// values) and the largest value outside them. The k-th largest of the threads'
// own maxima is a key that the part's k largest reach; the few threads that
// reach it read those steps again (from L2) and list what does. Bound by HBM
// while it reads (9 us of 26 for 16 x 8 beams over 128256 tokens, 66 MB), then
// by the latency of a few dependent passes; a list of candidates kept up during
// the reading took 31 us, k rounds of maxima over all values 121.
#include <cmath>

#include "mma_sync.cuh"
#include "paged.cuh"

namespace tllm {
namespace {

constexpr int kMaxK = 64;
constexpr int kMaxBeams = 32;
constexpr int kBeamWarps = 8;
constexpr int kBeamThreads = kBeamWarps * 32;
constexpr int kPerLane = 16;                          // logits of a lane in one step
constexpr int kStep = kBeamThreads * kPerLane;        // logits of a CTA in one step
constexpr int kCtasPerSm = 4;                         // parts are cut for so many
constexpr int kBatch = 4;                             // listed candidates of a thread
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
  int pad, groups, beams, vocab, k;
  int chunks, chunk;    // parts of a row, their logits (whole steps)
  float *out_scores;
  int *out_parents, *out_tokens, *out_done;
  int eos;
  int *counters;        // (groups)
  float2 *stats;        // (rows, chunks): max, sum of exponentials
  uint64_t *lists;      // (rows, chunks, k)
};

// A key that at least nth lanes' `best` reach: nth rounds of warp maxima over
// the values; equal values give up their lowest lane first, and the bound
// carries the highest index among the lanes taken with its value. 0 if fewer
// lanes have a key.
__device__ __forceinline__ uint64_t warp_bound(uint64_t best, int nth) {
  const int lane = threadIdx.x & 31;
  const uint32_t value = (uint32_t)(best >> 32);
  uint32_t left = value, top = 0;
  bool taken = false;
  for (int i = 0; i < nth; ++i) {
    top = __reduce_max_sync(~0u, left);
    if (top == 0) return 0;
    const int first = __ffs(__ballot_sync(~0u, left == top)) - 1;
    if (lane == first) {
      taken = true;
      left = 0;
    }
  }
  const uint32_t index =
      __reduce_max_sync(~0u, taken && value == top ? key_index(best) : 0u);
  return ((uint64_t)top << 32) | (uint32_t)~index;
}

// A bound that at least k keys of the CTA reach, from every thread's largest:
// for k <= 32 the best of the warps' k-th largest, beyond that the least of
// their ceil(k / 8)-th largest.
__device__ __forceinline__ uint64_t block_bound(uint64_t best, int k, uint64_t *s_warp) {
  const uint64_t mine = warp_bound(best, k <= 32 ? k : (k + kBeamWarps - 1) / kBeamWarps);
  if ((threadIdx.x & 31) == 0) s_warp[threadIdx.x >> 5] = mine;
  __syncthreads();
  uint64_t bound = s_warp[0];
#pragma unroll
  for (int w = 1; w < kBeamWarps; ++w)
    bound = (s_warp[w] > bound) == (k <= 32) ? s_warp[w] : bound;
  return bound;
}

// The k largest of the warp's 32 keys (all of them for k >= 16) into out, where
// 32 places are this warp's; returns their number.
__device__ __forceinline__ int warp_largest(uint64_t key, int k, uint64_t *out) {
  const int lane = threadIdx.x & 31;
  if (k >= 16) {
    out[lane] = key;
    return 32;
  }
  uint32_t left = (uint32_t)(key >> 32);
  for (int i = 0; i < k; ++i) {
    const uint32_t top = __reduce_max_sync(~0u, left);
    if (top == 0) {   // no keys left
      out[i] = 0;
      continue;
    }
    // equal values: the lower index first
    const uint32_t tie = left == top ? (uint32_t)key : 0;
    const uint32_t low = __reduce_max_sync(~0u, tie);
    if (left == top && tie == low) {
      out[i] = key;
      left = 0;
    }
  }
  return k;
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
__global__ void __launch_bounds__(kBeamThreads, kCtasPerSm)
    beam_select_kernel(const BeamParams p) {
  griddep_launch();
  griddep_wait();
  constexpr int kKeys = kBatch * kBeamThreads + kMaxK;
  static_assert(kBeamWarps * 32 <= kKeys, "the threads' keys use the same memory");
  __shared__ uint64_t s_list[kKeys], s_logit[kKeys];
  __shared__ uint64_t s_warp[kBeamWarps], s_top[kMaxK], s_token[kMaxK];
  __shared__ unsigned long long s_bound;
  __shared__ float s_m[kBeamWarps], s_s[kBeamWarps];
  __shared__ int s_n, s_last;
  __shared__ float s_base[kMaxBeams], s_max[kMaxBeams], s_log[kMaxBeams];
  __shared__ int s_done[kMaxBeams];
  const int chunk = blockIdx.x, row = blockIdx.y, group = row / p.beams;
  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int k = p.k;

  if (!(p.done && p.done[row])) {
    const float *x = p.logits + (size_t)row * p.ld;
    const int begin = chunk * p.chunk + warp * 32 * kPerLane;
    const int end = min(p.vocab, (chunk + 1) * p.chunk);
    // value i of this lane in a step: token t0 + at(i), ascending in i
    auto at = [&](int i) {
      return kVec ? (i >> 2) * 128 + 4 * lane + (i & 3) : i * 32 + lane;
    };
    auto load = [&](int t0, float (&v)[kPerLane]) {
      if (kVec && t0 + 32 * kPerLane <= end) {
#pragma unroll
        for (int i = 0; i < kPerLane; i += 4) {
          const float4 f = __ldg(reinterpret_cast<const float4 *>(x + t0 + at(i)));
          v[i] = f.x;
          v[i + 1] = f.y;
          v[i + 2] = f.z;
          v[i + 3] = f.w;
        }
      } else {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i)
          v[i] = t0 + at(i) < end ? __ldg(x + t0 + at(i)) : -INFINITY;
      }
    };
    // maxima of the best step, the second and the others
    float m = -INFINITY, m2 = -INFINITY, other = -INFINITY;
    float s = 0.f;                            // sum of 2^((v - m) log2 e)
    int best = begin, second = begin;
    auto sum_up = [&](const float (&v)[kPerLane], int t0) {
      float top = v[0];
#pragma unroll
      for (int i = 1; i < kPerLane; ++i) top = fmaxf(top, v[i]);
      // (a NaN anywhere, or +inf, makes the sum NaN; -inf alone leaves it 0)
      const float mn = fmaxf(m, top), base = mn == -INFINITY ? 0.f : mn;
      float add[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
      for (int i = 0; i < kPerLane; ++i) add[i & 3] += fast_exp2((v[i] - base) * kLog2e);
      // (a factor of exactly 1 while the maximum stays: a rounding of it would
      // compound over the steps)
      if (mn != m) s *= fast_exp2((m - mn) * kLog2e);
      s += (add[0] + add[1]) + (add[2] + add[3]);
      if (t0 == begin) {
        m = top;
        return;
      }
      const bool up = top > m, up2 = top > m2 || (second == begin && best == begin);
      other = fmaxf(other, up || up2 ? m2 : top);
      m2 = up ? m : up2 ? top : m2;
      second = up ? best : up2 ? t0 : second;
      m = up ? top : m;
      best = up ? t0 : best;
    };
    // two steps' values are in registers, one in use and one on the way
    {
      float va[kPerLane], vb[kPerLane];
      int t0 = begin;
      load(t0, va);
      while (t0 < end) {
        load(t0 + kStep, vb);
        sum_up(va, t0);
        t0 += kStep;
        if (t0 >= end) break;
        load(t0 + kStep, va);
        sum_up(vb, t0);
        t0 += kStep;
      }
    }
    // this thread's largest key
    float v[kPerLane];
    load(best, v);
    int first = kPerLane;
#pragma unroll
    for (int i = kPerLane - 1; i >= 0; --i)
      if (v[i] == m || (m == -INFINITY && i == 0)) first = i;
    const bool any = first < kPerLane && best + at(first) < end;
    const uint64_t mine = any ? rank_key(m, (uint32_t)(best + at(first))) : 0;
    float mm = m;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
    s = m == -INFINITY ? s : s * fast_exp2((m - mm) * kLog2e);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) s += __shfl_xor_sync(~0u, s, o);
    if (lane == 0) {
      s_m[warp] = mm;
      s_s[warp] = s;
    }
    // the k-th largest of all threads' keys (0: fewer than k have one)
    const int per = warp_largest(mine, k, s_list + warp * 32);
    if (tid == 0) {
      s_bound = 0;
      s_n = 0;
    }
    __syncthreads();
    // (four lanes a key, each against two warps' keys)
    for (int w = warp; w < per; w += kBeamWarps) {
      const uint64_t key = s_list[(lane >> 2) * 32 + w];
      int rank = 0;
#pragma unroll 4
      for (int q = 0; q < per; ++q) {
        rank += s_list[(lane & 3) * 64 + q] > key;
        rank += s_list[(lane & 3) * 64 + 32 + q] > key;
      }
      rank += __shfl_xor_sync(~0u, rank, 1);
      rank += __shfl_xor_sync(~0u, rank, 2);
      if (rank == k - 1 && key) s_bound = key;
    }
    __syncthreads();
    const uint64_t bound = s_bound;
    const float least = bound ? key_value(bound) : -INFINITY;
    // list the values that reach it; a thread's other steps only if their
    // largest value may (equal ones do not where the step starts past the
    // bound's index)
    if (mine >= bound && any) {
      auto list = [&](int t0) {
#pragma unroll
        for (int i = 0; i < kPerLane; ++i) {
          if (!(v[i] >= least) || t0 + at(i) >= end) continue;
          const uint64_t key = rank_key(v[i], (uint32_t)(t0 + at(i)));
          if (key < bound) continue;
          const int to = atomicAdd(&s_n, 1);
          if (to < kKeys) s_list[to] = key;
        }
      };
      auto may = [&](float top, int t) {
        return !bound || top > least || (top == least && t <= (int)key_index(bound));
      };
      list(best);
      if (second != best && may(m2, second)) {
        load(second, v);
        list(second);
      }
      if (may(other, begin)) {
#pragma unroll 1
        for (int t = begin; t < end; t += kStep) {
          if (t == best || t == second) continue;
          if (!may(other, t)) break;
          load(t, v);
          list(t);
        }
      }
    }
    __syncthreads();
    uint64_t *out = p.lists + ((size_t)row * p.chunks + chunk) * k;
    const int n = s_n;
    if (n <= kKeys) {
      rank_keys(s_list, n, k, [&](int rank, uint64_t key) { out[rank] = key; });
      for (int i = n + tid; i < k; i += kBeamThreads) out[i] = 0;   // a short last part
    } else {
      // more values above the bound than the list holds (they all lie in the
      // same threads' shares): k rounds of the largest below the last
      uint64_t last = ~0ull;
      for (int j = 0; j < k; ++j) {
        uint64_t top = 0;
        for (int t = begin; t < end; t += kStep) {
          load(t, v);
#pragma unroll
          for (int i = 0; i < kPerLane; ++i) {
            const uint64_t key = t + at(i) < end ? rank_key(v[i], (uint32_t)(t + at(i))) : 0;
            if (v[i] == v[i] && key < last && key > top) top = key;
          }
        }
        __syncthreads();
        warp_largest(top, 1, s_warp + warp);
        __syncthreads();
        last = 0;
#pragma unroll
        for (int w = 0; w < kBeamWarps; ++w) last = s_warp[w] > last ? s_warp[w] : last;
        if (tid == 0) out[j] = last;
      }
    }
    if (tid == 0) {
      float all = -INFINITY, ss = 0.f;
#pragma unroll
      for (int w = 0; w < kBeamWarps; ++w) all = fmaxf(all, s_m[w]);
#pragma unroll
      for (int w = 0; w < kBeamWarps; ++w)
        ss += s_m[w] == -INFINITY ? s_s[w] : s_s[w] * fast_exp2((s_m[w] - all) * kLog2e);
      p.stats[(size_t)row * p.chunks + chunk] = make_float2(all, ss);
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

  // ---- the last CTA of the group: the rows' logsumexp, then the k best.
  // The first batch of candidates is loaded beside the statistics.
  const int per = p.chunks * k, n = p.beams * per;
  const uint64_t *lists = p.lists + (size_t)group * n;
  uint64_t key[kBatch];
  auto load = [&](int i0) {
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kBeamThreads + tid;
      key[j] = i < n ? __ldcg(lists + i) : 0;
    }
  };
  load(0);
  for (int b = warp; b < p.beams; b += kBeamWarps) {
    const int r = group * p.beams + b;
    const bool done = p.done && p.done[r];
    const float base = p.scores[r];
    const float2 *stats = p.stats + (size_t)r * p.chunks;
    const float2 own = !done && lane < p.chunks ? __ldcg(stats + lane)
                                                : make_float2(-INFINITY, 0.f);
    float mm = own.x, ss = 0.f;
    if (!done)
      for (int c = lane + 32; c < p.chunks; c += 32) mm = fmaxf(mm, __ldcg(stats + c).x);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mm = fmaxf(mm, __shfl_xor_sync(~0u, mm, o));
    auto add = [&](float2 st) { ss += st.x == -INFINITY ? st.y : st.y * expf(st.x - mm); };
    add(own);
    if (!done)
      for (int c = lane + 32; c < p.chunks; c += 32) add(__ldcg(stats + c));
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ss += __shfl_xor_sync(~0u, ss, o);
    if (lane == 0) {
      s_done[b] = done;
      s_base[b] = base;
      s_max[b] = mm;
      s_log[b] = logf(ss);
    }
  }
  __syncthreads();
  // candidates in batches of kBatch per thread beside the best of those before:
  // the code of score and beam, then that of logit and token.
  int kept = 0;
  for (int i0 = 0; i0 < n; i0 += kBatch * kBeamThreads) {
    if (i0 > 0) load(i0);
    const uint64_t old = tid < kept ? s_top[tid] : 0;
    const uint64_t old_key = tid < kept ? s_token[tid] : 0;
    uint64_t best = old, code[kBatch];
#pragma unroll
    for (int j = 0; j < kBatch; ++j) {
      const int i = i0 + j * kBeamThreads + tid;
      code[j] = 0;
      if (i < n) {
        const int b = i / per, c = i - b * per;
        const float base = s_base[b], top = s_max[b], log_sum = s_log[b];
        float score = -INFINITY;
        bool is = true;
        if (s_done[b]) {
          // the pad token, then others at -inf in order
          is = c < k;
          if (c == 0) score = base;
          key[j] = rank_key(-INFINITY, c == 0 ? p.pad : c - 1 < p.pad ? c - 1 : c);
        } else if (!(fabsf(top) < INFINITY && fabsf(log_sum) < INFINITY &&
                     fabsf(base) < INFINITY)) {
          is = c < k;   // the beam has no finite candidate
          key[j] = rank_key(-INFINITY, c);
        } else {
          is = key[j] != 0;
          score = base + ((key_value(key[j]) - top) - log_sum);
        }
        if (!(score == score)) score = -INFINITY;
        // (impossible ones by beam and token)
        const uint32_t low = score == -INFINITY ? (uint32_t)b * p.vocab + key_index(key[j]) : b;
        if (is) code[j] = rank_key(score, low);
      }
      best = code[j] > best ? code[j] : best;
    }
    const uint64_t bound = block_bound(best, k, s_warp);
    auto keep = [&](uint64_t c, uint64_t logit) {
      if (c == 0 || c < bound) return;
      const int to = atomicAdd(&s_n, 1);
      s_list[to] = c;
      s_logit[to] = logit;
    };
    keep(old, old_key);
#pragma unroll
    for (int j = 0; j < kBatch; ++j) keep(code[j], key[j]);
    __syncthreads();
    const int found = s_n;
    for (int i = tid; i < found; i += kBeamThreads) {
      const uint64_t mine = s_list[i], logit = s_logit[i];
      int rank = 0, equal = 0;
      for (int j = 0; j < found; ++j) {
        const uint64_t other = s_list[j];
        rank += other > mine;
        equal += other == mine;
      }
      if (equal > 1)   // (rare)
        for (int j = 0; j < found; ++j) rank += s_list[j] == mine && s_logit[j] > logit;
      if (rank < k) {
        s_top[rank] = mine;
        s_token[rank] = logit;
      }
    }
    kept = min(found, k);
    __syncthreads();
    if (i0 + kBatch * kBeamThreads < n) {
      if (tid == 0) s_n = 0;
      __syncthreads();
    }
  }
  if (tid < k) {
    const float score = key_value(s_top[tid]);
    const uint32_t low = key_index(s_top[tid]);
    const int b = score == -INFINITY ? low / p.vocab : low, token = key_index(s_token[tid]);
    p.out_scores[(size_t)group * k + tid] = score;
    p.out_parents[(size_t)group * k + tid] = b;
    p.out_tokens[(size_t)group * k + tid] = token;
    if (p.out_done)
      p.out_done[(size_t)group * k + tid] = s_done[b] || token == p.eos;
  }
}

// Parts of a row: whole steps, as many parts as give every SM its CTAs.
int parts_of(int rows, int vocab, int *chunk) {
  const int steps = (vocab + kStep - 1) / kStep;
  long parts = (long)kCtasPerSm * sm_count() / (rows > 0 ? rows : 1);
  if (parts < 1) parts = 1;
  if (parts > steps) parts = steps;
  const int per = (int)((steps + parts - 1) / parts);
  *chunk = per * kStep;
  return (steps + per - 1) / per;
}

// --------------------------------------------------------------------------
// Reordering: one CTA per group, one thread per table column, which holds the
// column's entries of all beams (so the tables can change in place). Every
// warp works out the beams' parents by itself; no barriers.
// --------------------------------------------------------------------------
struct ReorderParams {
  const int *parents, *lens, *table_in;
  int *table_out;
  int beams, cols, page_size;
  int *copy_src, *copy_dst, *copy_fill;
  int *err;
};

template <int kBeams>   // at least p.beams
__global__ void __launch_bounds__(256) beam_reorder_kernel(const ReorderParams p) {
  griddep_launch();
  griddep_wait();
  __shared__ int s_ends[8][32];
  const int W = p.beams, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const size_t row0 = (size_t)blockIdx.x * W;
  const int len = p.lens[row0];
  const int up = lane < W ? p.parents[row0 + lane] : 0;
  const int c = len / p.page_size, f = len - c * p.page_size;
  const bool ok = __all_sync(~0u, up >= 0 && up < W && len >= 0 &&
                                      (f > 0 ? c < p.cols : c <= p.cols));
  // the page of column c: first children keep their parent's, in order the
  // others take those of the beams without a child
  const uint32_t same = __match_any_sync(~0u, lane < W ? up : -1 - lane);
  const bool first = (int)__ffs(same) - 1 == lane;
  uint32_t parents = lane < W ? 1u << (up & 31) : 0u;
  parents = __reduce_or_sync(~0u, parents);
  const uint32_t ends = (W == 32 ? ~0u : (1u << W) - 1) & ~parents;
  const uint32_t below = (1u << lane) - 1;
  if (ends >> lane & 1) s_ends[warp][__popc(ends & below)] = lane;
  __syncwarp();
  const uint32_t extra = __ballot_sync(~0u, lane < W && !first);
  const int target = lane < W && !first && ok ? s_ends[warp][__popc(extra & below)] : up;

  if (tid < W && !(ok && f > 0)) {
    p.copy_src[row0 + tid] = p.copy_dst[row0 + tid] = -1;
    p.copy_fill[row0 + tid] = 0;
  }
  if (tid == 0 && !ok) atomicOr(p.err, DEV_ERR_PAGE);
  for (int j0 = 0; j0 < p.cols; j0 += blockDim.x) {
    const int j = j0 + tid;
    const bool moved = ok && j < c, split = ok && j == c && f > 0;
    const bool work = j < p.cols && (p.table_out != p.table_in || moved || split);
    const int *in = p.table_in + row0 * p.cols + j;
    int v[kBeams], old[kBeams];
#pragma unroll
    for (int i = 0; i < kBeams; ++i) {
      const int u = __shfl_sync(~0u, up, i), t = __shfl_sync(~0u, target, i);
      if (i >= W || !work) continue;
      v[i] = in[(size_t)(moved ? u : split ? t : i) * p.cols];
      if (split) old[i] = in[(size_t)u * p.cols];
    }
#pragma unroll
    for (int i = 0; i < kBeams; ++i) {
      if (i >= W || !work) continue;
      p.table_out[(row0 + i) * p.cols + j] = v[i];
      if (split) {
        p.copy_src[row0 + i] = old[i];
        p.copy_dst[row0 + i] = v[i];
        p.copy_fill[row0 + i] = f;
      }
    }
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
  // the parts of all rows are at most as many (parts_of), whatever the vocabulary
  // and for fewer rows too
  const size_t rows = (size_t)groups * beams, most = (size_t)kCtasPerSm * sm_count();
  const size_t parts = rows > most ? rows : most;
  *bytes = kCounterBytes + align256(parts * sizeof(float2)) + parts * k * sizeof(uint64_t);
  return TLLM_OK;
}

extern "C" int tllm_beam_select(const tllm_beam_step *step, tllm_stream_t stream) {
  TLLM_INJECT("launch");
  TLLM_CHECK_ARG(step, "step is NULL");
  const float *logits = step->logits, *scores = step->scores;
  const int32_t *done = step->done;
  float *out_scores = step->out_scores;
  int32_t *out_parents = step->out_parents, *out_tokens = step->out_tokens;
  void *workspace = step->workspace;
  const size_t workspace_bytes = step->workspace_bytes;
  const long ld = step->ld;
  const int groups = step->groups, beams = step->beams, vocab = step->vocab, k = step->k;
  const int pad_token = step->pad_token;
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
  p.chunks = parts_of(groups * beams, vocab, &p.chunk);
  p.out_scores = out_scores;
  p.out_parents = out_parents;
  p.out_tokens = out_tokens;
  p.eos = step->eos_token;
  p.out_done = step->out_done;
  char *w = static_cast<char *>(workspace);
  p.counters = reinterpret_cast<int *>(w);
  w += kCounterBytes;
  p.stats = reinterpret_cast<float2 *>(w);
  w += align256((size_t)groups * beams * p.chunks * sizeof(float2));
  p.lists = reinterpret_cast<uint64_t *>(w);
  const bool vec = ((uintptr_t)logits & 15) == 0 && p.ld % 4 == 0;
  TLLM_CUDA(launch_pdl(vec ? beam_select_kernel<true> : beam_select_kernel<false>,
                       dim3(p.chunks, groups * beams), dim3(kBeamThreads), 0,
                       resolve(stream), p));
  return TLLM_OK;
}

extern "C" int tllm_beam_reorder(const tllm_beam_tables *t, tllm_stream_t stream) {
  TLLM_INJECT("launch");
  TLLM_CHECK_ARG(t, "tables is NULL");
  const int groups = t->groups, beams = t->beams, table_cols = t->table_cols;
  const int page_size = t->page_size;
  TLLM_CHECK_ARG(groups >= 0 && beams >= 1 && beams <= kMaxBeams,
                 "groups (%d) must be >= 0 and beams (%d) in [1, %d]", groups, beams, kMaxBeams);
  TLLM_CHECK_ARG(table_cols >= 0 && page_size >= 1, "invalid table: %d columns of %d slots",
                 table_cols, page_size);
  if (groups == 0) return TLLM_OK;
  TLLM_CHECK_ARG(t->parents && t->lens && t->copy_src && t->copy_dst && t->copy_fill &&
                     (table_cols == 0 || (t->table_in && t->table_out)),
                 "NULL pointer");
  ReorderParams p;
  p.parents = t->parents;
  p.lens = t->lens;
  p.table_in = t->table_in;
  p.table_out = t->table_out;
  p.beams = beams;
  p.cols = table_cols;
  p.page_size = page_size;
  p.copy_src = t->copy_src;
  p.copy_dst = t->copy_dst;
  p.copy_fill = t->copy_fill;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
  const int threads = table_cols >= 256 ? 256 : (table_cols + 31) / 32 * 32 > 32
                                                    ? (table_cols + 31) / 32 * 32
                                                    : 32;
  TLLM_CUDA(launch_pdl(beams <= 8 ? beam_reorder_kernel<8> : beam_reorder_kernel<kMaxBeams>,
                       dim3(groups), dim3(threads), 0, resolve(stream), p));
  return TLLM_OK;
}
