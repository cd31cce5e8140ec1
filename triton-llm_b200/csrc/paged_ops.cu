// Writing and moving the pages of a paged KV cache, for sm_100a: new tokens
// with rotary positions (tllm_paged_append) and page copies over the planes of
// an arena (tllm_page_copy).
#include "mma_sync.cuh"
#include "paged.cuh"

namespace tllm {
namespace {

// --------------------------------------------------------------------------
// Append
// --------------------------------------------------------------------------
struct AppendParams {
  PagedView kv;
  tllm_paged_rows in;
  bool stream;   // the results do not stay in L2
  int *err;
};

template <typename S>
__device__ __forceinline__ float load_src(const S *p) {
  if constexpr (sizeof(S) == 4)
    return *p;
  else
    return bf16_bits_to_f32(*p);
}

// Position of value d of a head in the source.
__device__ __forceinline__ int source_dim(int d, int D, int blocked) {
  if (!blocked) return d;
  const int half = D >> 1;
  return d < half ? (d >> 3) * 16 + (d & 7) : ((d - half) >> 3) * 16 + 8 + ((d - half) & 7);
}

__device__ __forceinline__ bool source_ok(const AppendParams &p, int src) {
  return src >= 0 && (p.in.src_rows == 0 || src < p.in.src_rows);
}

// Row `row` of the call: cache row index, position, page, slot; false (and an
// error bit) where an index is out of range.
struct AppendRow {
  int seq, pos, page, slot;
  size_t src;
};
__device__ __forceinline__ bool append_row(const AppendParams &p, int row, AppendRow *r) {
  r->seq = p.in.row_seq ? p.in.row_seq[row] : row;
  r->pos = p.in.row_pos[row];
  const int src = p.in.row_src ? p.in.row_src[row] : row;
  r->src = src;
  bool ok = source_ok(p, src) && r->seq >= 0 && r->seq < p.kv.n_seq && r->pos >= 0 &&
            r->pos < p.kv.table_cols * p.kv.page_size &&
            (!p.in.cos_t || r->pos < p.in.n_pos);
  if (ok) {
    const int col = p.kv.column(r->pos);
    r->slot = r->pos - col * p.kv.page_size;
    r->page = p.kv.table[(size_t)r->seq * p.kv.table_stride + col];
    ok = r->page >= 0 && r->page < p.kv.n_pages;
  }
  if (!ok && threadIdx.x == 0) atomicOr(p.err, DEV_ERR_PAGE);
  return ok;
}

// Any head_dim, rotary part and alignment: one thread per rotated pair or
// passed value.
template <typename S, typename T>
__global__ void append_kernel(const __grid_constant__ AppendParams p) {
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.x;
  AppendRow r;
  if (!append_row(p, row, &r)) return;
  if (threadIdx.x == 0 && p.in.lens_out) atomicMax(p.in.lens_out + r.seq, r.pos + 1);
  const int D = p.kv.head_dim, H = p.in.q ? p.in.n_head : 0, K = p.kv.n_kv;
  const int rot = p.in.cos_t ? p.in.rotary_dim : 0, pairs = rot >> 1;
  const int per = D - pairs;
  for (int i = threadIdx.x; i < (H + 2 * K) * per; i += blockDim.x) {
    const int head = i / per, u = i - head * per;
    const bool is_v = head >= H + K;
    const S *src;
    float *qo = nullptr;
    T *to = nullptr;
    if (head < H) {
      src = static_cast<const S *>(p.in.q) + r.src * p.in.q_row_stride +
            (size_t)head * p.in.q_head_stride;
      qo = p.in.q_out + (size_t)row * p.in.q_out_row_stride +
           (size_t)head * p.in.q_out_head_stride;
    } else if (!is_v) {
      src = static_cast<const S *>(p.in.k) + r.src * p.in.k_row_stride +
            (size_t)(head - H) * p.in.k_head_stride;
      to = static_cast<T *>(p.kv.k) + p.kv.offset(r.page, head - H, r.slot);
    } else {
      src = static_cast<const S *>(p.in.v) + r.src * p.in.v_row_stride +
            (size_t)(head - H - K) * p.in.v_head_stride;
      to = static_cast<T *>(p.kv.v) + p.kv.offset(r.page, head - H - K, r.slot);
    }
    auto put = [&](int d, float v) {
      if (qo)
        qo[d] = v;
      else if constexpr (sizeof(T) == 4)
        to[d] = v;
      else
        to[d] = f32_to_bf16_bits(v);
    };
    if (u < pairs) {
      const int a = p.in.interleaved ? 2 * u : u;
      const int b = p.in.interleaved ? 2 * u + 1 : u + pairs;
      const float x = load_src(src + source_dim(a, D, p.in.blocked));
      const float y = load_src(src + source_dim(b, D, p.in.blocked));
      float c = 1.f, s = 0.f;
      if (!is_v) {
        c = p.in.cos_t[(size_t)r.pos * pairs + u];
        s = p.in.sin_t[(size_t)r.pos * pairs + u];
      }
      put(a, is_v ? x : x * c - y * s);
      put(b, is_v ? y : y * c + x * s);
    } else {
      const int d = u + pairs;
      put(d, load_src(src + source_dim(d, D, p.in.blocked)));
    }
  }
}

// Four values of the source, and four results to fp32 or bf16.
__device__ __forceinline__ float4 load4(const float *p) {
  return __ldcs(reinterpret_cast<const float4 *>(p));
}
__device__ __forceinline__ float4 load4(const uint16_t *p) {
  const uint2 v = __ldcs(reinterpret_cast<const uint2 *>(p));
  return make_float4(bf16lo(v.x), bf16hi(v.x), bf16lo(v.y), bf16hi(v.y));
}
// (`stream`: not kept in L2)
__device__ __forceinline__ void store4(float *p, float4 v, bool stream) {
  if (stream)
    __stcs(reinterpret_cast<float4 *>(p), v);
  else
    *reinterpret_cast<float4 *>(p) = v;
}
__device__ __forceinline__ void store4(uint16_t *p, float4 v, bool stream) {
  const uint2 r = make_uint2(pack_bf16x2(v.x, v.y), pack_bf16x2(v.z, v.w));
  if (stream)
    __stcs(reinterpret_cast<uint2 *>(p), r);
  else
    *reinterpret_cast<uint2 *>(p) = r;
}

// Heads of whole 8-value units on 16-byte rows: one thread takes U units of two
// runs of four values (a pair's two sides, or eight neighbours), with all its
// loads issued before the row's page is known. U = 4 for many rows, bound by HBM
// (12001 rows of 24 / 8 heads of 128: 73 us, 0.94 of its bandwidth; with 2 or 8
// units 4 and 17 % more), U = 2 for few, bound by latency (64 rows: 2.8 us, with
// 4, 3.4). One CTA per row: a row moves a few KB, and 12 or more CTAs of an SM
// cover the chain of loads position -> page -> store.
template <typename S, typename T, int kUnits>
__global__ void __launch_bounds__(512)
    append_units_kernel(const __grid_constant__ AppendParams p) {
  griddep_launch();
  griddep_wait();
  const int row = blockIdx.x;
  const int D = p.kv.head_dim, H = p.in.q ? p.in.n_head : 0, K = p.kv.n_kv;
  const int rot = p.in.cos_t ? p.in.rotary_dim : 0, half = rot >> 1;
  const unsigned per = D >> 3, n = (H + 2 * K) * per;
  const int src_row = p.in.row_src ? p.in.row_src[row] : row;
  const size_t from = source_ok(p, src_row) ? src_row : 0;   // (else skipped below)
  float4 x[kUnits], y[kUnits];
  int heads[kUnits], at_a[kUnits], at_b[kUnits];   // (head * 2 + whether it turns)
  // runs a and b of unit u of a head
  auto runs = [&](int head, int u, int *a, int *b) {
    const bool turned = head < H + K && u < rot >> 3;
    *a = turned && !p.in.interleaved ? 4 * u : 8 * u;
    *b = *a + (turned && !p.in.interleaved ? half : 4);
    return turned;
  };
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const unsigned at = threadIdx.x + i * blockDim.x;
    if (at >= n) continue;
    const int head = at / per, u = at - head * per;
    int a, b;
    heads[i] = head * 2 + runs(head, u, &a, &b);
    at_a[i] = a;
    at_b[i] = b;
    const S *src;
    if (head < H)
      src = static_cast<const S *>(p.in.q) + from * p.in.q_row_stride +
            (size_t)head * p.in.q_head_stride;
    else if (head < H + K)
      src = static_cast<const S *>(p.in.k) + from * p.in.k_row_stride +
            (size_t)(head - H) * p.in.k_head_stride;
    else
      src = static_cast<const S *>(p.in.v) + from * p.in.v_row_stride +
            (size_t)(head - H - K) * p.in.v_head_stride;
    x[i] = load4(src + source_dim(a, D, p.in.blocked));
    y[i] = load4(src + source_dim(b, D, p.in.blocked));
  }
  AppendRow r;
  if (!append_row(p, row, &r)) return;
  if (threadIdx.x == 0 && p.in.lens_out) atomicMax(p.in.lens_out + r.seq, r.pos + 1);
#pragma unroll
  for (int i = 0; i < kUnits; ++i) {
    const unsigned at = threadIdx.x + i * blockDim.x;
    if (at >= n) continue;
    const int head = heads[i] >> 1, a = at_a[i], b = at_b[i];
    if (heads[i] & 1) {
      const size_t t = (size_t)r.pos * half + (p.in.interleaved ? a >> 1 : a);
      const float4 c = __ldg(reinterpret_cast<const float4 *>(p.in.cos_t + t));
      const float4 s = __ldg(reinterpret_cast<const float4 *>(p.in.sin_t + t));
      const float4 v = x[i], w = y[i];
      if (p.in.interleaved) {
        x[i] = make_float4(v.x * c.x - v.y * s.x, v.y * c.x + v.x * s.x,
                           v.z * c.y - v.w * s.y, v.w * c.y + v.z * s.y);
        y[i] = make_float4(w.x * c.z - w.y * s.z, w.y * c.z + w.x * s.z,
                           w.z * c.w - w.w * s.w, w.w * c.w + w.z * s.w);
      } else {
        x[i] = make_float4(v.x * c.x - w.x * s.x, v.y * c.y - w.y * s.y,
                           v.z * c.z - w.z * s.z, v.w * c.w - w.w * s.w);
        y[i] = make_float4(w.x * c.x + v.x * s.x, w.y * c.y + v.y * s.y,
                           w.z * c.z + v.z * s.z, w.w * c.w + v.w * s.w);
      }
    }
    if (head < H) {
      float *to = p.in.q_out + (size_t)row * p.in.q_out_row_stride +
                  (size_t)head * p.in.q_out_head_stride;
      store4(to + a, x[i], p.stream);
      store4(to + b, y[i], p.stream);
    } else {
      const bool is_v = head >= H + K;
      T *to = static_cast<T *>(is_v ? p.kv.v : p.kv.k) +
              p.kv.offset(r.page, head - H - (is_v ? K : 0), r.slot);
      store4(to + a, x[i], p.stream);
      store4(to + b, y[i], p.stream);
    }
  }
}

// Units of a thread, or 0 where a run of four values that the call touches may
// not be aligned, or a row does not fit one CTA.
int append_units(const AppendParams &p) {
  const tllm_paged_rows &in = p.in;
  const int src = in.src_dtype == TLLM_F32 ? 4 : 2;
  long strides = in.k_row_stride | in.k_head_stride | in.v_row_stride | in.v_head_stride |
                 p.kv.page_stride | p.kv.head_stride | p.kv.slot_stride;
  // addresses aligned to four values of their type
  bool ok = ((uintptr_t)in.k | (uintptr_t)in.v) % (4 * src) == 0 &&
            ((uintptr_t)p.kv.k | (uintptr_t)p.kv.v) % 16 == 0;
  if (in.q) {
    strides |= in.q_row_stride | in.q_head_stride | in.q_out_row_stride | in.q_out_head_stride;
    ok = ok && (uintptr_t)in.q % (4 * src) == 0 && (uintptr_t)in.q_out % 16 == 0;
  }
  if (in.cos_t)
    ok = ok && ((uintptr_t)in.cos_t | (uintptr_t)in.sin_t) % 16 == 0 && in.rotary_dim % 8 == 0;
  const long units = ((in.q ? in.n_head : 0) + 2L * p.kv.n_kv) * (p.kv.head_dim / 8);
  if (!ok || strides % 4 || p.kv.head_dim % 8 || units > 512 * 4) return 0;
  return in.rows <= 4 * sm_count() && units <= 512 * 2 ? 2 : 4;
}

template <typename S, typename T>
int launch_append(AppendParams &p, cudaStream_t st) {
  const int D = p.kv.head_dim, rot = p.in.cos_t ? p.in.rotary_dim : 0;
  const long heads = (p.in.q ? p.in.n_head : 0) + 2L * p.kv.n_kv;
  if (const int units = append_units(p)) {
    const long threads = (heads * (D / 8) + units - 1) / units;
    // Results of about the size of L2 (126 MB) would only push one another out:
    // past half of it they are stored as streams (12001 rows, 197 MB: 78 -> 73
    // us); smaller ones stay for the attention that reads them next.
    p.stream = (long)p.in.rows * D * (heads * 4L) > 64L << 20;
    TLLM_CUDA(launch_pdl(units == 2 ? append_units_kernel<S, T, 2> : append_units_kernel<S, T, 4>,
                         dim3(p.in.rows), dim3((unsigned)((threads + 31) / 32 * 32)), 0, st, p));
    return TLLM_OK;
  }
  const long items = heads * (D - rot / 2);
  const int threads = items >= 512 ? 512 : (int)((items + 31) / 32 * 32);
  TLLM_CUDA(launch_pdl(append_kernel<S, T>, dim3(p.in.rows), dim3(threads), 0, st, p));
  return TLLM_OK;
}

// --------------------------------------------------------------------------
// Page copies
// --------------------------------------------------------------------------
struct CopyParams {
  char *arena;
  const int *src, *dst, *fill;
  long plane_stride, page_stride, run_stride;
  int n_pages, heads, page_size, row_bytes;
  int *err;
};

// One CTA per (copy, plane). A warp takes pieces of kDeep units per lane of a
// run, all loaded before the first is stored: 8 warps x 32 lanes x 16 units of
// 16 bytes keep 64 KB of a CTA in flight (8 units: forking beams 27.4 us, 16:
// 26.4; compaction is at the copy bandwidth with either).
constexpr int kCopyWarps = 8, kDeep = 16;

template <typename U>
__global__ void __launch_bounds__(kCopyWarps * 32) page_copy_kernel(const CopyParams p) {
  griddep_launch();
  griddep_wait();
  const int i = blockIdx.x;
  const int src = p.src[i], dst = p.dst[i], fill = p.fill ? p.fill[i] : p.page_size;
  if (src < 0 || dst < 0 || src == dst) return;
  if (src >= p.n_pages || dst >= p.n_pages || fill < 0 || fill > p.page_size) {
    if (threadIdx.x == 0) atomicOr(p.err, DEV_ERR_PAGE);
    return;
  }
  const size_t plane = (size_t)blockIdx.y * p.plane_stride;
  const char *from = p.arena + plane + (size_t)src * p.page_stride;
  char *to = p.arena + plane + (size_t)dst * p.page_stride;
  const int n = (int)((size_t)fill * p.row_bytes / sizeof(U));   // units of a run
  const int pieces = (n + 32 * kDeep - 1) / (32 * kDeep);
  const int lane = threadIdx.x & 31;
  for (int k = threadIdx.x >> 5; k < pieces * p.heads; k += kCopyWarps) {
    const int h = k / pieces, first = (k - h * pieces) * 32 * kDeep + lane;
    const U *f = reinterpret_cast<const U *>(from + (size_t)h * p.run_stride);
    U *t = reinterpret_cast<U *>(to + (size_t)h * p.run_stride);
    U v[kDeep];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      if (first + d * 32 < n) v[d] = f[first + d * 32];
#pragma unroll
    for (int d = 0; d < kDeep; ++d)
      if (first + d * 32 < n) t[first + d * 32] = v[d];
  }
}

}  // namespace
}  // namespace tllm

using namespace tllm;

extern "C" int tllm_paged_append(const tllm_paged_kv *kv, const tllm_paged_rows *in,
                                 tllm_stream_t stream) {
  TLLM_INJECT("launch");
  AppendParams p;
  int rc = paged_view(kv, &p.kv);
  if (rc) return rc;
  TLLM_CHECK_ARG(in, "rows is NULL");
  const int D = kv->head_dim;
  TLLM_CHECK_ARG(in->rows >= 0 && in->src_rows >= 0, "rows (%d) and src_rows (%d) must be >= 0",
                 in->rows, in->src_rows);
  TLLM_CHECK_ARG(in->row_src || in->src_rows == 0 || in->rows <= in->src_rows,
                 "%d rows of %d source rows", in->rows, in->src_rows);
  TLLM_CHECK_ARG(in->src_dtype == TLLM_F32 || in->src_dtype == TLLM_BF16,
                 "src_dtype must be F32 or BF16");
  TLLM_CHECK_ARG(!in->q || in->n_head > 0, "n_head (%d) must be > 0", in->n_head);
  if (in->rows == 0) return TLLM_OK;
  TLLM_CHECK_ARG(in->k && in->v && in->row_pos, "NULL tensor pointer");
  TLLM_CHECK_ARG(!in->q || in->q_out, "q without q_out");
  TLLM_CHECK_ARG(in->row_seq || in->rows <= kv->n_seq,
                 "%d rows for a table of %d sequences (pass row_seq)", in->rows, kv->n_seq);
  TLLM_CHECK_ARG(!in->cos_t == !in->sin_t, "cos_t and sin_t go together");
  if (in->cos_t)
    TLLM_CHECK_ARG(in->rotary_dim >= 2 && in->rotary_dim % 2 == 0 && in->rotary_dim <= D &&
                       in->n_pos > 0,
                   "rotary_dim (%d) must be even, within head_dim (%d), and n_pos (%d) > 0",
                   in->rotary_dim, D, in->n_pos);
  TLLM_CHECK_ARG(!in->blocked || D % 16 == 0, "blocked heads need head_dim %% 16 == 0");
  TLLM_CHECK_ARG(in->q_row_stride >= 0 && in->q_head_stride >= 0 && in->k_row_stride >= 0 &&
                     in->k_head_stride >= 0 && in->v_row_stride >= 0 &&
                     in->v_head_stride >= 0 && in->q_out_row_stride >= 0 &&
                     in->q_out_head_stride >= 0,
                 "negative stride");
  TLLM_CHECK_ARG((const void *)in->q_out != in->q || !in->q ||
                     (!in->blocked && !in->row_src && in->src_dtype == TLLM_F32 &&
                      in->q_row_stride == in->q_out_row_stride &&
                      in->q_head_stride == in->q_out_head_stride),
                 "q in place needs fp32 rows in plain order with the same strides");
  p.in = *in;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
  cudaStream_t st = resolve(stream);
  const bool t32 = kv->kv_dtype == TLLM_F32;
  if (in->src_dtype == TLLM_F32)
    return t32 ? launch_append<float, float>(p, st) : launch_append<float, uint16_t>(p, st);
  return t32 ? launch_append<uint16_t, float>(p, st) : launch_append<uint16_t, uint16_t>(p, st);
}

extern "C" int tllm_page_copy(void *arena, long plane_stride, int planes, long page_stride,
                              int n_pages, int heads, long run_stride, int page_size,
                              int row_bytes, const int32_t *src, const int32_t *dst,
                              const int32_t *fill, int n_copies, tllm_stream_t stream) {
  TLLM_INJECT("launch");
  TLLM_CHECK_ARG(planes >= 0 && planes <= 65535 && n_pages >= 0 && heads >= 0 &&
                     page_size >= 1 && row_bytes >= 1 && n_copies >= 0,
                 "invalid arena: %d planes, %d pages of %d runs of %d slots of %d bytes, %d copies",
                 planes, n_pages, heads, page_size, row_bytes, n_copies);
  TLLM_CHECK_ARG((long)page_size * row_bytes <= (1L << 30), "a run of a page must be at most 1 GiB");
  TLLM_CHECK_ARG(plane_stride >= 0 && page_stride >= 0 && run_stride >= 0, "negative stride");
  if (planes == 0 || heads == 0 || n_copies == 0) return TLLM_OK;
  TLLM_CHECK_ARG(arena && src && dst, "NULL pointer");
  CopyParams p;
  p.arena = static_cast<char *>(arena);
  p.src = src;
  p.dst = dst;
  p.fill = fill;
  p.plane_stride = plane_stride;
  p.page_stride = page_stride;
  p.run_stride = run_stride;
  p.n_pages = n_pages;
  p.heads = heads;
  p.page_size = page_size;
  p.row_bytes = row_bytes;
  p.err = device_error_ptr();
  TLLM_CHECK_ARG(p.err, "device error word unavailable");
  cudaStream_t st = resolve(stream);
  const unsigned long bits = (unsigned long)(uintptr_t)arena | plane_stride | page_stride |
                             run_stride | row_bytes;
  const dim3 grid(n_copies, planes);
  if (bits % 16 == 0)
    TLLM_CUDA(launch_pdl(page_copy_kernel<uint4>, grid, dim3(kCopyWarps * 32), 0, st, p));
  else if (bits % 4 == 0)
    TLLM_CUDA(launch_pdl(page_copy_kernel<uint32_t>, grid, dim3(kCopyWarps * 32), 0, st, p));
  else
    TLLM_CUDA(launch_pdl(page_copy_kernel<uint8_t>, grid, dim3(kCopyWarps * 32), 0, st, p));
  return TLLM_OK;
}
