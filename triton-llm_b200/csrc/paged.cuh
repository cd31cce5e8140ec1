// Device view of a paged KV cache (tllm_paged_kv) shared by the kernels that
// read and write it, and the host-side checks of its fields.
#pragma once

#include "common.cuh"

namespace tllm {

// Slot s of head h of page p starts at element
// p * page_stride + h * head_stride + s * slot_stride of k and v.
struct PagedView {
  void *k, *v;
  const int *table;      // (n_seq, table_cols), rows table_stride apart
  long page_stride, head_stride, slot_stride, table_stride;
  int n_pages, page_size, page_shift;   // page_shift: log2(page_size) or -1
  int n_kv, head_dim, n_seq, table_cols;

  // Table column and slot of position pos.
  __device__ __forceinline__ int column(int pos) const {
    return page_shift >= 0 ? pos >> page_shift : (int)((unsigned)pos / (unsigned)page_size);
  }
  __device__ __forceinline__ size_t offset(int page, int head, int slot) const {
    return (size_t)page * page_stride + (size_t)head * head_stride +
           (size_t)slot * slot_stride;
  }
};

// Checks kv and fills view; `what` names the entry point's tensors in errors.
int paged_view(const tllm_paged_kv *kv, PagedView *view);

}  // namespace tllm
