// A paged key/value cache as the kernels see it: row r of sequence b lies in page table[b][r / page] at r % page.
// A table entry outside [0, P) holds nothing: its rows are masked when read and dropped when written, so that no
// entry can lead a kernel out of the cache.
#pragma once
#include "common.cuh"

namespace kb {

struct PagedView {
  char* k;
  char* v;
  float* k_scale;
  float* v_scale;
  int64_t k_page, k_head, k_row;     // elements
  int64_t v_page, v_head, v_row;
  int64_t ks_page, ks_head, ks_row;
  int64_t vs_page, vs_head, vs_row;
  const int32_t* table;
  int64_t table_b, table_m;
  const int32_t* lens;
  int64_t lens_b;
  int32_t P, page, capacity;         // capacity: M * page rows
  KbFastDiv fd_page;

  // The sequence's rows: its length, within what its table can name.
  __device__ __forceinline__ int32_t rows(int32_t b) const { return kb_clamp_len(lens[b * lens_b], capacity); }
  // Page of a row below `capacity` (-1: none) and the row's place in it.
  __device__ __forceinline__ int32_t locate(int32_t b, int32_t row, int32_t& at) const {
    const int32_t m = kb_fastdiv(row, fd_page);
    at = row - m * page;
    const int32_t id = table[b * table_b + m * table_m];
    return (uint32_t)id < (uint32_t)P ? id : -1;
  }
  __device__ __forceinline__ bool has_page(int32_t b, int32_t m) const { return (uint32_t)table[b * table_b + m * table_m] < (uint32_t)P; }
};

inline PagedView make_paged_view(const kb_paged_cache& c) {
  PagedView w{};
  w.k = static_cast<char*>(c.k), w.v = static_cast<char*>(c.v);
  w.k_scale = c.k_scale, w.v_scale = c.v_scale;
  w.k_page = c.k_stride[0], w.k_head = c.k_stride[1], w.k_row = c.k_stride[2];
  w.v_page = c.v_stride[0], w.v_head = c.v_stride[1], w.v_row = c.v_stride[2];
  w.ks_page = c.k_scale_stride[0], w.ks_head = c.k_scale_stride[1], w.ks_row = c.k_scale_stride[2];
  w.vs_page = c.v_scale_stride[0], w.vs_head = c.v_scale_stride[1], w.vs_row = c.v_scale_stride[2];
  w.table = c.page_table, w.table_b = c.table_stride[0], w.table_m = c.table_stride[1];
  w.lens = c.lens, w.lens_b = c.lens_stride;
  w.P = c.P, w.page = c.page, w.capacity = c.M * c.page;
  w.fd_page = kb_fastdiv_make(c.page);
  return w;
}

// Whether every row of the pages starts on a 16-byte boundary.
inline bool paged_rows_aligned(const kb_paged_cache& c, int elsize) {
  if (reinterpret_cast<uintptr_t>(c.k) % 16 || reinterpret_cast<uintptr_t>(c.v) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (c.k_stride[i] * elsize % 16 || c.v_stride[i] * elsize % 16) return false;
  return true;
}

// Launches of one call overlap: a kernel started with `launch_after` may start while the one before it in the stream still
// runs, and waits for it, its writes included, where it calls `wait_for_launch_before` (before it reads or writes anything that
// the other touches).
__device__ __forceinline__ void wait_for_launch_before() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void let_next_launch_start() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }

template <typename... Args>
int launch_after(void (*kernel)(Args...), dim3 grid, int threads, cudaStream_t s, const Args&... args) {
  cudaLaunchConfig_t c = {};
  c.gridDim = grid, c.blockDim = dim3(threads), c.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeProgrammaticStreamSerialization;
  at.val.programmaticStreamSerializationAllowed = 1;
  c.attrs = &at, c.numAttrs = 1;
  KB_CUDA_TRY(cudaLaunchKernelEx(&c, kernel, args...));
  count_launch();
  return KB_OK;
}

inline int dtype_size(int32_t dtype) { return dtype == KB_F32 ? 4 : dtype == KB_E4M3 ? 1 : 2; }

}  // namespace kb
