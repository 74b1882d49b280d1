// The upkeep of a paged key/value cache: new tokens are written into their rows, and rows are evicted by the attention
// weight that they have received.
//
// WRITE.  Token t < n_b of sequence b goes to row len_b - n_b + t.  HBM-bound: every element is read once and written
// once.  A row of one head is eight elements per thread, D / 8 neighbouring threads: its largest magnitude, which sets
// the scale of an 8-bit row, is a few shuffles away, and rows stay independent of one another.
//
// EVICT.  Rows rank by (position among the newest `recent`, then weight, then the lower row); the first `budget` stay.
// The kept rows below the budget stay where they are, and the i-th kept row behind it moves to the i-th place that came
// free before it.  Attention does not depend on the rows' order, so nothing else has to move: a cache that is one row
// over its budget moves one row, not half of them.  Sources lie behind the budget and destinations before it, so all
// moves are independent.  Two kernels: one block per (sequence, head) picks the rows, then the moves are spread over
// the GPU.
#include "common.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace kb {
namespace {

// ---- write -----------------------------------------------------------------------------------------------------------

constexpr int kWriteThreads = 256, kPerThread = 8;

struct WriteArgs {
  PagedView c;
  const void* x[2];  // k, v
  int64_t sb[2], sh[2], st[2], sd[2];
  const int32_t* new_lens;
  int64_t new_lens_b;
  const int32_t* positions;
  int64_t pos_b, pos_t;
  float* weights;
  int32_t* row_positions;
  int64_t w_b, w_h, p_b, p_h;
  int32_t B, H_kv, T, D, rows_per_cta;
  KbFastDiv fd_T, fd_H;
  bool aligned;
};

// x / scale, correctly rounded: the row's elements as its 8-bit form holds them
__device__ __forceinline__ uint2 quantize8(const float (&f)[8], float scale) {
  return make_uint2(sm100::pack_e4m3x4(__fdiv_rn(f[0], scale), __fdiv_rn(f[1], scale), __fdiv_rn(f[2], scale), __fdiv_rn(f[3], scale)),
                    sm100::pack_e4m3x4(__fdiv_rn(f[4], scale), __fdiv_rn(f[5], scale), __fdiv_rn(f[6], scale), __fdiv_rn(f[7], scale)));
}

// T: the tokens' type; F8: the cache holds e4m3, otherwise T
template <typename T, bool F8>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteArgs a) {
  const int lanes = a.D / kPerThread;  // 2, 4, 8, 16 or 32 threads per row
  const int lane = threadIdx.x & (lanes - 1);
  const int64_t row_id = (int64_t)blockIdx.x * a.rows_per_cta + threadIdx.x / lanes;  // (b, h, t)
  const int which = blockIdx.y;
  bool live = row_id < (int64_t)a.B * a.H_kv * a.T;
  int32_t b = 0, h = 0, t = 0, at = 0, page = -1;
  if (live) {
    const int32_t bh = kb_fastdiv((int32_t)row_id, a.fd_T);
    t = (int32_t)row_id - bh * a.T;
    b = kb_fastdiv(bh, a.fd_H);
    h = bh - b * a.H_kv;
    const int32_t n = a.new_lens ? kb_clamp_len(a.new_lens[b * a.new_lens_b], a.T) : a.T;
    const int64_t row = (int64_t)a.c.lens[b * a.c.lens_b] - n + t;
    live = t < n && row >= 0 && row < a.c.capacity;
    if (live) {
      page = a.c.locate(b, (int32_t)row, at);
      if (which == 0 && lane == 0) {
        if (a.weights) a.weights[b * a.w_b + h * a.w_h + row] = 0.f;
        if (a.row_positions) a.row_positions[b * a.p_b + h * a.p_h + row] = a.positions ? a.positions[b * a.pos_b + t * a.pos_t] : (int32_t)row;
      }
    }
  }
  live = live && page >= 0;
  T e[kPerThread];
  const int d = lane * kPerThread;
  if (live) {
    const T* x = static_cast<const T*>(a.x[which]) + b * a.sb[which] + h * a.sh[which] + t * a.st[which] + d * a.sd[which];
    if (a.aligned) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * kPerThread / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldcs(reinterpret_cast<const uint4*>(x) + i);
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) e[i] = x[i * a.sd[which]];
    }
  } else {
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) e[i] = from_f32<T>(0.f);
  }
  const int64_t at_page = which ? page * a.c.v_page + h * a.c.v_head + at * a.c.v_row : page * a.c.k_page + h * a.c.k_head + at * a.c.k_row;
  char* base = which ? a.c.v : a.c.k;
  if constexpr (F8) {
    float f[kPerThread];
    // as bits without the sign: numbers keep their order, and a NaN is above them all, so that it reaches the scale
    uint32_t m = 0;
#pragma unroll
    for (int i = 0; i < kPerThread; ++i) {
      f[i] = to_f32(e[i]);
      m = max(m, __float_as_uint(f[i]) & 0x7fffffffu);
    }
    for (int s = lanes / 2; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
    float scale = __fmul_rn(__uint_as_float(m), 1.f / 448.f);
    if (scale < 1e-12f) scale = 1e-12f;  // (a NaN stays)
    if (live) {
      if (lane == 0) {
        if (which) a.c.v_scale[page * a.c.vs_page + h * a.c.vs_head + at * a.c.vs_row] = scale;
        else a.c.k_scale[page * a.c.ks_page + h * a.c.ks_head + at * a.c.ks_row] = scale;
      }
      const uint2 w = quantize8(f, scale);
      uint8_t* out = reinterpret_cast<uint8_t*>(base) + at_page + d;
      if (a.aligned) {
        *reinterpret_cast<uint2*>(out) = w;
      } else {
        const uint8_t* wb = reinterpret_cast<const uint8_t*>(&w);
#pragma unroll
        for (int i = 0; i < kPerThread; ++i) out[i] = wb[i];
      }
    }
  } else if (live) {
    T* out = reinterpret_cast<T*>(base) + at_page + d;
    if (a.aligned) {
#pragma unroll
      for (int i = 0; i < (int)sizeof(T) * kPerThread / 16; ++i) reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(e)[i];
    } else {
#pragma unroll
      for (int i = 0; i < kPerThread; ++i) out[i] = e[i];
    }
  }
}

template <typename T>
int launch_write(const WriteArgs& a, bool f8, cudaStream_t s) {
  const int64_t rows = (int64_t)a.B * a.H_kv * a.T;
  const dim3 grid((unsigned)((rows + a.rows_per_cta - 1) / a.rows_per_cta), 2);
  if (f8) paged_write_kernel<T, true><<<grid, kWriteThreads, 0, s>>>(a);
  else paged_write_kernel<T, false><<<grid, kWriteThreads, 0, s>>>(a);
  KB_LAUNCH_CHECK("paged_write_kernel");
  return KB_OK;
}

// ---- evict -----------------------------------------------------------------------------------------------------------

constexpr int kSelectThreads = 1024, kMoveThreads = 256;

struct EvictArgs {
  PagedView c;
  const float* weights;
  const int32_t* positions;
  float* weights_out;
  int32_t* positions_out;
  int32_t* lens_out;
  int64_t w_b, w_h, p_b, p_h, wo_b, wo_h, po_b, po_h, lens_out_b;
  int32_t H_kv, D, budget, recent, most_moves, elsize;
  int32_t* counts;  // [B, H_kv]
  int32_t* src;     // [B, H_kv, most_moves]
  int32_t* dst;
  bool in_place, aligned;
};

// Weights as whole numbers of the same order; a NaN is below them all, the newest rows are above.
__device__ __forceinline__ uint32_t rank_key(float w, bool newest) {
  if (newest) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (one zero)
  if (w != w) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

__device__ __forceinline__ int block_sum(int x, int* red) {
  x = __reduce_add_sync(0xffffffffu, x);
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, (int)(threadIdx.x & 31) < (int)(blockDim.x >> 5) ? red[threadIdx.x & 31] : 0);
}

// Sum over the warps before this one of x (the same in all lanes of a warp).
__device__ __forceinline__ int warps_before(int x, int* red) {
  __syncthreads();
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = x;
  __syncthreads();
  return __reduce_add_sync(0xffffffffu, (threadIdx.x & 31) < (threadIdx.x >> 5) ? red[threadIdx.x & 31] : 0);
}

__global__ void __launch_bounds__(kSelectThreads) paged_select_kernel(const EvictArgs a) {
  __shared__ int red[32];
  const int32_t h = blockIdx.x, b = blockIdx.y;
  const int32_t n = a.c.rows(b);
  const float* w = a.weights + b * a.w_b + h * a.w_h;
  const int32_t* pos = a.positions + b * a.p_b + h * a.p_h;
  float* wo = a.weights_out + b * a.wo_b + h * a.wo_h;
  int32_t* po = a.positions_out + b * a.po_b + h * a.po_h;
  if (!a.in_place)
    for (int i = threadIdx.x; i < min(n, a.budget); i += kSelectThreads) wo[i] = w[i], po[i] = pos[i];
  int32_t* count = a.counts + (int64_t)b * a.H_kv + h;
  if (n <= a.budget) {
    if (threadIdx.x == 0) *count = 0;
    return;
  }
  int32_t newest = INT32_MIN;
  for (int i = threadIdx.x; i < n; i += kSelectThreads) newest = max(newest, pos[i]);
  newest = __reduce_max_sync(0xffffffffu, newest);
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = newest;
  __syncthreads();
  newest = __reduce_max_sync(0xffffffffu, red[threadIdx.x & 31]);
  const int64_t from = (int64_t)newest - a.recent;  // positions above it are among the newest
  auto key = [&](int i) { return rank_key(w[i], pos[i] > from); };

  // the largest threshold that at least `budget` keys reach, bit by bit
  uint32_t least = 0;
  for (uint32_t bit = 0x80000000u; bit; bit >>= 1) {
    int reach = 0;
    for (int i = threadIdx.x; i < n; i += kSelectThreads) reach += key(i) >= (least | bit);
    if (block_sum(reach, red) >= a.budget) least |= bit;
  }
  // A warp owns a run of rows, 32 at a time, so that ranks within it are ballots.
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const uint32_t below = (1u << lane) - 1;
  const int per_warp = ((n + kSelectThreads - 1) / kSelectThreads) * 32;
  const int begin = min(warp * per_warp, n), end = min(begin + per_warp, n);
  int above = 0, equal = 0;
  for (int i0 = begin; i0 < end; i0 += 32) {
    const uint32_t k = i0 + lane < end ? key(i0 + lane) : 0;
    above += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k > least));
    equal += __popc(__ballot_sync(0xffffffffu, i0 + lane < end && k == least));
  }
  const int ties = a.budget - block_sum(lane == 0 ? above : 0, red);  // so many of the equal keys stay, the lowest rows
  const int equal_before = warps_before(equal, red);
  for (int pass = 0, holes = 0, movers = 0; pass < 2; ++pass) {
    int ties_seen = equal_before, hole_at = 0, mover_at = 0;
    if (pass) hole_at = warps_before(holes, red), mover_at = warps_before(movers, red);
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool in = i < end;
      const uint32_t k = in ? key(i) : 0;
      const uint32_t eq = __ballot_sync(0xffffffffu, in && k == least);
      const bool keep = in && (k > least || (k == least && ties_seen + __popc(eq & below) < ties));
      ties_seen += __popc(eq);
      const bool hole = in && !keep && i < a.budget, mover = keep && i >= a.budget;
      const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
      if (pass) {
        const int64_t list = ((int64_t)b * a.H_kv + h) * a.most_moves;
        if (hole) a.dst[list + hole_at + __popc(hb & below)] = i;
        if (mover) a.src[list + mover_at + __popc(mb & below)] = i;
        hole_at += __popc(hb), mover_at += __popc(mb);
      } else {
        holes += __popc(hb), movers += __popc(mb);
      }
    }
    if (pass == 0) {
      const int moves = block_sum(lane == 0 ? movers : 0, red);
      if (threadIdx.x == 0) *count = moves;
    }
  }
}

__device__ __forceinline__ void copy_row(char* to, const char* from, int bytes, int lane, bool aligned) {
  if (aligned) {
    if (lane * 16 < bytes) *reinterpret_cast<uint4*>(to + lane * 16) = *reinterpret_cast<const uint4*>(from + lane * 16);
    if ((lane + 32) * 16 < bytes) *reinterpret_cast<uint4*>(to + (lane + 32) * 16) = *reinterpret_cast<const uint4*>(from + (lane + 32) * 16);
  } else {
    for (int i = lane; i < bytes; i += 32) to[i] = from[i];
  }
}

// A warp moves a row at a time.
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const EvictArgs a) {
  const int32_t h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31;
  const int64_t bh = (int64_t)b * a.H_kv + h;
  // (in place, no other block reads the lengths any more: the rows come from the lists)
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lens_out[b * a.lens_out_b] = min(max(a.c.lens[b * a.c.lens_b], 0), a.budget);
  const int32_t moves = a.counts[bh];
  const int row_bytes = a.D * a.elsize;
  for (int32_t i = blockIdx.x * (kMoveThreads / 32) + (threadIdx.x >> 5); i < moves; i += gridDim.x * (kMoveThreads / 32)) {
    const int32_t src = a.src[bh * a.most_moves + i], dst = a.dst[bh * a.most_moves + i];
    int32_t sr, dr;
    const int32_t sp = a.c.locate(b, src, sr), dp = a.c.locate(b, dst, dr);
    if (lane == 0) {
      a.weights_out[b * a.wo_b + h * a.wo_h + dst] = a.weights[b * a.w_b + h * a.w_h + src];
      a.positions_out[b * a.po_b + h * a.po_h + dst] = a.positions[b * a.p_b + h * a.p_h + src];
    }
    if (sp < 0 || dp < 0) continue;
    const PagedView& c = a.c;
    copy_row(c.k + (dp * c.k_page + h * c.k_head + dr * c.k_row) * a.elsize, c.k + (sp * c.k_page + h * c.k_head + sr * c.k_row) * a.elsize,
             row_bytes, lane, a.aligned);
    copy_row(c.v + (dp * c.v_page + h * c.v_head + dr * c.v_row) * a.elsize, c.v + (sp * c.v_page + h * c.v_head + sr * c.v_row) * a.elsize,
             row_bytes, lane, a.aligned);
    if (c.k_scale && lane == 0) {
      c.k_scale[dp * c.ks_page + h * c.ks_head + dr * c.ks_row] = c.k_scale[sp * c.ks_page + h * c.ks_head + sr * c.ks_row];
      c.v_scale[dp * c.vs_page + h * c.vs_head + dr * c.vs_row] = c.v_scale[sp * c.vs_page + h * c.vs_head + sr * c.vs_row];
    }
  }
}

// Rows of a sequence that can move: kept ones behind the budget, into places before it.
int32_t most_moves(const kb_paged_cache& c, int32_t budget) {
  const int64_t capacity = (int64_t)c.M * c.page;
  return (int32_t)(capacity <= budget ? 0 : kb_min_i32(budget, (int32_t)(capacity - budget)));
}

}  // namespace

int paged_write(const kb_paged_write_params& p, cudaStream_t s) {
  const bool f8 = p.cache.dtype == KB_E4M3;
  if (!f8 && p.cache.dtype != p.dtype) return KB_ERR_UNSUPPORTED;
  const int64_t rows = (int64_t)p.cache.B * p.cache.H_kv * p.T;
  if (rows > (int64_t)1 << 30) return KB_ERR_TOO_LARGE;
  WriteArgs a{};
  a.c = make_paged_view(p.cache);
  const kb_tensor4* x[2] = {&p.k, &p.v};
  const int elsize = dtype_size(p.dtype);
  a.aligned = paged_rows_aligned(p.cache, dtype_size(p.cache.dtype));
  for (int i = 0; i < 2; ++i) {
    a.x[i] = x[i]->data;
    a.sb[i] = x[i]->stride[0], a.sh[i] = x[i]->stride[1], a.st[i] = x[i]->stride[2], a.sd[i] = x[i]->stride[3];
    a.aligned = a.aligned && a.sd[i] == 1 && reinterpret_cast<uintptr_t>(a.x[i]) % 16 == 0 && a.sb[i] * elsize % 16 == 0 && a.sh[i] * elsize % 16 == 0 &&
                a.st[i] * elsize % 16 == 0;
  }
  a.new_lens = p.new_lens, a.new_lens_b = p.new_lens_stride;
  a.positions = p.positions, a.pos_b = p.positions_stride[0], a.pos_t = p.positions_stride[1];
  a.weights = p.weights, a.w_b = p.weights_stride[0], a.w_h = p.weights_stride[1];
  a.row_positions = p.row_positions, a.p_b = p.row_positions_stride[0], a.p_h = p.row_positions_stride[1];
  a.B = p.cache.B, a.H_kv = p.cache.H_kv, a.T = p.T, a.D = p.cache.D;
  a.rows_per_cta = kWriteThreads / (a.D / kPerThread);
  a.fd_T = kb_fastdiv_make(a.T), a.fd_H = kb_fastdiv_make(a.H_kv);
  switch (p.dtype) {
    case KB_F32: return launch_write<float>(a, f8, s);
    case KB_F16: return launch_write<__half>(a, f8, s);
    default: return launch_write<__nv_bfloat16>(a, f8, s);
  }
}

size_t paged_evict_workspace_bytes(const kb_paged_cache& c, int32_t budget) {
  return ((size_t)c.B * c.H_kv * (1 + 2 * (size_t)most_moves(c, budget))) * sizeof(int32_t);
}

int paged_evict(const kb_paged_evict_params& p, cudaStream_t s) {
  const kb_paged_cache& c = p.cache;
  EvictArgs a{};
  a.c = make_paged_view(c);
  a.weights = p.weights, a.w_b = p.weights_stride[0], a.w_h = p.weights_stride[1];
  a.positions = p.row_positions, a.p_b = p.row_positions_stride[0], a.p_h = p.row_positions_stride[1];
  a.weights_out = p.weights_out, a.wo_b = p.weights_out_stride[0], a.wo_h = p.weights_out_stride[1];
  a.positions_out = p.row_positions_out, a.po_b = p.row_positions_out_stride[0], a.po_h = p.row_positions_out_stride[1];
  a.lens_out = p.lens_out, a.lens_out_b = p.lens_out_stride;
  a.H_kv = c.H_kv, a.D = c.D, a.budget = p.budget, a.recent = p.recent;
  a.most_moves = most_moves(c, p.budget);
  a.elsize = dtype_size(c.dtype);
  a.aligned = paged_rows_aligned(c, a.elsize);
  a.in_place = p.weights == p.weights_out;
  const size_t heads = (size_t)c.B * c.H_kv;
  a.counts = static_cast<int32_t*>(p.workspace);
  a.src = a.counts + heads;
  a.dst = a.src + heads * a.most_moves;
  paged_select_kernel<<<dim3((unsigned)c.H_kv, (unsigned)c.B), kSelectThreads, 0, s>>>(a);
  KB_LAUNCH_CHECK("paged_select_kernel");
  // eight rows per block at a time; a few blocks per head are enough where there are many heads
  const int64_t most = ((int64_t)a.most_moves + 7) / 8, want = kb_max_i32(1, (int32_t)((148 * 16 + heads - 1) / heads));
  paged_move_kernel<<<dim3((unsigned)(most < want ? (most < 1 ? 1 : most) : want), (unsigned)c.H_kv, (unsigned)c.B), kMoveThreads, 0, s>>>(a);
  KB_LAUNCH_CHECK("paged_move_kernel");
  return KB_OK;
}

}  // namespace kb
