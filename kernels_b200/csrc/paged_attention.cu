// Attention of one new token per sequence over a paged key/value cache: o = softmax(q k^T scale) v over the rows that the
// token sees, its log-sum-exp, and on request every row's weight added to a running sum.
//
// HBM-bound: two FLOPs per byte and query head; all that counts is to read every cached row once, at full rate.  The query
// heads that share a key/value head are therefore worked on together, and the rows of a sequence are split over so
// many blocks that the GPU is full even for one sequence.  A block keeps, per head, the running maximum, the sum and the
// unnormalised output (all fp32), and a second kernel joins the blocks of a head in their order:
//   m = max m_s,  l = sum l_s 2^(m_s - m),  o = sum o_s 2^(m_s - m) / l.
// Rows' weights need the final m and l, so the scores go to the workspace (4 bytes per row and query head, against
// 2 D elements per row and key/value head read) and a third kernel turns them into weights and adds them up: every sum has one
// writer, so results do not depend on the order of anything.
//
// Generic kernel (this file): CUDA cores, every type, head dim and alignment.  A row is a few neighbouring lanes, 16 bytes
// each; a group of lanes has a softmax of its own, joined at the end of the block.
#include <cuda_fp8.h>

#include "common.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

namespace kb {
namespace {

constexpr int kThreads = 128, kWarps = kThreads / 32;

struct AttendArgs {
  PagedView c;
  const void* q;
  int64_t q_b, q_h, q_d;
  void* o;
  float* lse;
  float* weights;
  int64_t w_b, w_h;
  int32_t dtype, B, H, H_kv, D, group;   // group: query heads per key/value head
  int32_t head_tiles;                    // blocks per group
  int32_t context, back;                 // context 0: every row is seen
  int32_t splits;
  float scale_log2;
  float* part_o;    // [B, H, splits, D]
  float2* part_ml;  // [B, H, splits]
  float* scores;    // [B, H, capacity], base-2 logits
  KbFastDiv fd_context;
};

// The rows that the token sees: [first, end).
__device__ __forceinline__ void seen_rows(const AttendArgs& a, int32_t b, int32_t& first, int32_t& end) {
  end = a.c.rows(b);
  first = 0;
  if (a.context && end > 0) first = kb_max_i32(0, kb_fastdiv(end - 1, a.fd_context) - a.back) * a.context;
}

// Part `split` of them, in whole tiles.
__device__ __forceinline__ void split_rows(const AttendArgs& a, int32_t split, int32_t tile, int32_t& first, int32_t& end) {
  const int32_t tiles = kb_cdiv_i32(end - first, tile), each = kb_cdiv_i32(tiles, a.splits);
  const int64_t from = (int64_t)first + (int64_t)split * each * tile, to = from + (int64_t)each * tile;
  first = from < end ? (int32_t)from : end;
  end = to < end ? (int32_t)to : end;
}

__device__ __forceinline__ float load_any(const void* p, int64_t i, int32_t dtype) {
  if (dtype == KB_F32) return static_cast<const float*>(p)[i];
  if (dtype == KB_F16) return __half2float(static_cast<const __half*>(p)[i]);
  return __bfloat162float(static_cast<const __nv_bfloat16*>(p)[i]);
}
__device__ __forceinline__ void store_any(void* p, int64_t i, int32_t dtype, float x) {
  if (dtype == KB_F32) static_cast<float*>(p)[i] = x;
  else if (dtype == KB_F16) static_cast<__half*>(p)[i] = __float2half_rn(x);
  else static_cast<__nv_bfloat16*>(p)[i] = __float2bfloat16_rn(x);
}

// ---- generic kernel --------------------------------------------------------------------------------------------------

template <typename T, int N>
struct RowPart {
  float f[N];
  __device__ __forceinline__ void load(const T* p, bool aligned) {
    if (aligned && N * sizeof(T) % 16 == 0) {
      T e[N];
#pragma unroll
      for (int i = 0; i < (int)(N * sizeof(T)) / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_f32(e[i]);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) f[i] = to_f32(p[i]);
    }
  }
};
template <int N>
struct RowPart<uint8_t, N> {  // e4m3
  float f[N];
  __device__ __forceinline__ void load(const uint8_t* p, bool aligned) {
    uint8_t e[N];
    if (aligned && N % 16 == 0) {
#pragma unroll
      for (int i = 0; i < N / 16; ++i) reinterpret_cast<uint4*>(e)[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) e[i] = p[i];
    }
#pragma unroll
    for (int i = 0; i < N; ++i) {
      __half_raw r = __nv_cvt_fp8_to_halfraw(e[i], __NV_E4M3);
      f[i] = __half2float(__half(r));
    }
  }
};

// T: the cache's elements (uint8_t: e4m3); G: query heads per block
template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads) paged_attend_kernel(const AttendArgs a, bool aligned) {
  constexpr int kLanes = D * (int)sizeof(T) / 16 < 1 ? 1 : D * (int)sizeof(T) / 16 > 32 ? 32 : D * (int)sizeof(T) / 16;  // per row
  constexpr int N = D / kLanes;                     // elements per lane
  constexpr int kRows = 32 / kLanes;                // rows of a warp at a time
  constexpr int kTile = kWarps * kRows;
  __shared__ float q_s[G][D];
  __shared__ float m_s[kWarps][G], l_s[kWarps][G], o_s[kWarps][G][D];
  const int32_t split = blockIdx.x, hk = blockIdx.y / a.head_tiles, b = blockIdx.z;
  const int32_t h0 = hk * a.group + (blockIdx.y - hk * a.head_tiles) * G, heads = min(G, (hk + 1) * a.group - h0);
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kLanes, part = lane % kLanes;
  int32_t first, end;
  seen_rows(a, b, first, end);
  split_rows(a, split, kTile, first, end);

  for (int i = threadIdx.x; i < G * D; i += kThreads) {
    const int g = i / D, d = i % D;
    q_s[g][d] = g < heads ? load_any(a.q, b * a.q_b + (h0 + g) * a.q_h + d * a.q_d, a.dtype) * a.scale_log2 : 0.f;
  }
  __syncthreads();
  float q[G][N], o[G][N], m[G], l[G];
#pragma unroll
  for (int g = 0; g < G; ++g) {
    m[g] = -INFINITY, l[g] = 0.f;
#pragma unroll
    for (int i = 0; i < N; ++i) q[g][i] = q_s[g][part * N + i], o[g][i] = 0.f;
  }
  for (int32_t r0 = first; r0 < end; r0 += kTile) {
    const int32_t r = r0 + warp * kRows + sub;
    int32_t at = 0, page = -1;
    if (r < end) page = a.c.locate(b, r, at);
    const bool live = page >= 0;
    RowPart<T, N> k, v;
    float ks = 1.f, vs = 1.f;
    if (live) {
      k.load(reinterpret_cast<const T*>(a.c.k) + page * a.c.k_page + hk * a.c.k_head + at * a.c.k_row + part * N, aligned);
      v.load(reinterpret_cast<const T*>(a.c.v) + page * a.c.v_page + hk * a.c.v_head + at * a.c.v_row + part * N, aligned);
      if (sizeof(T) == 1) {
        ks = a.c.k_scale[page * a.c.ks_page + hk * a.c.ks_head + at * a.c.ks_row];
        vs = a.c.v_scale[page * a.c.vs_page + hk * a.c.vs_head + at * a.c.vs_row];
      }
    } else {
#pragma unroll
      for (int i = 0; i < N; ++i) k.f[i] = 0.f, v.f[i] = 0.f;
    }
#pragma unroll
    for (int g = 0; g < G; ++g) {
      float s = 0.f;
#pragma unroll
      for (int i = 0; i < N; ++i) s = fmaf(q[g][i], k.f[i], s);
#pragma unroll
      for (int x = kLanes / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
      s = live ? s * ks : -INFINITY;
      if (a.scores && part == 0 && r < end && g < heads) a.scores[((int64_t)b * a.H + h0 + g) * a.c.capacity + r] = s;
      const float top = fmaxf(m[g], s), base = top == -INFINITY ? 0.f : top;
      const float p = live ? exp2f(s - base) : 0.f, keep = exp2f(m[g] - base);
      m[g] = top;
      l[g] = l[g] * keep + p;
      const float pv = p * vs;
#pragma unroll
      for (int i = 0; i < N; ++i) o[g][i] = fmaf(pv, v.f[i], o[g][i] * keep);
    }
  }
  // the lane groups of a warp, then the warps
#pragma unroll
  for (int g = 0; g < G; ++g) {
    float top = m[g];
#pragma unroll
    for (int x = kLanes; x < 32; x <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
    const float keep = exp2f(m[g] - (top == -INFINITY ? 0.f : top));
    float sum = l[g] * keep;
#pragma unroll
    for (int x = kLanes; x < 32; x <<= 1) sum += __shfl_xor_sync(0xffffffffu, sum, x);
    if (lane == 0) m_s[warp][g] = top, l_s[warp][g] = sum;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      float x = o[g][i] * keep;
#pragma unroll
      for (int y = kLanes; y < 32; y <<= 1) x += __shfl_xor_sync(0xffffffffu, x, y);
      if (sub == 0) o_s[warp][g][part * N + i] = x;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * D; i += kThreads) {
    const int g = i / D, d = i % D;
    float top = m_s[0][g];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][g]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float keep = exp2f(m_s[w][g] - base);
      sum += l_s[w][g] * keep;
      x += o_s[w][g][d] * keep;
    }
    const int64_t bh = (int64_t)b * a.H + h0 + g;
    if (a.splits == 1) {
      store_any(a.o, bh * D + d, a.dtype, sum == 0.f ? 0.f : x / sum);
      if (a.lse && d == 0) a.lse[bh] = sum == 0.f ? 0.f : base + log2f(sum);
    } else {
      a.part_o[(bh * a.splits + split) * D + d] = x;
      if (d == 0) a.part_ml[bh * a.splits + split] = make_float2(top, sum);
    }
  }
}

// ---- the parts of a head joined ------------------------------------------------------------------------------------------

__global__ void paged_join_kernel(const AttendArgs a) {
  const int64_t bh = blockIdx.x;
  const int d = threadIdx.x;
  const float2* ml = a.part_ml + bh * a.splits;
  float top = -INFINITY;
  for (int s = 0; s < a.splits; ++s) top = fmaxf(top, ml[s].x);
  const float base = top == -INFINITY ? 0.f : top;
  float sum = 0.f, x = 0.f;
  for (int s = 0; s < a.splits; ++s) {
    const float keep = exp2f(ml[s].x - base);
    sum += ml[s].y * keep;
    x += a.part_o[(bh * a.splits + s) * a.D + d] * keep;
  }
  store_any(a.o, bh * a.D + d, a.dtype, sum == 0.f ? 0.f : x / sum);
  if (a.lse && d == 0) a.lse[bh] = sum == 0.f ? 0.f : base + log2f(sum);
}

// ---- rows' weights -------------------------------------------------------------------------------------------------------

__global__ void __launch_bounds__(256) paged_weigh_kernel(const AttendArgs a) {
  const int32_t hk = blockIdx.y, b = blockIdx.z;
  int32_t first, end;
  seen_rows(a, b, first, end);
  for (int64_t r = (int64_t)first + blockIdx.x * 256 + threadIdx.x; r < end; r += (int64_t)gridDim.x * 256) {
    float w = 0.f;
    for (int g = 0; g < a.group; ++g) {
      const int64_t bh = (int64_t)b * a.H + hk * a.group + g;
      w += exp2f(a.scores[bh * a.c.capacity + r] - a.lse[bh]);
    }
    a.weights[b * a.w_b + hk * a.w_h + r] += w;
  }
}

template <typename T, int D>
int launch_heads(AttendArgs& a, bool aligned, cudaStream_t s) {
  if (a.group == 1) {
    a.head_tiles = 1;
    paged_attend_kernel<T, D, 1><<<dim3(a.splits, a.H_kv, a.B), kThreads, 0, s>>>(a, aligned);
  } else {
    a.head_tiles = (a.group + 3) / 4;
    paged_attend_kernel<T, D, 4><<<dim3(a.splits, a.H_kv * a.head_tiles, a.B), kThreads, 0, s>>>(a, aligned);
  }
  KB_LAUNCH_CHECK("paged_attend_kernel");
  return KB_OK;
}

template <typename T>
int launch_dim(AttendArgs& a, bool aligned, cudaStream_t s) {
  switch (a.D) {
    case 16: return launch_heads<T, 16>(a, aligned, s);
    case 32: return launch_heads<T, 32>(a, aligned, s);
    case 64: return launch_heads<T, 64>(a, aligned, s);
    case 128: return launch_heads<T, 128>(a, aligned, s);
    default: return launch_heads<T, 256>(a, aligned, s);
  }
}

// Rows that a token can see at most, from sizes alone: the lengths are on the device.
int32_t most_rows(const kb_paged_attention_params& p) {
  const int64_t capacity = (int64_t)p.cache.M * p.cache.page;
  const int64_t window = p.context_size > 0 ? ((int64_t)p.back_contexts + 1) * p.context_size : capacity;
  return (int32_t)(window < capacity ? window : capacity);
}

// Blocks per head: as many as fill the GPU a few times over, none shorter than 256 rows.
int32_t split_count(const kb_paged_attention_params& p) {
  const int64_t items = (int64_t)p.cache.B * p.cache.H_kv;
  const int64_t fill = (148 * 8 + items - 1) / items, most = kb_cdiv_i32(most_rows(p), 256);
  return (int32_t)(fill < most ? fill : most < 1 ? 1 : most);
}

}  // namespace

size_t paged_attention_workspace_bytes(const kb_paged_attention_params& p) {
  const size_t heads = (size_t)p.cache.B * p.H, splits = split_count(p);
  size_t n = splits > 1 ? heads * splits * (p.cache.D + 2) : 0;
  if (p.weights) n += heads * p.cache.M * p.cache.page;
  return n * sizeof(float);
}

int paged_attention(const kb_paged_attention_params& p, cudaStream_t s) {
  const kb_paged_cache& c = p.cache;
  AttendArgs a{};
  a.c = make_paged_view(c);
  a.q = p.q, a.q_b = p.q_stride[0], a.q_h = p.q_stride[1], a.q_d = p.q_stride[2];
  a.o = p.o, a.lse = p.lse;
  a.weights = p.weights, a.w_b = p.weights_stride[0], a.w_h = p.weights_stride[1];
  a.dtype = p.dtype, a.B = c.B, a.H = p.H, a.H_kv = c.H_kv, a.D = c.D, a.group = p.H / c.H_kv;
  if (p.context_size > 0) {
    a.context = kb_clamp_context(p.context_size, a.c.capacity);
    a.back = kb_clamp_back(p.back_contexts, a.c.capacity, a.context);
    a.fd_context = kb_fastdiv_make(a.context);
  }
  a.splits = split_count(p);
  a.scale_log2 = p.sm_scale * kLog2e;
  float* w = static_cast<float*>(p.workspace);
  const size_t heads = (size_t)c.B * p.H;
  if (a.splits > 1) {
    a.part_ml = reinterpret_cast<float2*>(w);
    a.part_o = w + heads * a.splits * 2;
    w = a.part_o + heads * a.splits * c.D;
  }
  if (p.weights) a.scores = w;
  const bool aligned = paged_rows_aligned(c, dtype_size(c.dtype));
  int rc;
  switch (c.dtype) {
    case KB_F32: rc = launch_dim<float>(a, aligned, s); break;
    case KB_F16: rc = launch_dim<__half>(a, aligned, s); break;
    case KB_BF16: rc = launch_dim<__nv_bfloat16>(a, aligned, s); break;
    default: rc = launch_dim<uint8_t>(a, aligned, s); break;
  }
  if (rc) return rc;
  if (a.splits > 1) {
    paged_join_kernel<<<(unsigned)heads, a.D, 0, s>>>(a);
    KB_LAUNCH_CHECK("paged_join_kernel");
  }
  if (p.weights) {
    const int32_t blocks = kb_cdiv_i32(most_rows(p), 256), fill = kb_max_i32(1, 148 * 16 / kb_max_i32(1, c.B * c.H_kv));
    paged_weigh_kernel<<<dim3(blocks < fill ? kb_max_i32(1, blocks) : fill, c.H_kv, c.B), 256, 0, s>>>(a);
    KB_LAUNCH_CHECK("paged_weigh_kernel");
  }
  return KB_OK;
}

}  // namespace kb
