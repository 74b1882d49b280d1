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
#include "sm100_host.h"
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

// ---- tensor-core kernel ----------------------------------------------------------------------------------------------
//
// 16-bit and e4m3 caches of head dim 64 and 128.  A warp multiplies the 16 (or 8) query heads of a block with 16 keys at a time
// (m16n8k16): the heads are the rows, so up to 16 heads cost what one does, and what the tensor cores have to do is a
// small part of the time that the keys take to arrive.  That time is all there is to hide, and every warp hides it for itself: it
// has tiles of kR rows of its own (every fourth of the block's), a ring of kStages of them in shared memory filled by
// 16-byte asynchronous copies, and a softmax of its own, so that no warp waits for another before the end.
//
// Rows are found one by one (a lane looks up a row), so pages of any size and order are read the same way; a row that is
// masked is filled with zeros without being read, so that nothing in it can reach a sum.
//
// e4m3 elements become f16, exactly.  q does too (bf16 q after a multiplication by a power of two that brings its largest element to
// 2^14: what is lost lies 2^-38 below the largest).  A row's value scale belongs to its weight: the weights that are
// multiplied are p * v_scale, so the running maximum is taken over score + log2(v_scale), which keeps them within f16.
// f16 weights start at 2^7 and may grow to 2^15 before sums are rescaled: seven bits more for the small ones.
// Weights are rounded to 16 bits for the product with V (as in the operator's forward kernel); their sum is taken before that.

__device__ __forceinline__ void cp_async16(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(to), "l"(from), "r"(live ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t to, const void* from, bool live) {
  asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(to), "l"(from), "r"(live ? 4 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N>
__device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }

__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
// c += a b, 16 x 8 x 16; with HALF the rows 8 .. 15 are not there
template <bool BF16, bool HALF>
__device__ __forceinline__ void mma16(float (&c)[HALF ? 2 : 4], const uint32_t (&a)[HALF ? 2 : 4], uint32_t b0, uint32_t b1) {
  float x2, x3;
  if constexpr (HALF) {
    if constexpr (BF16)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %8, %5, %8}, {%6, %7}, {%0, %1, %9, %9};"
          : "+f"(c[0]), "+f"(c[1]), "=f"(x2), "=f"(x3) : "r"(a[0]), "r"(a[1]), "r"(b0), "r"(b1), "r"(0), "f"(0.f));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %8, %5, %8}, {%6, %7}, {%0, %1, %9, %9};"
          : "+f"(c[0]), "+f"(c[1]), "=f"(x2), "=f"(x3) : "r"(a[0]), "r"(a[1]), "r"(b0), "r"(b1), "r"(0), "f"(0.f));
  } else {
    if constexpr (BF16)
      asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
    else
      asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
          : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
  }
}
__device__ __forceinline__ uint32_t e4m3x2_to_f16x2(uint32_t two) {
  uint32_t r;
  asm("{\n\t.reg .b16 x;\n\tcvt.u16.u32 x, %1;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\t}" : "=r"(r) : "r"(two));
  return r;
}

// kF8: e4m3 cache (products in f16); kBf16: products in bf16, otherwise in f16; kHalf: at most eight query heads per block
template <bool kF8, bool kBf16, int kD, bool kHalf>
struct MmaTile {
  static constexpr int kRowBytes = kF8 ? kD : 2 * kD, kChunks = kRowBytes / 16;
  static constexpr int kR = kRowBytes == 256 ? 16 : 32;            // rows of a tile
  static constexpr int kStages = kRowBytes == 64 ? 4 : 3;
  static constexpr int kScaleBytes = kF8 ? 2 * kR * 4 : 0;
  static constexpr int kStageBytes = 2 * kR * kRowBytes + kScaleBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kHeads = kHalf ? 8 : 16, kS = kHalf ? 1 : 2; // kS: heads per thread
  static constexpr int kSmem = kWarps * kWarpBytes;
  // Where chunk c of row r lies: at c ^ swizzle(r).  The eight rows of a matrix load hit different banks, and so do the two rows
  // and four chunks of a 16-byte load of e4m3 keys.
  static __device__ __forceinline__ int swizzle(int r) { return !kF8 ? r & 7 : kD == 128 ? ((r & 1) << 2) | ((r >> 1) & 3) : (r >> 1) & 3; }
  static_assert(kSmem >= kWarps * kHeads * kD * 4, "the warps' outputs are joined where the ring was");
};

template <bool kF8, bool kBf16, int kD, bool kHalf>
__global__ void __launch_bounds__(kThreads) paged_attend_mma_kernel(const AttendArgs a) {
  using Tile = MmaTile<kF8, kBf16, kD, kHalf>;
  constexpr int kR = Tile::kR, kStages = Tile::kStages, kChunks = Tile::kChunks, kRowBytes = Tile::kRowBytes, kHeads = Tile::kHeads, kS = Tile::kS;
  constexpr int kSteps = kD / 16, kNt = kR / 8, kDt = kD / 8, kA = 2 * kS;
  constexpr float kOffset = kBf16 ? 0.f : 7.f, kSlack = 8.f;
  extern __shared__ __align__(128) uint8_t smem[];
  __shared__ float m_s[kWarps][16], l_s[kWarps][16];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, oct = lane >> 2;
  const int32_t split = blockIdx.x, hk = blockIdx.y / a.head_tiles, b = blockIdx.z;
  const int32_t h0 = hk * a.group + (blockIdx.y - hk * a.head_tiles) * kHeads, heads = min(kHeads, (hk + 1) * a.group - h0);
  int32_t first, end;
  seen_rows(a, b, first, end);
  split_rows(a, split, kWarps * kR, first, end);
  const uint32_t ring = sm100::smem_u32(smem) + warp * Tile::kWarpBytes;

  // ---- copies: lane r looks up row r of the tile
  const char* kbase = a.c.k + hk * a.c.k_head * (kF8 ? 1 : 2);
  const char* vbase = a.c.v + hk * a.c.v_head * (kF8 ? 1 : 2);
  constexpr uint32_t kNoRow = 0xffffffffu;
  int32_t next_row = first + warp * kR + (lane & (kR - 1));  // the row that this lane looks up next
  uint32_t live_bits[kStages - 1];                           // of the tiles in the ring, oldest first
  auto issue = [&](int stage) -> uint32_t {
    uint32_t at16 = kNoRow;
    int32_t at = 0, page = -1;
    if (next_row < end) page = a.c.locate(b, next_row, at);
    if (page >= 0) at16 = (uint32_t)((uint64_t)((page * a.c.k_page + at * a.c.k_row) * (kF8 ? 1 : 2)) >> 4);
    const uint32_t live = __ballot_sync(0xffffffffu, page >= 0);
    const uint32_t to = ring + stage * Tile::kStageBytes;
    constexpr int kRowsAtOnce = 32 / kChunks;
    const int chunk = lane % kChunks, sub = lane / kChunks;
#pragma unroll
    for (int i = 0; i < kR / kRowsAtOnce; ++i) {
      const int r = i * kRowsAtOnce + sub;
      const uint32_t row16 = __shfl_sync(0xffffffffu, at16, r);
      const bool ok = row16 != kNoRow;
      const uint64_t off = ok ? ((uint64_t)row16 + chunk) * 16 : 0;
      const uint32_t place = r * kRowBytes + ((chunk ^ Tile::swizzle(r)) * 16);
      cp_async16(to + place, kbase + off, ok);
      cp_async16(to + kR * kRowBytes + place, vbase + off, ok);
    }
    if constexpr (kF8) {
      const int64_t so = page >= 0 ? page * a.c.ks_page + hk * a.c.ks_head + at * a.c.ks_row : 0;
      cp_async4(to + 2 * kR * kRowBytes + lane * 4, a.c.k_scale + so, page >= 0);
      cp_async4(to + 2 * kR * kRowBytes + kR * 4 + lane * 4, a.c.v_scale + so, page >= 0);
    }
    next_row += kWarps * kR;
    return live;
  };
  // (tiles behind the last are empty: nothing is read)
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    live_bits[s] = issue(s);
    cp_async_commit();
  }

  // ---- q as the products' left operand; with an e4m3 cache a lane's elements are the ones its 16-byte key loads hold
  uint32_t q[kSteps][kA];
  float back_scale[kS];
#pragma unroll
  for (int s = 0; s < kS; ++s) {
    const int g = oct + 8 * s;
    const bool there = g < heads;
    const int64_t base = b * a.q_b + (int64_t)(h0 + (there ? g : 0)) * a.q_h;
    float up = 1.f;
    back_scale[s] = a.scale_log2;
    if (kF8 && a.dtype == KB_BF16) {
      float top = 0.f;
      for (int d = quad; d < kD; d += 4) top = fmaxf(top, there ? fabsf(load_any(a.q, base + d * a.q_d, a.dtype)) : 0.f);
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 1));
      top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, 2));
      const int e = (int)(__float_as_uint(top) >> 23) - 127;  // top in [2^e, 2^(e+1))
      if (top > 0.f && e < 128) {
        const int by = max(-100, min(100, 14 - e));
        up = __uint_as_float((uint32_t)(by + 127) << 23);
        back_scale[s] *= __uint_as_float((uint32_t)(127 - by) << 23);
      }
    }
#pragma unroll
    for (int t = 0; t < kSteps; ++t)
#pragma unroll
      for (int p = 0; p < 2; ++p) {
        const int d = kF8 ? t / 4 * 64 + quad * 16 + t % 4 * 4 + 2 * p : t * 16 + 8 * p + quad * 2;
        const float x = there ? load_any(a.q, base + d * a.q_d, a.dtype) * up : 0.f;
        const float y = there ? load_any(a.q, base + (d + 1) * a.q_d, a.dtype) * up : 0.f;
        q[t][p * kS + s] = sm100::pack16x2<kBf16>(x, y);
      }
  }

  float o[kDt][kA], m[kS], l[kS];
#pragma unroll
  for (int s = 0; s < kS; ++s) m[s] = -INFINITY, l[s] = 0.f;
#pragma unroll
  for (int j = 0; j < kDt; ++j)
#pragma unroll
    for (int i = 0; i < kA; ++i) o[j][i] = 0.f;

  int stage = 0;
  for (int32_t r0 = first + warp * kR; r0 < end; r0 += kWarps * kR) {
    cp_async_wait<kStages - 2>();
    __syncwarp();
    const uint32_t at = ring + stage * Tile::kStageBytes, vat = at + kR * kRowBytes;
    const uint32_t live = live_bits[0];
    // every lane is through with the tile before this one: the next copies take its place
#pragma unroll
    for (int s = 0; s < kStages - 2; ++s) live_bits[s] = live_bits[s + 1];
    live_bits[kStages - 2] = issue(stage == 0 ? kStages - 1 : stage - 1);
    cp_async_commit();

    // scores
    float sc[kNt][kA];
#pragma unroll
    for (int j = 0; j < kNt; ++j)
#pragma unroll
      for (int i = 0; i < kA; ++i) sc[j][i] = 0.f;
    if constexpr (!kF8) {
#pragma unroll
      for (int t = 0; t < kSteps; ++t)
#pragma unroll
        for (int j = 0; j < kNt; j += 2) {
          const int key = j * 8 + (lane & 7) + (lane >> 4) * 8, chunk = t * 2 + ((lane >> 3) & 1);
          uint32_t r[4];
          ldsm4(r, at + key * kRowBytes + ((chunk ^ Tile::swizzle(key)) * 16));
          mma16<kBf16, kHalf>(sc[j], q[t], r[0], r[1]);
          mma16<kBf16, kHalf>(sc[j + 1], q[t], r[2], r[3]);
        }
    } else {
#pragma unroll
      for (int t4 = 0; t4 < kSteps / 4; ++t4)
#pragma unroll
        for (int j = 0; j < kNt; ++j) {
          const int key = j * 8 + oct, chunk = t4 * 4 + quad;
          uint32_t r[4];
          asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
                       : "r"(at + key * kRowBytes + ((chunk ^ Tile::swizzle(key)) * 16)) : "memory");
#pragma unroll
          for (int t = 0; t < 4; ++t) mma16<kBf16, kHalf>(sc[j], q[t4 * 4 + t], e4m3x2_to_f16x2(r[t]), e4m3x2_to_f16x2(r[t] >> 16));
        }
    }
    // base-2 logits; what a row's value scale adds to the maximum
    float top[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) top[s] = -INFINITY;
    float vs[kF8 ? kNt : 1][2];
#pragma unroll
    for (int j = 0; j < kNt; ++j) {
      float ks[2] = {1.f, 1.f}, lift[2] = {0.f, 0.f};
      if constexpr (kF8) {
        const uint32_t sa = at + 2 * kR * kRowBytes + (j * 8 + quad * 2) * 4;
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(ks[0]), "=f"(ks[1]) : "r"(sa) : "memory");
        asm volatile("ld.shared.v2.f32 {%0, %1}, [%2];" : "=f"(vs[j][0]), "=f"(vs[j][1]) : "r"(sa + kR * 4) : "memory");
#pragma unroll
        for (int i = 0; i < 2; ++i) lift[i] = __log2f(fmaxf(fabsf(vs[j][i]), 7.9e-31f));  // 2^-100: no lower, or the sum of the weights leaves fp32
      }
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
          float x = sc[j][2 * s + i] * back_scale[s];
          if (kF8) x *= ks[i];
          sc[j][2 * s + i] = x;
        }
      if (live != 0xffffffffu) {
#pragma unroll
        for (int i = 0; i < 2; ++i)
          if (!((live >> (j * 8 + quad * 2 + i)) & 1)) {
#pragma unroll
            for (int s = 0; s < kS; ++s) sc[j][2 * s + i] = -INFINITY;
          }
      }
#pragma unroll
      for (int s = 0; s < kS; ++s)
#pragma unroll
        for (int i = 0; i < 2; ++i) top[s] = fmaxf(top[s], kF8 ? sc[j][2 * s + i] + lift[i] : sc[j][2 * s + i]);
    }
    if (a.scores) {
#pragma unroll
      for (int s = 0; s < kS; ++s)
        if (oct + 8 * s < heads) {
          float* out = a.scores + ((int64_t)b * a.H + h0 + oct + 8 * s) * a.c.capacity + r0 + quad * 2;
#pragma unroll
          for (int j = 0; j < kNt; ++j)
#pragma unroll
            for (int i = 0; i < 2; ++i)
              if (r0 + j * 8 + quad * 2 + i < end) out[j * 8 + i] = sc[j][2 * s + i];
        }
    }
    bool raise = false;
#pragma unroll
    for (int s = 0; s < kS; ++s) {
      top[s] = fmaxf(top[s], __shfl_xor_sync(0xffffffffu, top[s], 1));
      top[s] = fmaxf(top[s], __shfl_xor_sync(0xffffffffu, top[s], 2));
      raise = raise || top[s] > m[s] + kSlack;
    }
    if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
      for (int s = 0; s < kS; ++s) {
        const float to = fmaxf(m[s], top[s]);
        const float keep = to == -INFINITY ? 0.f : sm100::ex2_approx(m[s] - to);
        m[s] = to;
        l[s] *= keep;
#pragma unroll
        for (int j = 0; j < kDt; ++j) o[j][2 * s] *= keep, o[j][2 * s + 1] *= keep;
      }
    }
    float base[kS];
#pragma unroll
    for (int s = 0; s < kS; ++s) base[s] = m[s] == -INFINITY ? 0.f : m[s] - kOffset;
    // weights and their products with V, 16 keys at a time
#pragma unroll
    for (int j = 0; j < kNt; j += 2) {
      uint32_t p[kA];
#pragma unroll
      for (int u = 0; u < 2; ++u)
#pragma unroll
        for (int s = 0; s < kS; ++s) {
          float x = sm100::ex2_approx(sc[j + u][2 * s] - base[s]), y = sm100::ex2_approx(sc[j + u][2 * s + 1] - base[s]);
          l[s] += x + y;
          if constexpr (kF8) x *= vs[j + u][0], y *= vs[j + u][1];
          p[u * kS + s] = sm100::pack16x2<kBf16>(x, y);
        }
      const int key = j * 8 + (lane & 15);
      if constexpr (!kF8) {
#pragma unroll
        for (int d = 0; d < kDt; d += 2) {
          uint32_t r[4];
          ldsm4_t(r, vat + key * kRowBytes + (((d + (lane >> 4)) ^ Tile::swizzle(key)) * 16));
          mma16<kBf16, kHalf>(o[d], p, r[0], r[1]);
          mma16<kBf16, kHalf>(o[d + 1], p, r[2], r[3]);
        }
      } else {
        // a 16-bit column of the transposed load is a pair of neighbouring elements; they go to products of their own
#pragma unroll
        for (int d = 0; d < kDt; d += 4) {
          uint32_t r[4];
          ldsm4_t(r, vat + key * kRowBytes + (((d / 2 + (lane >> 4)) ^ Tile::swizzle(key)) * 16));
#pragma unroll
          for (int c = 0; c < 2; ++c) {
            const uint32_t lo0 = e4m3x2_to_f16x2(r[2 * c]), lo1 = e4m3x2_to_f16x2(r[2 * c] >> 16);
            const uint32_t hi0 = e4m3x2_to_f16x2(r[2 * c + 1]), hi1 = e4m3x2_to_f16x2(r[2 * c + 1] >> 16);
            mma16<kBf16, kHalf>(o[d + 2 * c], p, __byte_perm(lo0, lo1, 0x5410), __byte_perm(hi0, hi1, 0x5410));
            mma16<kBf16, kHalf>(o[d + 2 * c + 1], p, __byte_perm(lo0, lo1, 0x7632), __byte_perm(hi0, hi1, 0x7632));
          }
        }
      }
    }
    stage = stage == kStages - 1 ? 0 : stage + 1;
  }
  cp_async_wait<0>();
  __syncthreads();

  // ---- the warps joined; element i of thread (oct, quad) of output tile j
#pragma unroll
  for (int s = 0; s < kS; ++s) {
    l[s] += __shfl_xor_sync(0xffffffffu, l[s], 1);
    l[s] += __shfl_xor_sync(0xffffffffu, l[s], 2);
    if (quad == 0) m_s[warp][oct + 8 * s] = m[s], l_s[warp][oct + 8 * s] = l[s];
  }
  float* o_s = reinterpret_cast<float*>(smem) + warp * kHeads * kD;
#pragma unroll
  for (int j = 0; j < kDt; ++j)
#pragma unroll
    for (int s = 0; s < kS; ++s)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        const int col = quad * 2 + i;
        const int d = kF8 ? j / 2 * 16 + col * 2 + (j & 1) : j * 8 + col;
        o_s[(oct + 8 * s) * kD + d] = o[j][2 * s + i];
      }
  __syncthreads();
  for (int i = threadIdx.x; i < heads * kD; i += kThreads) {
    const int g = i / kD, d = i % kD;
    float top = m_s[0][g];
#pragma unroll
    for (int w = 1; w < kWarps; ++w) top = fmaxf(top, m_s[w][g]);
    const float base = top == -INFINITY ? 0.f : top;
    float sum = 0.f, x = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float keep = exp2f(m_s[w][g] - base);
      sum += l_s[w][g] * keep;
      x += reinterpret_cast<const float*>(smem)[(w * kHeads + g) * kD + d] * keep;
    }
    const int64_t bh = (int64_t)b * a.H + h0 + g;
    if (a.splits == 1) {
      store_any(a.o, bh * kD + d, a.dtype, sum == 0.f ? 0.f : x / sum);
      if (a.lse && d == 0) a.lse[bh] = sum == 0.f ? 0.f : base - kOffset + log2f(sum);
    } else {
      a.part_o[(bh * a.splits + split) * kD + d] = x;
      if (d == 0) a.part_ml[bh * a.splits + split] = make_float2(top - kOffset, sum);
    }
  }
}

template <bool kF8, bool kBf16, int kD, bool kHalf>
int launch_mma(AttendArgs& a, cudaStream_t s) {
  using Tile = MmaTile<kF8, kBf16, kD, kHalf>;
  static std::atomic<bool> done[kMaxDevices];
  int dev = 0, n_sm = 0;
  if (!device_sm_count(&dev, &n_sm)) return KB_ERR_LAUNCH;
  KB_CUDA_TRY(opt_in_smem_once(paged_attend_mma_kernel<kF8, kBf16, kD, kHalf>, Tile::kSmem, dev, done));
  a.head_tiles = kb_cdiv_i32(a.group, Tile::kHeads);
  paged_attend_mma_kernel<kF8, kBf16, kD, kHalf><<<dim3(a.splits, a.H_kv * a.head_tiles, a.B), kThreads, Tile::kSmem, s>>>(a);
  KB_LAUNCH_CHECK("paged_attend_mma_kernel");
  return KB_OK;
}
template <bool kF8, bool kBf16>
int launch_mma(AttendArgs& a, cudaStream_t s) {
  if (a.D == 64) return a.group <= 8 ? launch_mma<kF8, kBf16, 64, true>(a, s) : launch_mma<kF8, kBf16, 64, false>(a, s);
  return a.group <= 8 ? launch_mma<kF8, kBf16, 128, true>(a, s) : launch_mma<kF8, kBf16, 128, false>(a, s);
}

// Whether the tensor-core kernel takes the call: a 16-bit q of head dim 64 or 128; keys and values of one layout, with rows on 16-byte
// boundaries, within 2^32 such units.
bool takes_mma(const kb_paged_attention_params& p) {
  const kb_paged_cache& c = p.cache;
  const int e = dtype_size(c.dtype);
  if (p.dtype == KB_F32 || (c.D != 64 && c.D != 128) || !paged_rows_aligned(c, e)) return false;
  int64_t last = 0;
  const int32_t extent[3] = {c.P, c.H_kv, c.page};
  for (int i = 0; i < 3; ++i) {
    if (c.k_stride[i] != c.v_stride[i] || c.k_stride[i] < 0 || c.k_stride[i] > (int64_t)1 << 40) return false;
    if (c.dtype == KB_E4M3 && c.k_scale_stride[i] != c.v_scale_stride[i]) return false;
    if (i != 1) last += c.k_stride[i] * kb_max_i32(extent[i] - 1, 0);
    if (last > (int64_t)1 << 40) return false;
  }
  return last * e / 16 < 0xffffffff - 64;
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
  if (takes_mma(p)) rc = c.dtype == KB_E4M3 ? launch_mma<true, false>(a, s) : c.dtype == KB_BF16 ? launch_mma<false, true>(a, s) : launch_mma<false, false>(a, s);
  else switch (c.dtype) {
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
