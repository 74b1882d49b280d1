// Attention of one new token per sequence over a paged key/value cache: o = softmax(q k^T scale) v over the rows that the
// token sees, its log-sum-exp, and on request every row's weight added to a running sum.
//
// HBM-bound: two FLOPs per byte and query head; all that counts is to read every cached row once, at full rate.  The query
// heads that share a key/value head are therefore worked on together (an item: a sequence and up to 24 query heads), and the rows
// of all items, cut into tiles, form one line that is shared out evenly: every unit (a warp of the tensor-core
// kernel, a block of the generic one) walks over a stretch of it, whatever the lengths are, and as many units are
// launched as the GPU holds.  A unit keeps, per head, the running maximum, the sum and the unnormalised output (fp32).  An item that lies
// within a unit's stretch is finished there.  Of the others each unit leaves a part (its first and its last item
// at most), and a second kernel joins an item's parts in their order:
//   m = max m_s,  l = sum l_s 2^(m_s - m),  o = sum o_s 2^(m_s - m) / l.
// Rows' weights need the final m and l, so the scores go to the workspace (4 bytes per row and query head, against
// 2 D elements per row and key/value head read) and a third kernel turns them into weights and adds them up: every sum has one
// writer, so results do not depend on the order of anything.
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
  int32_t heads, head_tiles;             // query heads of an item, items per group
  int32_t context, back;                 // context 0: every row is seen
  int32_t units, least_tiles;            // least_tiles: no unit gets fewer, as far as there are any
  int32_t by_item;                       // no more items than units
  float scale_log2;
  int4* join;       // [items] with by_item, otherwise by the unit that starts the item, [units]: {first part (-1: none), its unit, last unit, item}
  float* part_o;    // [2 units, heads, D]
  float4* part_ml;  // [2 units, heads]: maximum, sum of the weights, sum of what was multiplied with V (the weights as rounded), 0
  float* scores;    // [B, H, most_rows], base-2 logits, from the first row that is seen
  int32_t most_rows;  // that a token can see
  KbFastDiv fd_context;
  uint32_t row16[3], scale_at[3];  // tensor-core kernel: page, head and row strides of keys and values in 16 bytes, of their scales in elements
};

// The rows that the token sees: [first, end).
__device__ __forceinline__ void seen_rows(const AttendArgs& a, int32_t b, int32_t& first, int32_t& end) {
  end = a.c.rows(b);
  first = 0;
  if (a.context && end > 0) first = kb_max_i32(0, kb_fastdiv(end - 1, a.fd_context) - a.back) * a.context;
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

// ---- the line of tiles -------------------------------------------------------------------------------------------------

// Where a unit stands: tile `tile` of the `tiles` of item (b, hy), with `left` tiles of its stretch to go.  A sequence without rows has one
// tile, without rows, so that its output is written.
struct Place {
  int32_t b, hy, tile, tiles, first, end;
  int64_t left;

  __device__ __forceinline__ void enter(const AttendArgs& a, int32_t rows) {
    seen_rows(a, b, first, end);
    tiles = kb_max_i32(1, (end - first + rows - 1) / rows);
  }
  // n tiles on, to the end of the item at most
  __device__ __forceinline__ void advance(const AttendArgs& a, int32_t rows, int32_t n) {
    tile += n, left -= n;
    if (tile == tiles && left > 0) {
      tile = 0;
      if (++hy == a.H_kv * a.head_tiles) {
        hy = 0, ++b;
        enter(a, rows);
      }
    }
  }
};

__device__ __forceinline__ int64_t warp_sum(int64_t x) {
#pragma unroll
  for (int s = 16; s > 0; s >>= 1) x += __shfl_xor_sync(0xffffffffu, x, s);
  return x;
}

struct Stretch {
  Place at;           // left 0: nothing to do
  int64_t begin, each;  // the unit's first tile, and tiles per unit
  bool whole;           // instead of that: an item per unit
};

// Found by a whole warp.  `rows`: of a tile.
__device__ __forceinline__ Stretch find_stretch(const AttendArgs& a, int32_t unit, int32_t rows) {
  const int lane = threadIdx.x & 31;
  const int64_t per_seq = (int64_t)a.H_kv * a.head_tiles;
  Place p{};
  int64_t total = 0;
  int32_t longest = 0;
  for (p.b = lane; p.b < a.B; p.b += 32) {
    p.enter(a, rows);
    total += p.tiles;
    longest = max(longest, p.tiles);
  }
  total = warp_sum(total) * per_seq;
  longest = __reduce_max_sync(0xffffffffu, longest);
  Stretch s;
  s.each = total < (int64_t)a.units * a.least_tiles ? a.least_tiles : (total + a.units - 1) / a.units;
  // Items of much the same length, one for a unit: taken whole they need no joining, which costs more than an uneven share.
  // (64 sequences with windows of 513 to 640 rows, 16 heads: 31 us, and 35 us with shares of 16 tiles.)
  s.whole = a.by_item && 4 * (int64_t)longest <= 5 * s.each;
  if (s.whole) {
    const bool there = unit < a.B * per_seq;
    s.at = p;
    s.at.b = there ? (int32_t)(unit / per_seq) : 0, s.at.hy = there ? (int32_t)(unit - s.at.b * per_seq) : 0, s.at.tile = 0;
    s.at.enter(a, rows);
    s.at.left = there ? s.at.tiles : 0;
    s.begin = 0;
    return s;
  }
  s.begin = unit * s.each;
  p.left = s.begin >= total ? 0 : min(s.each, total - s.begin);
  if (p.left) {
    int64_t before = 0;
    for (int32_t b0 = 0; b0 < a.B; b0 += 32) {
      p.b = b0 + lane;
      if (p.b < a.B) p.enter(a, rows);
      const int64_t mine = p.b < a.B ? p.tiles * per_seq : 0;
      int64_t upto = mine;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int64_t y = __shfl_up_sync(0xffffffffu, upto, x);
        if (lane >= x) upto += y;
      }
      const uint32_t found = __ballot_sync(0xffffffffu, s.begin < before + upto);
      if (found) {
        const int src = __ffs(found) - 1;
        const int64_t off = s.begin - (before + __shfl_sync(0xffffffffu, upto - mine, src));
        p.b = b0 + src;
        p.enter(a, rows);
        p.hy = (int32_t)(off / p.tiles);
        p.tile = (int32_t)(off - (int64_t)p.hy * p.tiles);
        break;
      }
      before += __shfl_sync(0xffffffffu, upto, 31);
    }
  }
  s.at = p;
  return s;
}

// What becomes of the unit's part of an item: -1, it is the whole item, otherwise where the part goes.  `seen` tiles of the stretch lie before it.
// The unit that starts an item leaves word of its parts (one lane calls with `tell`).
__device__ __forceinline__ int32_t part_of_item(const AttendArgs& a, const Stretch& s, const Place& p, int32_t unit, int64_t seen, int32_t n, bool tell) {
  const int32_t slot = 2 * unit + (seen ? 1 : 0);
  const bool starts = p.tile == 0;
  const int64_t item = (int64_t)p.b * a.H_kv * a.head_tiles + p.hy;
  const bool whole = starts && n == p.tiles;
  if (tell && starts) {
    const int32_t last = whole ? unit : (int32_t)((s.begin + seen + p.tiles - 1) / s.each);
    if (a.by_item) a.join[item] = make_int4(whole ? -1 : slot, unit, last, (int32_t)item);
    else if (!whole) a.join[unit] = make_int4(slot, unit, last, (int32_t)item);
  }
  return whole ? -1 : slot;
}

// ---- generic kernel --------------------------------------------------------------------------------------------------
//
// CUDA cores, every type, head dim and alignment.  A row is a few neighbouring lanes of 16 bytes each; a group of such lanes has a softmax of
// its own, joined with the others' at the end of an item, and kAhead rows in flight.

template <int kBytes>
struct RowPart {
  uint4 raw[kBytes / 16];
  __device__ __forceinline__ void load(const char* p, bool aligned) {
    if (aligned) {
#pragma unroll
      for (int i = 0; i < kBytes / 16; ++i) raw[i] = __ldg(reinterpret_cast<const uint4*>(p) + i);
    } else {
#pragma unroll
      for (int i = 0; i < kBytes / 4; ++i) {
        const uint8_t* e = reinterpret_cast<const uint8_t*>(p) + 4 * i;
        reinterpret_cast<uint32_t*>(raw)[i] = e[0] | e[1] << 8 | e[2] << 16 | (uint32_t)e[3] << 24;
      }
    }
  }
  template <typename T>
  __device__ __forceinline__ float get(int i) const {
    if constexpr (sizeof(T) == 1) {
      return __half2float(__half(__nv_cvt_fp8_to_halfraw(reinterpret_cast<const uint8_t*>(raw)[i], __NV_E4M3)));
    } else {
      return to_f32(reinterpret_cast<const T*>(raw)[i]);
    }
  }
};

template <typename T, int D>
struct GenericTile {
  static constexpr int kBytes = D * (int)sizeof(T) > 512 ? 32 : 16;  // of a lane
  static constexpr int kLanes = D * (int)sizeof(T) / kBytes;         // per row
  static constexpr int N = D / kLanes;                               // elements per lane
  static constexpr int kAhead = 4;
  static constexpr int kGroups = 32 / kLanes;                        // rows of a warp at a time
  static constexpr int kRows = kWarps * kGroups * kAhead;
};

// T: the cache's elements (uint8_t: e4m3); G: query heads per item
template <typename T, int D, int G>
__global__ void __launch_bounds__(kThreads) paged_attend_kernel(const AttendArgs a, bool aligned) {
  using Tile = GenericTile<T, D>;
  constexpr int kLanes = Tile::kLanes, N = Tile::N, kGroups = Tile::kGroups, kAhead = Tile::kAhead, kRows = Tile::kRows;
  __shared__ float q_s[G][D];
  __shared__ float m_s[kWarps][G], l_s[kWarps][G], o_s[kWarps][G][D];
  const int32_t unit = blockIdx.x;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, sub = lane / kLanes, piece = lane % kLanes;
  if (threadIdx.x == 0 && !a.by_item) a.join[unit].x = -1;
  let_next_launch_start();
  const Stretch stretch = find_stretch(a, unit, kRows);
  Place at = stretch.at;
  for (int64_t seen = 0; at.left > 0;) {
    const int32_t n = (int32_t)min((int64_t)(at.tiles - at.tile), at.left);
    const int32_t b = at.b, hk = at.hy / a.head_tiles, h0 = hk * a.group + (at.hy - hk * a.head_tiles) * G, heads = min(G, (hk + 1) * a.group - h0);
    const int32_t slot = part_of_item(a, stretch, at, unit, seen, n, threadIdx.x == 0);
    const int32_t first = at.first, begin = first + at.tile * kRows, end = kb_min_i32(at.end, begin + n * kRows);
    at.advance(a, kRows, n);
    seen += n;

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
      for (int i = 0; i < N; ++i) q[g][i] = q_s[g][piece * N + i], o[g][i] = 0.f;
    }
    for (int32_t r0 = begin + warp * kGroups * kAhead + sub; r0 - sub < end; r0 += kRows) {
      RowPart<Tile::kBytes> k[kAhead], v[kAhead];
      float ks[kAhead], vs[kAhead];
      int32_t page[kAhead], row[kAhead];
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        page[j] = -1;
        if (r0 + j * kGroups < end) page[j] = a.c.locate(b, r0 + j * kGroups, row[j]);
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        ks[j] = vs[j] = 1.f;
        if (page[j] < 0) continue;
        k[j].load(a.c.k + (page[j] * a.c.k_page + hk * a.c.k_head + row[j] * a.c.k_row + piece * N) * (int64_t)sizeof(T), aligned);
        v[j].load(a.c.v + (page[j] * a.c.v_page + hk * a.c.v_head + row[j] * a.c.v_row + piece * N) * (int64_t)sizeof(T), aligned);
        if (sizeof(T) == 1) {
          ks[j] = a.c.k_scale[page[j] * a.c.ks_page + hk * a.c.ks_head + row[j] * a.c.ks_row];
          vs[j] = a.c.v_scale[page[j] * a.c.vs_page + hk * a.c.vs_head + row[j] * a.c.vs_row];
        }
      }
#pragma unroll
      for (int j = 0; j < kAhead; ++j) {
        const bool live = page[j] >= 0;
        const int32_t r = r0 + j * kGroups;
#pragma unroll
        for (int g = 0; g < G; ++g) {
          float s = 0.f;
#pragma unroll
          for (int i = 0; i < N; ++i) s = fmaf(q[g][i], live ? k[j].template get<T>(i) : 0.f, s);
#pragma unroll
          for (int x = kLanes / 2; x > 0; x >>= 1) s += __shfl_xor_sync(0xffffffffu, s, x);
          s = live ? s * ks[j] : -INFINITY;
          if (a.scores && piece == 0 && r < end && g < heads) a.scores[((int64_t)b * a.H + h0 + g) * a.most_rows + (r - first)] = s;
          if (!live) continue;
          const float top = fmaxf(m[g], s), base = top == -INFINITY ? 0.f : top;
          const float p = exp2f(s - base), keep = exp2f(m[g] - base);
          m[g] = top;
          l[g] = l[g] * keep + p;
          const float pv = p * vs[j];
#pragma unroll
          for (int i = 0; i < N; ++i) o[g][i] = fmaf(pv, v[j].template get<T>(i), o[g][i] * keep);
        }
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
        if (sub == 0) o_s[warp][g][piece * N + i] = x;
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
      if (slot < 0) {
        store_any(a.o, bh * D + d, a.dtype, sum == 0.f ? 0.f : x / sum);
        if (a.lse && d == 0) a.lse[bh] = sum == 0.f ? 0.f : base + log2f(sum);
      } else {
        a.part_o[((int64_t)slot * G + g) * D + d] = x;
        if (d == 0) a.part_ml[(int64_t)slot * G + g] = make_float4(top, sum, sum, 0.f);
      }
    }
    __syncthreads();  // (q_s and o_s are the next item's)
  }
}

// ---- tensor-core kernel ----------------------------------------------------------------------------------------------
//
// Caches of head dim 64 and 128.  Sixteen keys are the rows of a product (m16n8k16, m16n8k8 for fp32) and eight query heads its
// columns: S^T = K Q^T, then O^T += V^T P^T with the weights turned over in registers.  So up to eight heads cost what one does, and what
// the tensor cores have to do is a small part of the time that the keys take to arrive.  That time is all there is to hide, and
// every warp hides it for itself: it is a unit with a ring of kStages tiles of kR rows in shared memory, filled by 16-byte
// asynchronous copies that run on from one item into the next, and it never waits for another warp.
//
// Rows are found one by one (a lane looks up a row), so pages of any size and order are read the same way; a row that is
// masked is filled with zeros without being read, so that nothing in it can reach a sum.
//
// e4m3 elements become f16, exactly.  q does too (bf16 q after a multiplication by a power of two that brings its largest element to
// 2^14: what is lost lies 2^-38 below the largest).  A row's value scale belongs to its weight: the weights that are
// multiplied are p * v_scale, so the running maximum is taken over score + log2(v_scale), which keeps them within f16.  (The row of an infinite
// value is written with an infinite scale: its heads come out NaN, as 0 times infinity does; their log-sum-exp and weights do not depend on values.)
// f16 weights start at 2^7 and may grow to 2^15 before sums are rescaled: seven bits more for the small ones.
// Weights are rounded to 16 bits for the product with V (as in the operator's forward kernel).  A 16-bit cache's output is divided by the sum of
// the rounded weights, so that what their roundings have in common cancels (one row that outweighs the others comes out exact); the
// log-sum-exp is that of the weights as they were.
//
// fp32 is cut in two: x = hi + lo, hi the 11 leading bits (tf32), lo the next 11, and a product is hi hi + lo hi + hi lo, which leaves out
// some 2^-23 of it (and makes NaN of what fp32 has infinities for).  The tensor cores cut sums off where an addition rounds, so what
// they add to a long sum goes in by an addition.  (On CUDA cores a row costs 4 D flops per query head and the sums over lanes besides: 16
// sequences of 4096 rows, 32 / 8 heads of 128, took 434 us, five times what the rows take to be read; this kernel 97 us.)
//
// Measured: 64 sequences of 4096-8192 rows, 32 / 8 heads of 128, bf16 (1.6 GB): 250 us, 6.4 TB/s, the kernel alone 240 us; 131 001 rows of e4m3: 58 us, of
// which 50 this kernel (5.5 TB/s; its conversions keep 42 % of the issue slots busy); tensor pipe 9-17 %.

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
__device__ __forceinline__ void lds4(uint32_t (&r)[4], uint32_t at) {
  asm volatile("ld.shared.v4.u32 {%0, %1, %2, %3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(at) : "memory");
}
__device__ __forceinline__ float lds_f32(uint32_t at) {
  float x;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(x) : "r"(at) : "memory");
  return x;
}
template <bool BF16>
__device__ __forceinline__ float low16(uint32_t two) { return BF16 ? __uint_as_float(two << 16) : __half2float(__ushort_as_half((unsigned short)two)); }
template <bool BF16>
__device__ __forceinline__ float high16(uint32_t two) { return BF16 ? __uint_as_float(two & 0xffff0000u) : __half2float(__ushort_as_half((unsigned short)(two >> 16))); }
// an 8 x 8 matrix of 16-bit elements, a row per four lanes, turned over
__device__ __forceinline__ uint32_t transpose8x8(uint32_t x) {
  uint32_t y;
  asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
  return y;
}
// c += a b, 16 x 8 x 16
template <bool BF16>
__device__ __forceinline__ void mma16(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  if constexpr (BF16)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
        : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// c += a b, 16 x 8 x 8, in tf32
__device__ __forceinline__ void mma8(float (&c)[4], const uint32_t (&a)[4], const uint32_t (&b)[2]) {
  asm("mma.sync.aligned.m16n8k8.row.col.f32.tf32.tf32.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3]) : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b[0]), "r"(b[1]));
}
// hi: to nearest, so that lo, which is cut off, has either sign.  (A NaN stays one, in hi or in lo; so does an infinity, as a NaN.)
template <int N>
__device__ __forceinline__ void split_tf32(const uint32_t (&x)[N], uint32_t (&hi)[N], uint32_t (&lo)[N]) {
#pragma unroll
  for (int i = 0; i < N; ++i) {
    hi[i] = (x[i] + 0x1000u) & 0xffffe000u;
    lo[i] = __float_as_uint(__uint_as_float(x[i]) - __uint_as_float(hi[i])) & 0xffffe000u;
  }
}
// four e4m3 to two pairs of f16
__device__ __forceinline__ void e4m3x4_to_f16x2(uint32_t four, uint32_t& lo, uint32_t& hi) {
  asm("{\n\t.reg .b16 x, y;\n\tmov.b32 {x, y}, %2;\n\tcvt.rn.f16x2.e4m3x2 %0, x;\n\tcvt.rn.f16x2.e4m3x2 %1, y;\n\t}" : "=r"(lo), "=r"(hi) : "r"(four));
}

// kType: of the cache; products are in f16 for e4m3.  kN: eights of query heads per item
template <int kType, int kD, int kN>
struct MmaTile {
  static constexpr int kElem = kType == KB_F32 ? 4 : kType == KB_E4M3 ? 1 : 2;
  static constexpr int kRowBytes = kD * kElem, kChunks = kRowBytes / 16;
  static constexpr int kR = kRowBytes >= 256 ? 16 : 32;  // rows of a tile
  static constexpr int kStages = kRowBytes >= 256 ? 2 : kRowBytes == 128 ? 3 : 4;
  static constexpr int kScaleBytes = kType == KB_E4M3 ? 2 * kR * 4 : 0;
  static constexpr int kStageBytes = 2 * kR * kRowBytes + kScaleBytes;
  static constexpr int kWarpBytes = kStages * kStageBytes;
  static constexpr int kHeads = 8 * kN;
  static constexpr int kSmem = kWarps * kWarpBytes;
  // per SM: what shared memory and registers allow
  static constexpr int kBlocks = kRowBytes == 512 ? 1 : kRowBytes == 256 && kN == 1 ? 3 : 2;
  // Matrix loads address chunks of a row by exclusive or, within a row's bytes: rows start on multiples of them, from the ring's start on.
  static_assert(kStageBytes % kRowBytes == 0 && kStageBytes % 128 == 0 && kRowBytes <= 512, "rows start on multiples of their bytes");
  // Where chunk c of row r lies: at c ^ swizzle(r), so that what a matrix load (eight rows of a chunk) or a quarter of a 16-byte
  // load takes (two keys by four chunks; in fp32 also four rows by two chunks) lies in different banks.
  static __device__ __forceinline__ int swizzle(int r) {
    if (kType == KB_F32) return ((r & 1) << 2) | (r & 2);
    if (kType == KB_E4M3) return kD == 128 ? ((r & 1) << 2) | ((r >> 1) & 3) : (r >> 1) & 3;
    return r & 7;
  }
};

template <int kType, int kD, int kN>
__global__ void __launch_bounds__(kThreads, MmaTile<kType, kD, kN>::kBlocks) paged_attend_mma_kernel(const AttendArgs a) {
  using Tile = MmaTile<kType, kD, kN>;
  constexpr bool kF8 = kType == KB_E4M3, kBf16 = kType == KB_BF16, kF32 = kType == KB_F32, kRounded = !kF8 && !kF32;
  constexpr int kR = Tile::kR, kStages = Tile::kStages, kChunks = Tile::kChunks, kRowBytes = Tile::kRowBytes, kHeads = Tile::kHeads;
  constexpr int kSteps = kD / 16, kU = kR / 16, kDt = kD / 16;
  constexpr float kOffset = kF8 || kType == KB_F16 ? 7.f : 0.f, kSlack = 8.f;
  extern __shared__ __align__(512) uint8_t smem[];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, quad = lane & 3, oct = lane >> 2;
  const int32_t unit = blockIdx.x * kWarps + warp;
  if (lane == 0 && unit < a.units && !a.by_item) a.join[unit].x = -1;
  let_next_launch_start();
  const Stretch stretch = find_stretch(a, unit, kR);
  const uint32_t ring = sm100::smem_u32(smem) + warp * Tile::kWarpBytes;

  // ---- copies: lane r looks up row r of a tile, a tile ahead of its copy
  constexpr int kRowsAtOnce = 32 / kChunks;
  const int chunk = lane % kChunks, sub = lane / kChunks;
  const char *kfrom = a.c.k + chunk * 16, *vfrom = a.c.v + chunk * 16;
  const uint32_t place = sub * kRowBytes + ((chunk ^ Tile::swizzle(sub)) * 16);
  Place ahead = stretch.at;
  int32_t next_at = 0, next_page = -1, next_head = 0;
  auto look_up = [&]() {
    next_page = -1;
    if (ahead.left == 0) return;
    const int32_t row = ahead.first + ahead.tile * kR + (lane & (kR - 1));
    if (row < ahead.end) next_page = a.c.locate(ahead.b, row, next_at);
    next_head = a.head_tiles == 1 ? ahead.hy : ahead.hy / a.head_tiles;
    ahead.advance(a, kR, 1);
  };
  uint32_t live_bits[kStages - 1];  // of the tiles in the ring, oldest first
  auto issue = [&](int stage) -> uint32_t {
    const bool have = next_page >= 0;
    const uint32_t row16 = have ? next_page * a.row16[0] + next_head * a.row16[1] + next_at * a.row16[2] : 0u;
    const uint32_t live = __ballot_sync(0xffffffffu, have);
    const uint32_t to = ring + stage * Tile::kStageBytes;
#pragma unroll
    for (int i = 0; i < kR / kRowsAtOnce; ++i) {
      const uint64_t off = (uint64_t)__shfl_sync(0xffffffffu, row16, i * kRowsAtOnce + sub) * 16;
      const bool ok = (live >> (i * kRowsAtOnce + sub)) & 1;
      const uint32_t there = to + i * kRowsAtOnce * kRowBytes + (place ^ (Tile::swizzle(i * kRowsAtOnce) * 16));
      cp_async16(there, kfrom + off, ok);
      cp_async16(there + kR * kRowBytes, vfrom + off, ok);
    }
    if constexpr (kF8) {
      const uint32_t at = have ? next_page * a.scale_at[0] + next_head * a.scale_at[1] + next_at * a.scale_at[2] : 0u;
      if (lane < kR) {
        cp_async4(to + 2 * kR * kRowBytes + lane * 4, a.c.k_scale + at, have);
        cp_async4(to + 2 * kR * kRowBytes + kR * 4 + lane * 4, a.c.v_scale + at, have);
      }
    }
    look_up();
    __syncwarp();  // (the matrix loads and products want the warp together again)
    return live;
  };
  look_up();
  // (tiles behind the last are empty: nothing is read)
#pragma unroll
  for (int s = 0; s < kStages - 1; ++s) {
    live_bits[s] = issue(s);
    cp_async_commit();
  }

  // where this lane's matrix loads start in a tile; chunks and keys further on are an exclusive or and an offset away
  const int kkey = kF8 || kF32 ? oct : lane & 15, kchunk = kF8 || kF32 ? quad : lane >> 4;
  const int vkey = kF32 ? quad : kF8 ? lane & 15 : (lane & 7) + (lane >> 4) * 8, vchunk = kF32 ? oct : kF8 ? lane >> 4 : (lane >> 3) & 1;
  const uint32_t kplace = kkey * kRowBytes + ((kchunk ^ Tile::swizzle(kkey)) * 16);
  const uint32_t vplace = (kR + vkey) * kRowBytes + ((vchunk ^ Tile::swizzle(vkey)) * 16);
  int stage = 0;
  Place now = stretch.at;
  for (int64_t seen = 0; now.left > 0;) {
    const int32_t n = (int32_t)min((int64_t)(now.tiles - now.tile), now.left);
    const int32_t b = now.b, hk = now.hy / a.head_tiles, h0 = hk * a.group + (now.hy - hk * a.head_tiles) * kHeads, heads = min(kHeads, (hk + 1) * a.group - h0);
    const int32_t slot = part_of_item(a, stretch, now, unit, seen, n, lane == 0);
    int32_t r0 = now.tile * kR;  // counted from the first row that is seen, as the scores lie
    const int32_t end = now.end - now.first;
    now.advance(a, kR, n);
    seen += n;

    // ---- q as the products' right operand: lane (oct, quad) has elements of head oct, with e4m3 and fp32 caches the ones that its 16-byte key loads hold
    uint32_t q[kSteps][kN][kF32 ? 4 : 2];
    float back_scale[kF8 ? kN : 1][2];  // of heads 2 quad and 2 quad + 1, as the scores lie
#pragma unroll
    for (int e = 0; e < kN; ++e) {
      const int g = oct + 8 * e;
      const int64_t head = b * a.q_b + (int64_t)(h0 + (g < heads ? g : 0)) * a.q_h;
      if constexpr (kF32) {
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
#pragma unroll
          for (int p = 0; p < 4; ++p) q[t][e][p] = g < heads ? __ldg(static_cast<const uint32_t*>(a.q) + head + t * 16 + quad * 4 + p) : 0u;
      }
      const uint16_t* from = static_cast<const uint16_t*>(a.q) + head;
#pragma unroll
      for (int t = 0; t < (kF32 ? 0 : kSteps); ++t)
#pragma unroll
        for (int p = 0; p < 2; ++p) {
          const int d = kF8 ? t / 4 * 64 + quad * 16 + t % 4 * 4 + 2 * p : t * 16 + 8 * p + quad * 2;
          q[t][e][p] = g < heads ? __ldg(reinterpret_cast<const uint32_t*>(from + d)) : 0u;
        }
      if constexpr (kF8) {
        float down = a.scale_log2;
        if (a.dtype == KB_BF16) {
          // (bf16 magnitudes without their signs order like whole numbers; what is not a number stays above)
          uint32_t most = 0;
#pragma unroll
          for (int t = 0; t < kSteps; ++t)
#pragma unroll
            for (int p = 0; p < 2; ++p) most = __vmaxu2(most, q[t][e][p] & 0x7fff7fffu);
          most = max(most & 0xffffu, most >> 16);
          most = max(most, __shfl_xor_sync(0xffffffffu, most, 1));
          most = max(most, __shfl_xor_sync(0xffffffffu, most, 2));
          const int x = (int)(most >> 7) - 127;  // the largest lies in [2^x, 2^(x + 1))
          const int by = most == 0 || x == 128 ? 0 : min(126, 14 - x);  // (-113 to 126: a normal number either way up)
          const float up = __uint_as_float((uint32_t)(by + 127) << 23);
          down *= __uint_as_float((uint32_t)(127 - by) << 23);
#pragma unroll
          for (int t = 0; t < kSteps; ++t)
#pragma unroll
            for (int p = 0; p < 2; ++p) {
              const uint32_t w = q[t][e][p];
              q[t][e][p] = sm100::pack_f16x2(__uint_as_float(w << 16) * up, __uint_as_float(w & 0xffff0000u) * up);
            }
        }
#pragma unroll
        for (int i = 0; i < 2; ++i) back_scale[e][i] = __shfl_sync(0xffffffffu, down, (quad * 2 + i) * 4);
      }
    }

    // element (2 r + i) of a product's lane: key (or element of the head) oct + 8 r, query head 2 quad + i
    float o[kDt][kN][4], m[kN][2], l[kN][2], z[kRounded ? kN : 1][2];
#pragma unroll
    for (int e = 0; e < kN; ++e) {
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        m[e][i] = -INFINITY, l[e][i] = 0.f;
        if constexpr (kRounded) z[e][i] = 0.f;
      }
#pragma unroll
      for (int j = 0; j < kDt; ++j)
#pragma unroll
        for (int i = 0; i < 4; ++i) o[j][e][i] = 0.f;
    }

    for (int32_t i_tile = 0; i_tile < n; ++i_tile, r0 += kR) {
      cp_async_wait<kStages - 2>();
      __syncwarp();
      const uint32_t at = ring + stage * Tile::kStageBytes, kat = at + kplace, vat = at + vplace;
      const uint32_t live = live_bits[0];
      // every lane is through with the tile before this one: the next copies take its place
#pragma unroll
      for (int s = 0; s < kStages - 2; ++s) live_bits[s] = live_bits[s + 1];
      live_bits[kStages - 2] = issue(stage == 0 ? kStages - 1 : stage - 1);
      cp_async_commit();

      // scores
      float sc[kU][kN][4];
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int e = 0; e < kN; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[u][e][i] = 0.f;
      if constexpr (kF32) {
        float small[kN][4] = {};
#pragma unroll
        for (int t = 0; t < kSteps; ++t) {
          uint32_t x[4], y[4];
          lds4(x, kat ^ (t * 64));
          lds4(y, (kat ^ (t * 64)) + 8 * kRowBytes);
#pragma unroll
          for (int p = 0; p < 4; p += 2) {
            const uint32_t r[4] = {x[p], y[p], x[p + 1], y[p + 1]};
            uint32_t hi[4], lo[4];
            split_tf32(r, hi, lo);
#pragma unroll
            for (int e = 0; e < kN; ++e) {
              const uint32_t w[2] = {q[t][e][p], q[t][e][p + 1]};
              uint32_t qhi[2], qlo[2];
              split_tf32(w, qhi, qlo);
              mma8(small[e], lo, qhi);
              mma8(small[e], hi, qlo);
              float step[4] = {0.f, 0.f, 0.f, 0.f};
              mma8(step, hi, qhi);
#pragma unroll
              for (int i = 0; i < 4; ++i) sc[0][e][i] += step[i];
            }
          }
        }
#pragma unroll
        for (int e = 0; e < kN; ++e)
#pragma unroll
          for (int i = 0; i < 4; ++i) sc[0][e][i] += small[e][i];
      } else if constexpr (!kF8) {
#pragma unroll
        for (int t = 0; t < kSteps; ++t)
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            uint32_t r[4];
            ldsm4(r, (kat ^ (t * 32)) + u * 16 * kRowBytes);
#pragma unroll
            for (int e = 0; e < kN; ++e) mma16<kBf16>(sc[u][e], r, q[t][e]);
          }
      } else {
#pragma unroll
        for (int t4 = 0; t4 < kSteps / 4; ++t4)
#pragma unroll
          for (int u = 0; u < kU; ++u) {
            uint32_t x[4], y[4];
            lds4(x, (kat ^ (t4 * 64)) + u * 16 * kRowBytes);
            lds4(y, (kat ^ (t4 * 64)) + (u * 16 + 8) * kRowBytes);
#pragma unroll
            for (int t = 0; t < 4; ++t) {
              uint32_t r[4];
              e4m3x4_to_f16x2(x[t], r[0], r[2]);
              e4m3x4_to_f16x2(y[t], r[1], r[3]);
#pragma unroll
              for (int e = 0; e < kN; ++e) mma16<kBf16>(sc[u][e], r, q[t4 * 4 + t][e]);
            }
          }
      }
      // base-2 logits; what a row's value scale adds to the maximum
      float top[kN][2], vs[kF8 ? kU : 1][2];
#pragma unroll
      for (int e = 0; e < kN; ++e) top[e][0] = top[e][1] = -INFINITY;
#pragma unroll
      for (int u = 0; u < kU; ++u)
#pragma unroll
        for (int r = 0; r < 2; ++r) {
          const int key = u * 16 + r * 8 + oct;
          float ks = 1.f, lift = 0.f;
          if constexpr (kF8) {
            ks = lds_f32(at + 2 * kR * kRowBytes + key * 4);
            vs[u][r] = lds_f32(at + 2 * kR * kRowBytes + kR * 4 + key * 4);
            // (2^-80: no lower, or the sum of the weights leaves fp32: a weight is 2^(offset + slack + 80) = 2^95 at most, and there are 2^30
            // rows at most.  What is multiplied with V then loses bits where all scales are below that.  With a scale of 2^L the largest weight is
            // 2^(offset - L) at least, and those below 2^(L - 133) of it are 0 in fp32: too little to show up to L = 88.  A scale that is not
            // finite makes the products with V NaN, whatever its weight: it has no part in the maximum, so that the sum of the weights stays what it is.)
            const float size = fabsf(vs[u][r]);
            lift = size < INFINITY ? __log2f(fmaxf(size, 8.3e-25f)) : 0.f;
          }
          const bool there = (live >> key) & 1;
#pragma unroll
          for (int e = 0; e < kN; ++e)
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              float x = sc[u][e][2 * r + i] * (kF8 ? back_scale[e][i] * ks : a.scale_log2);
              x = there ? x : -INFINITY;
              sc[u][e][2 * r + i] = x;
              top[e][i] = fmaxf(top[e][i], kF8 ? x + lift : x);
            }
        }
      if (a.scores) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const int g = 8 * e + 2 * quad + i;
            if (g >= heads) continue;
            float* out = a.scores + ((int64_t)b * a.H + h0 + g) * a.most_rows + r0 + oct;
#pragma unroll
            for (int u = 0; u < kU; ++u)
#pragma unroll
              for (int r = 0; r < 2; ++r)
                if (r0 + u * 16 + r * 8 + oct < end) out[u * 16 + r * 8] = sc[u][e][2 * r + i];
          }
        __syncwarp();
      }
      bool raise = false;
#pragma unroll
      for (int e = 0; e < kN; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
          for (int x = 4; x < 32; x <<= 1) top[e][i] = fmaxf(top[e][i], __shfl_xor_sync(0xffffffffu, top[e][i], x));
          raise = raise || top[e][i] > m[e][i] + kSlack;
        }
      if (__any_sync(0xffffffffu, raise)) {
#pragma unroll
        for (int e = 0; e < kN; ++e)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            const float to = fmaxf(m[e][i], top[e][i]);
            const float keep = to == -INFINITY ? 0.f : sm100::ex2_approx(m[e][i] - to);
            m[e][i] = to;
            l[e][i] *= keep;
            if constexpr (kRounded) z[e][i] *= keep;
#pragma unroll
            for (int j = 0; j < kDt; ++j) o[j][e][i] *= keep, o[j][e][2 + i] *= keep;
          }
      }
      float base[kN][2];
#pragma unroll
      for (int e = 0; e < kN; ++e)
#pragma unroll
        for (int i = 0; i < 2; ++i) base[e][i] = m[e][i] == -INFINITY ? 0.f : m[e][i] - kOffset;
      // weights and their products with V, 16 keys at a time
#pragma unroll
      for (int u = 0; u < kU; ++u) {
        uint32_t p[kN][2];
        float pf[kF32 ? kN : 1][4];
#pragma unroll
        for (int e = 0; e < kN; ++e)
#pragma unroll
          for (int r = 0; r < 2; ++r) {
            float x = sm100::ex2_approx(sc[u][e][2 * r] - base[e][0]), y = sm100::ex2_approx(sc[u][e][2 * r + 1] - base[e][1]);
            l[e][0] += x, l[e][1] += y;
            if constexpr (kF8) x *= vs[u][r], y *= vs[u][r];
            if constexpr (kF32) {
              pf[e][2 * r] = x, pf[e][2 * r + 1] = y;
            } else {
              const uint32_t both = sm100::pack16x2<kBf16>(x, y);
              if constexpr (kRounded) z[e][0] += low16<kBf16>(both), z[e][1] += high16<kBf16>(both);
              p[e][r] = transpose8x8(both);
            }
          }
        if constexpr (kF32) {
#pragma unroll
          for (int h = 0; h < 2; ++h) {  // eight keys: 8 h + quad and 8 h + quad + 4
            uint32_t phi[kN][2], plo[kN][2];
#pragma unroll
            for (int e = 0; e < kN; ++e) {
#pragma unroll
              for (int k = 0; k < 2; ++k) {  // turned over: from key oct, heads 2 quad and 2 quad + 1 to key quad + 4 k, head oct
                const int from = (quad + 4 * k) * 4 + (oct >> 1);
                const float x = __shfl_sync(0xffffffffu, pf[e][2 * h], from), y = __shfl_sync(0xffffffffu, pf[e][2 * h + 1], from);
                p[e][k] = __float_as_uint(oct & 1 ? y : x);
              }
              split_tf32(p[e], phi[e], plo[e]);
            }
#pragma unroll
            for (int j = 0; j < kDt; j += 2) {
              uint32_t x[4], y[4];
              lds4(x, (vat ^ (j * 64)) + 8 * h * kRowBytes);
              lds4(y, (vat ^ (j * 64)) + (8 * h + 4) * kRowBytes);
#pragma unroll
              for (int c = 0; c < 2; ++c) {
                const uint32_t r[4] = {x[2 * c], x[2 * c + 1], y[2 * c], y[2 * c + 1]};
                uint32_t hi[4], lo[4];
                split_tf32(r, hi, lo);
#pragma unroll
                for (int e = 0; e < kN; ++e) {
                  float step[4] = {0.f, 0.f, 0.f, 0.f};
                  mma8(step, lo, phi[e]);
                  mma8(step, hi, plo[e]);
                  mma8(step, hi, phi[e]);
#pragma unroll
                  for (int i = 0; i < 4; ++i) o[j + c][e][i] += step[i];
                }
              }
            }
          }
        } else if constexpr (!kF8) {
#pragma unroll
          for (int j = 0; j < kDt; ++j) {
            uint32_t r[4];
            ldsm4_t(r, (vat ^ (j * 32)) + u * 16 * kRowBytes);
#pragma unroll
            for (int e = 0; e < kN; ++e) mma16<kBf16>(o[j][e], r, p[e]);
          }
        } else {
          // a 16-bit column of the transposed load is a pair of neighbouring elements: rows oct and oct + 8 of a product
#pragma unroll
          for (int j = 0; j < kDt; j += 2) {
            uint32_t w[4];
            ldsm4_t(w, (vat ^ (j * 16)) + u * 16 * kRowBytes);
#pragma unroll
            for (int c = 0; c < 2; ++c) {
              uint32_t r[4];  // (keys 2 quad and 2 quad + 1 of one element side by side, then of its neighbour)
              e4m3x4_to_f16x2(__byte_perm(w[2 * c], 0, 0x3120), r[0], r[1]);
              e4m3x4_to_f16x2(__byte_perm(w[2 * c + 1], 0, 0x3120), r[2], r[3]);
#pragma unroll
              for (int e = 0; e < kN; ++e) mma16<kBf16>(o[j + c][e], r, p[e]);
            }
          }
        }
      }
      stage = stage == kStages - 1 ? 0 : stage + 1;
    }

    // ---- what the item, or this part of it, comes to
#pragma unroll
    for (int e = 0; e < kN; ++e)
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        float sum = l[e][i], by_sum = kRounded ? z[kRounded ? e : 0][i] : 0.f;
#pragma unroll
        for (int x = 4; x < 32; x <<= 1) {
          sum += __shfl_xor_sync(0xffffffffu, sum, x);
          if constexpr (kRounded) by_sum += __shfl_xor_sync(0xffffffffu, by_sum, x);
        }
        if constexpr (!kRounded) by_sum = sum;
        const int g = 8 * e + 2 * quad + i;
        if (g >= heads) continue;
        const int64_t bh = (int64_t)b * a.H + h0 + g, part = (int64_t)slot * kHeads + g;
        // (a head without weights is 0 even where what it would be divided by is not: 0 * 0)
        const bool none = sum == 0.f;
        const float by = slot >= 0 ? 1.f : 1.f / by_sum;
        if (oct == 0) {
          if (slot >= 0) a.part_ml[part] = make_float4(m[e][i] - kOffset, sum, by_sum, 0.f);
          else if (a.lse) a.lse[bh] = none ? 0.f : m[e][i] - kOffset + log2f(sum);
        }
#pragma unroll
        for (int j = 0; j < kDt; ++j) {
          const float x = none ? 0.f : o[j][e][i] * by, y = none ? 0.f : o[j][e][2 + i] * by;
          const int d = kF32 ? j / 2 * 32 + oct * 4 + j % 2 * 2 : kF8 ? j * 16 + 2 * oct : j * 16 + oct, d2 = kF8 || kF32 ? d + 1 : d + 8;
          if (slot >= 0) {
            a.part_o[part * kD + d] = x, a.part_o[part * kD + d2] = y;
          } else {
            const int32_t type = kF8 ? a.dtype : kType;
            store_any(a.o, bh * kD + d, type, x), store_any(a.o, bh * kD + d2, type, y);
          }
        }
      }
  }
  cp_async_wait<0>();
}

// ---- the parts of an item joined -----------------------------------------------------------------------------------------

constexpr int kMostJoinThreads = 1024;

// A block per item and head.  Groups of D / 4 threads take every so many-th part, four elements per thread; the groups are added up in order.
__global__ void __launch_bounds__(kMostJoinThreads) paged_join_kernel(const AttendArgs a) {
  __shared__ float red[kMostJoinThreads / 32], sums[kMostJoinThreads / 4][2];
  __shared__ __align__(16) float o_s[kMostJoinThreads * 4];
  const int threads = blockDim.x;
  let_next_launch_start();
  wait_for_launch_before();
  const int4 word = a.join[blockIdx.x];  // first part, its unit, last unit, item
  const int32_t g = blockIdx.y;
  if (word.x < 0) return;
  const int32_t per_seq = a.H_kv * a.head_tiles, b = word.w / per_seq, hy = word.w - b * per_seq, hk = hy / a.head_tiles;
  const int32_t h = hk * a.group + (hy - hk * a.head_tiles) * a.heads + g;
  if (h >= (hk + 1) * a.group) return;
  const int32_t n = word.z - word.y + 1;
  auto part_at = [&](int32_t i) { return (int64_t)(i == 0 ? word.x : 2 * (word.y + i)) * a.heads + g; };
  float top = -INFINITY;
  for (int i = threadIdx.x; i < n; i += threads) top = fmaxf(top, a.part_ml[part_at(i)].x);
#pragma unroll
  for (int x = 16; x > 0; x >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, x));
  if ((threadIdx.x & 31) == 0) red[threadIdx.x >> 5] = top;
  __syncthreads();
  for (int w = 0; w < threads / 32; ++w) top = fmaxf(top, red[w]);
  const float base = top == -INFINITY ? 0.f : top;

  const int width = a.D / 4, groups = threads / width, group = threadIdx.x / width, d = (threadIdx.x - group * width) * 4;
  float sum = 0.f, by = 0.f;
  float4 x = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll 4
  for (int i = group; i < n; i += groups) {
    const float4 e = a.part_ml[part_at(i)];
    const float4 y = *reinterpret_cast<const float4*>(a.part_o + part_at(i) * a.D + d);
    const float keep = exp2f(e.x - base);
    sum = fmaf(e.y, keep, sum), by = fmaf(e.z, keep, by);
    x.x = fmaf(y.x, keep, x.x), x.y = fmaf(y.y, keep, x.y), x.z = fmaf(y.z, keep, x.z), x.w = fmaf(y.w, keep, x.w);
  }
  *reinterpret_cast<float4*>(o_s + group * a.D + d) = x;
  if (d == 0) sums[group][0] = sum, sums[group][1] = by;
  __syncthreads();
  const int64_t bh = (int64_t)b * a.H + h;
  for (int i = threadIdx.x; i < a.D; i += threads) {
    float s = 0.f, z = 0.f, y = 0.f;
    for (int k = 0; k < groups; ++k) s += sums[k][0], z += sums[k][1], y += o_s[k * a.D + i];
    store_any(a.o, bh * a.D + i, a.dtype, s == 0.f ? 0.f : y / z);
    if (a.lse && i == 0) a.lse[bh] = s == 0.f ? 0.f : base + log2f(s);
  }
}

// ---- rows' weights -------------------------------------------------------------------------------------------------------

constexpr int kWeighRows = 1024;  // of a block, four per thread

// A block takes rows of one sequence and key/value head; the group's log-sum-exps are the same for all of them.
__global__ void __launch_bounds__(256) paged_weigh_kernel(const AttendArgs a) {
  constexpr int kEach = kWeighRows / 256;
  const int32_t hk = blockIdx.y, b = blockIdx.z;
  const int64_t bh = (int64_t)b * a.H + hk * a.group;
  int32_t first, end;
  seen_rows(a, b, first, end);
  wait_for_launch_before();
  const int32_t r0 = first + blockIdx.x * kWeighRows + threadIdx.x;
  if (r0 >= end) return;
  const float *scores = a.scores + bh * a.most_rows + (r0 - first), *lse = a.lse + bh;
  float* to = a.weights + b * a.w_b + hk * a.w_h + r0;
  float w[kEach], x[kEach];
#pragma unroll
  for (int i = 0; i < kEach; ++i) w[i] = 0.f;
  for (int g = 0; g < a.group; ++g, scores += a.most_rows) {
    const float base = lse[g];
#pragma unroll
    for (int i = 0; i < kEach; ++i) x[i] = r0 + i * 256 < end ? __ldcs(scores + i * 256) : -INFINITY;
#pragma unroll
    for (int i = 0; i < kEach; ++i) w[i] += sm100::ex2_approx(x[i] - base);
  }
#pragma unroll
  for (int i = 0; i < kEach; ++i)
    if (r0 + i * 256 < end) to[i * 256] += w[i];
}

// Whether the tensor-core kernel takes the call: head dim 64 or 128; dense heads of q, which has 16 bits where the cache has 8; keys and values of
// one layout, with rows on 16-byte boundaries, within 2^32 such units; their scales of one layout, within 2^32 elements.
bool takes_mma(const kb_paged_attention_params& p) {
  const kb_paged_cache& c = p.cache;
  const int e = dtype_size(c.dtype);
  if ((p.dtype == KB_F32 && c.dtype != KB_F32) || (c.D != 64 && c.D != 128) || !paged_rows_aligned(c, e)) return false;
  if (p.q_stride[2] != 1) return false;
  if (p.dtype != KB_F32 && (p.q_stride[0] % 2 || p.q_stride[1] % 2 || reinterpret_cast<uintptr_t>(p.q) % 4)) return false;
  const int32_t extent[3] = {c.P, c.H_kv, c.page};
  const auto within = [&](const int64_t (&x)[3], const int64_t (&y)[3], int64_t unit) {
    uint64_t last = 0;
    for (int i = 0; i < 3; ++i) {
      if (x[i] != y[i] || x[i] < 0 || x[i] >= (int64_t)1 << 36) return false;
      last += (uint64_t)x[i] * (extent[i] > 1 ? extent[i] - 1 : 0) / unit;  // (below 2^36 * 2^31)
      if (last >= 0xffffff00u) return false;
    }
    return true;
  };
  return within(c.k_stride, c.v_stride, 16 / e) && (c.dtype != KB_E4M3 || within(c.k_scale_stride, c.v_scale_stride, 1));
}

// ---- launches --------------------------------------------------------------------------------------------------------------

constexpr int kSms = 148;

template <int kType, int kD, int kN>
struct MmaKernel {
  using Tile = MmaTile<kType, kD, kN>;
  static constexpr int kHeads = Tile::kHeads, kRows = Tile::kR, kUnits = kSms * Tile::kBlocks * kWarps;
  static constexpr int kLeast = 64 / kRows;  // tiles: short stretches leave parts that cost more to join than they save
  static int launch(const AttendArgs& a, bool, cudaStream_t s) {
    static std::atomic<bool> done[kMaxDevices];
    int dev = 0, n_sm = 0;
    if (!device_sm_count(&dev, &n_sm)) return KB_ERR_LAUNCH;
    KB_CUDA_TRY(opt_in_smem_once(paged_attend_mma_kernel<kType, kD, kN>, Tile::kSmem, dev, done));
    paged_attend_mma_kernel<kType, kD, kN><<<kb_cdiv_i32(a.units, kWarps), kThreads, Tile::kSmem, s>>>(a);
    KB_LAUNCH_CHECK("paged_attend_mma_kernel");
    return KB_OK;
  }
};
template <typename T, int D, int G>
struct GenericKernel {
  static constexpr int kHeads = G, kRows = GenericTile<T, D>::kRows, kUnits = kSms * (G == 1 ? 4 : 2), kLeast = 1;
  static int launch(const AttendArgs& a, bool aligned, cudaStream_t s) {
    paged_attend_kernel<T, D, G><<<a.units, kThreads, 0, s>>>(a, aligned);
    KB_LAUNCH_CHECK("paged_attend_kernel");
    return KB_OK;
  }
};

// f(a kernel): the one for the call
template <int kType, int kD, typename F>
auto with_eights(const kb_paged_attention_params& p, F f) {
  // As few items as three eights of heads each allow (two where a third would not fit into the registers), and those alike.  Twenty heads on one
  // key/value head, 16 384 rows of 128 in f16: 47 us at once, 61 us in two items; 64 x 8192 rows of e4m3: 89 us and 77 us.
  constexpr int32_t most = kType == KB_F32 || (kType == KB_E4M3 && kD == 128) ? 2 : 3;
  const int32_t eights = kb_cdiv_i32(p.H / p.cache.H_kv, 8), n = kb_cdiv_i32(eights, kb_cdiv_i32(eights, most));
  if (n == 1) return f(MmaKernel<kType, kD, 1>());
  if constexpr (most == 3) {
    if (n == 3) return f(MmaKernel<kType, kD, 3>());
  }
  return f(MmaKernel<kType, kD, 2>());
}
template <int kType, typename F>
auto with_mma(const kb_paged_attention_params& p, F f) {
  return p.cache.D == 64 ? with_eights<kType, 64>(p, f) : with_eights<kType, 128>(p, f);
}
template <typename T, int D, typename F>
auto with_group(const kb_paged_attention_params& p, F f) {
  return p.H == p.cache.H_kv ? f(GenericKernel<T, D, 1>()) : f(GenericKernel<T, D, 4>());
}
template <typename T, typename F>
auto with_generic(const kb_paged_attention_params& p, F f) {
  switch (p.cache.D) {
    case 16: return with_group<T, 16>(p, f);
    case 32: return with_group<T, 32>(p, f);
    case 64: return with_group<T, 64>(p, f);
    case 128: return with_group<T, 128>(p, f);
    default: return with_group<T, 256>(p, f);
  }
}
template <typename F>
auto with_kernel(const kb_paged_attention_params& p, F f) {
  const int32_t dtype = p.cache.dtype;
  if (takes_mma(p)) {
    switch (dtype) {
      case KB_F32: return with_mma<KB_F32>(p, f);
      case KB_F16: return with_mma<KB_F16>(p, f);
      case KB_BF16: return with_mma<KB_BF16>(p, f);
      default: return with_mma<KB_E4M3>(p, f);
    }
  }
  switch (dtype) {
    case KB_F32: return with_generic<float>(p, f);
    case KB_F16: return with_generic<__half>(p, f);
    case KB_BF16: return with_generic<__nv_bfloat16>(p, f);
    default: return with_generic<uint8_t>(p, f);
  }
}

// What follows from the sizes alone (the lengths are on the device).
struct Plan {
  int32_t heads, head_tiles, units, least, most_rows;
  int64_t items;
  bool by_item, joins;
  size_t join_bytes, part_bytes, ml_bytes, score_bytes;
};

template <typename K>
Plan make_plan(const kb_paged_attention_params& p) {
  Plan n{};
  const kb_paged_cache& c = p.cache;
  n.heads = K::kHeads;
  n.head_tiles = kb_cdiv_i32(p.H / c.H_kv, K::kHeads);
  n.least = K::kLeast;
  const int64_t capacity = (int64_t)c.M * c.page, window = p.context_size > 0 ? ((int64_t)p.back_contexts + 1) * p.context_size : capacity;
  n.most_rows = (int32_t)(window < capacity ? window : capacity);
  const int64_t items = n.items = (int64_t)c.B * c.H_kv * n.head_tiles, tiles = (n.most_rows + K::kRows - 1) / K::kRows;
  const int64_t stretches = (items * (tiles < 1 ? 1 : tiles) + K::kLeast - 1) / K::kLeast;
  n.units = (int32_t)(stretches < K::kUnits ? stretches : K::kUnits);
  n.by_item = items <= n.units;
  n.joins = n.units > 1;
  const size_t entries = n.by_item ? items : n.units, parts = 2 * (size_t)n.units * n.heads;
  n.join_bytes = entries * sizeof(int4);
  n.part_bytes = parts * c.D * sizeof(float);
  n.ml_bytes = parts * sizeof(float4);
  // (a window's first row is the first of a chunk: from there to the last row there are most_rows at most)
  n.score_bytes = p.weights ? (size_t)c.B * p.H * n.most_rows * sizeof(float) : 0;
  return n;
}

}  // namespace

size_t paged_attention_workspace_bytes(const kb_paged_attention_params& p) {
  return with_kernel(p, [&](auto kernel) {
    const Plan n = make_plan<decltype(kernel)>(p);
    return n.join_bytes + n.part_bytes + n.ml_bytes + n.score_bytes;
  });
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
  a.scale_log2 = p.sm_scale * kLog2e;
  for (int i = 0; i < 3; ++i) a.row16[i] = (uint32_t)(c.k_stride[i] * dtype_size(c.dtype) / 16), a.scale_at[i] = (uint32_t)c.k_scale_stride[i];
  return with_kernel(p, [&](auto kernel) {
    const Plan n = make_plan<decltype(kernel)>(p);
    a.heads = n.heads, a.head_tiles = n.head_tiles, a.units = n.units, a.least_tiles = n.least, a.by_item = n.by_item;
    char* w = static_cast<char*>(p.workspace);
    a.join = reinterpret_cast<int4*>(w), w += n.join_bytes;
    a.part_o = reinterpret_cast<float*>(w), w += n.part_bytes;
    a.part_ml = reinterpret_cast<float4*>(w), w += n.ml_bytes;
    if (p.weights) a.scores = reinterpret_cast<float*>(w), a.most_rows = n.most_rows;
    if (int rc = kernel.launch(a, paged_rows_aligned(c, dtype_size(c.dtype)), s)) return rc;
    if (n.joins) {
      const dim3 grid((unsigned)(n.join_bytes / sizeof(int4)), kb_min_i32(n.heads, a.group));
      // a group of D / 4 threads for every second part of an item or so
      int32_t threads = 128;
      while (threads < kMostJoinThreads && threads < (int64_t)n.units / n.items * (c.D / 8)) threads *= 2;
      if (int rc = launch_after(paged_join_kernel, grid, threads, s, a)) return rc;
    }
    if (p.weights) {
      const dim3 grid(kb_max_i32(1, kb_cdiv_i32(n.most_rows, kWeighRows)), c.H_kv, c.B);
      if (int rc = launch_after(paged_weigh_kernel, grid, 256, s, a)) return rc;
    }
    return (int)KB_OK;
  });
}

}  // namespace kb
