// The upkeep of a paged key/value cache: new tokens are written into their rows, and rows are evicted by the attention
// weight that they have received.
//
// WRITE.  Token t < n_b of sequence b goes to row len_b - n_b + t.  HBM-bound: every element is read once and written
// once.  A row of one head is eight or sixteen elements per thread, a few neighbouring threads: its largest magnitude, which sets
// the scale of an 8-bit row, is a few shuffles away.  The threads look up a token's place once and walk over its heads.
//
// EVICT.  Rows rank by (position among the newest `recent`, then weight, then the lower row); the first `budget` stay.  Where the newest alone are
// more than the budget they rank by position, so that a token just written is never the one that goes.  Rows without a page (an entry of the
// table outside the pages) hold nothing: they are passed over, and so are places without one.
// The kept rows below the budget stay where they are, and the i-th kept row behind it moves to the i-th place that came
// free before it.  Attention does not depend on the rows' order, so nothing else has to move: a cache that is one row
// over its budget moves one row, not half of them.  Sources lie behind the budget and destinations before it, so all
// moves are independent.  Two kernels: a block per (sequence, head), or a cluster of blocks where the table is long, picks the rows, then the
// moves are spread over the GPU.
#include "common.cuh"
#include "paged.cuh"
#include "sm100_ptx.cuh"

#include <type_traits>

namespace kb {
namespace {

// ---- write -----------------------------------------------------------------------------------------------------------

constexpr int kWriteThreads = 256;

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
  int32_t B, H_kv, T, D, heads_per_cta;
  KbFastDiv fd_T;
};

template <typename T, int N>
struct alignas(N * sizeof(T) % 16 == 0 ? 16 : alignof(T)) Several { T v[N]; };

template <typename T, int N, bool kAligned>
__device__ __forceinline__ void load_several(Several<T, N>& e, const T* x, int64_t sd) {
  if constexpr (kAligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(&e)[i] = __ldcs(reinterpret_cast<const uint4*>(x) + i);
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) e.v[i] = x[i * sd];
  }
}
template <typename T, int N, bool kAligned>
__device__ __forceinline__ void store_several(T* out, const Several<T, N>& e) {
  if constexpr (kAligned) {
#pragma unroll
    for (int i = 0; i < (int)sizeof(e) / 16; ++i) reinterpret_cast<uint4*>(out)[i] = reinterpret_cast<const uint4*>(&e)[i];
  } else {
#pragma unroll
    for (int i = 0; i < N; ++i) out[i] = e.v[i];
  }
}

// The largest magnitude's bits.  Bits without the sign: numbers keep their order, and a NaN is above them all, so that it reaches the scale.
template <typename T, int N>
__device__ __forceinline__ uint32_t largest_bits(const Several<T, N>& e) {
  const uint32_t* w = reinterpret_cast<const uint32_t*>(&e);
  uint32_t m = 0;
  if constexpr (sizeof(T) == 4) {
#pragma unroll
    for (int i = 0; i < N; ++i) m = max(m, w[i] & 0x7fffffffu);
    return m;
  } else {
#pragma unroll
    for (int i = 0; i < N / 2; ++i) m = __vmaxu2(m, w[i] & 0x7fff7fffu);
    const uint16_t h = (uint16_t)max(m & 0xffffu, m >> 16);
    return __float_as_uint(to_f32(*reinterpret_cast<const T*>(&h)));
  }
}

// The row's elements as its 8-bit form holds them: x / scale correctly rounded (div_by, two at a time), then rounded to e4m3.
template <typename T, int N>
__device__ __forceinline__ Several<uint8_t, N> quantize(const Several<T, N>& e, float scale, float r) {
  float f[N];
  if (scale <= 1e37f) {
    const uint64_t r2 = sm100::f2_pack(r, r), down = sm100::f2_pack(-scale, -scale);
#pragma unroll
    for (int i = 0; i < N; i += 2) {
      const uint64_t x = sm100::f2_pack(to_f32(e.v[i]), to_f32(e.v[i + 1])), q = sm100::f2_mul(x, r2);
      sm100::f2_unpack(sm100::f2_fma(sm100::f2_fma(q, down, x), r2, q), f[i], f[i + 1]);
    }
  } else {  // an infinity or a NaN in the row
#pragma unroll
    for (int i = 0; i < N; ++i) f[i] = to_f32(e.v[i]) / scale;
  }
  Several<uint8_t, N> out;
#pragma unroll
  for (int i = 0; i < N / 4; ++i) {
    // the signs as they come: the correction above turns -0 into 0
    uint32_t sign;
    const uint32_t* w = reinterpret_cast<const uint32_t*>(&e) + i * sizeof(T);
    if constexpr (sizeof(T) == 2) sign = __byte_perm(w[0], w[1], 0x7531);
    else sign = __byte_perm(__byte_perm(w[0], w[1], 0x0073), __byte_perm(w[2], w[3], 0x0073), 0x5410);
    reinterpret_cast<uint32_t*>(&out)[i] = sm100::pack_e4m3x4(f[4 * i], f[4 * i + 1], f[4 * i + 2], f[4 * i + 3]) | (sign & 0x80808080u);
  }
  return out;
}

// 8-bit rows: sixteen, so that a row's largest magnitude is three exchanges away instead of four (head dim 128).
template <typename T, bool kF8>
constexpr __host__ __device__ int elements_per_thread() { return kF8 ? 16 : 8; }

// T: the tokens' type; kF8: the cache holds e4m3, otherwise T
template <typename T, bool kF8, bool kAligned>
__global__ void __launch_bounds__(kWriteThreads) paged_write_kernel(const WriteArgs a) {
  constexpr int kPerThread = elements_per_thread<T, kF8>();
  const int lanes = a.D / kPerThread;  // a power of two up to 32
  const int lane = threadIdx.x & (lanes - 1), d = lane * kPerThread;
  const int64_t token = (int64_t)blockIdx.x * (kWriteThreads / lanes) + threadIdx.x / lanes;
  const int32_t h0 = blockIdx.y * a.heads_per_cta, h1 = kb_min_i32(h0 + a.heads_per_cta, a.H_kv);
  bool live = token < (int64_t)a.B * a.T;
  int32_t b = 0, t = 0, at = 0, page = -1;
  int64_t row = 0;
  if (live) {
    b = kb_fastdiv((int32_t)token, a.fd_T);
    t = (int32_t)token - b * a.T;
    const int32_t n = a.new_lens ? kb_clamp_len(a.new_lens[b * a.new_lens_b], a.T) : a.T;
    row = (int64_t)a.c.lens[b * a.c.lens_b] - n + t;
    live = t < n && row >= 0 && row < a.c.capacity;
  }
  if (live) {
    page = a.c.locate(b, (int32_t)row, at);
    const int32_t position = a.positions ? a.positions[b * a.pos_b + t * a.pos_t] : (int32_t)row;
    for (int32_t h = h0 + lane; h < h1; h += lanes) {
      if (a.weights) a.weights[b * a.w_b + h * a.w_h + row] = 0.f;
      if (a.row_positions) a.row_positions[b * a.p_b + h * a.p_h + row] = position;
    }
  }
  live = live && page >= 0;
  if (!__any_sync(0xffffffffu, live)) return;
  // One head's keys and values in flight per thread leave room for more threads.  8 prompts of 4096-8192 tokens into 8-bit pages take 62 us with one,
  // 65 with two, 68 with four (eight elements per thread; sixteen: 53 us, 4.9 TB/s for the 41 398 tokens that they hold).
  constexpr int kHeadsAtOnce = kF8 ? 1 : 2;
  using Out = typename std::conditional<kF8, uint8_t, T>::type;
  const T* from[2];
  Out* to[2];
  float* scale_to[2];
#pragma unroll
  for (int w = 0; w < 2; ++w) from[w] = static_cast<const T*>(a.x[w]) + b * a.sb[w] + t * a.st[w] + d * a.sd[w] + h0 * a.sh[w];
  to[0] = reinterpret_cast<Out*>(a.c.k) + page * a.c.k_page + at * a.c.k_row + h0 * a.c.k_head + d;
  to[1] = reinterpret_cast<Out*>(a.c.v) + page * a.c.v_page + at * a.c.v_row + h0 * a.c.v_head + d;
  if constexpr (kF8) {
    scale_to[0] = a.c.k_scale + page * a.c.ks_page + at * a.c.ks_row + h0 * a.c.ks_head;
    scale_to[1] = a.c.v_scale + page * a.c.vs_page + at * a.c.vs_row + h0 * a.c.vs_head;
  }
  const int64_t head[2] = {a.c.k_head, a.c.v_head}, scale_head[2] = {a.c.ks_head, a.c.vs_head};
  for (int32_t h2 = h0; h2 < h1; h2 += kHeadsAtOnce) {
    Several<T, kPerThread> e[kHeadsAtOnce][2];
#pragma unroll
    for (int u = 0; u < kHeadsAtOnce; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        if (live && h2 + u < h1) {
          load_several<T, kPerThread, kAligned>(e[u][w], from[w], a.sd[w]);
        } else {
#pragma unroll
          for (int i = 0; i < kPerThread; ++i) e[u][w].v[i] = from_f32<T>(0.f);
        }
        from[w] += a.sh[w];
      }
#pragma unroll
    for (int u = 0; u < kHeadsAtOnce; ++u)
#pragma unroll
      for (int w = 0; w < 2; ++w) {
        const bool write = live && h2 + u < h1;
        if constexpr (kF8) {
          uint32_t m = largest_bits(e[u][w]);
          for (int s = lanes / 2; s > 0; s >>= 1) m = max(m, __shfl_xor_sync(0xffffffffu, m, s));
          float scale = __fmul_rn(__uint_as_float(m), 1.f / 448.f);
          if (scale < 1e-12f) scale = 1e-12f;  // (a NaN stays)
          if (write) {
            if (lane == 0) *scale_to[w] = scale;
            store_several<uint8_t, kPerThread, kAligned>(to[w], quantize(e[u][w], scale, 1.f / scale));
          }
          scale_to[w] += scale_head[w];
        } else if (write) {
          store_several<T, kPerThread, kAligned>(to[w], e[u][w]);
        }
        to[w] += head[w];
      }
  }
}

template <typename T>
int launch_write(const WriteArgs& in, bool f8, bool aligned, cudaStream_t s) {
  WriteArgs a = in;
  const int64_t tokens = (int64_t)a.B * a.T, each = kWriteThreads / (a.D / (f8 ? elements_per_thread<T, true>() : elements_per_thread<T, false>()));
  const int64_t ctas = (tokens + each - 1) / each;
  // few tokens: the heads go to blocks of their own
  a.heads_per_cta = ctas >= 148 * 4 ? a.H_kv : kb_min_i32(2, a.H_kv);
  const dim3 grid((unsigned)ctas, (unsigned)kb_cdiv_i32(a.H_kv, a.heads_per_cta));
  if (f8) {
    if (aligned) paged_write_kernel<T, true, true><<<grid, kWriteThreads, 0, s>>>(a);
    else paged_write_kernel<T, true, false><<<grid, kWriteThreads, 0, s>>>(a);
  } else {
    if (aligned) paged_write_kernel<T, false, true><<<grid, kWriteThreads, 0, s>>>(a);
    else paged_write_kernel<T, false, false><<<grid, kWriteThreads, 0, s>>>(a);
  }
  KB_LAUNCH_CHECK("paged_write_kernel");
  return KB_OK;
}

// ---- evict -----------------------------------------------------------------------------------------------------------

constexpr int kMoveThreads = 256;
constexpr int kKeys = 16, kWarpRows = 32 * kKeys;     // rows of a warp whose keys its lanes hold
constexpr int kBlockRows = 32 * kWarpRows, kMostCluster = 8;

struct EvictArgs {
  PagedView c;
  const float* weights;
  const int32_t* positions;
  float* weights_out;
  int32_t* positions_out;
  int32_t* lens_out;
  int64_t w_b, w_h, p_b, p_h, wo_b, wo_h, po_b, po_h, lens_out_b;
  int32_t H_kv, D, budget, recent, most_moves, elsize, cluster;
  int32_t* counts;  // [B, H_kv]
  int32_t* src;     // [B, H_kv, most_moves]
  int32_t* dst;
  bool in_place;
};

// Weights as whole numbers of the same order; a NaN is below them all, the newest rows are above.  (Where those alone are more than the budget, a second
// search ranks them by their positions; see `by_position`.)
__device__ __forceinline__ uint32_t rank_key(float w, bool newest) {
  if (newest) return 0xffffffffu;
  const uint32_t u = __float_as_uint(w + 0.f);  // (one zero)
  if (w != w) return 0u;
  return (u & 0x80000000u) ? ~u : (u | 0x80000000u);
}

// The newest rows by their positions, the others behind them (0: does not count).
__device__ __forceinline__ uint32_t position_key(int32_t position, int64_t from) { return position > from ? (uint32_t)(position - from) : 0u; }

// What the warps of a cluster's blocks have in common.  Each value goes through shared memory once; buffers alternate, so that one
// barrier per value is enough.
struct Team {
  int (*red)[32];       // [2][warps]: this block's
  int (*of_rank)[8];    // [2][ranks]
  int size, rank, turn; // of the cluster

  // Every thread of the cluster's blocks.  (The barrier wants whole warps that are together again, which code that only some lanes run leaves open.)
  static __device__ __forceinline__ void meet() {
    __syncwarp();
    sm100::cluster_sync_all();
  }
  // `x` into `to`, a variable of every block's shared memory
  __device__ __forceinline__ void tell(uint32_t* to, uint32_t x) const {
    if (size == 1) {
      *to = x;
      return;
    }
    for (int r = 0; r < size; ++r) {
      uint32_t there;
      asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(there) : "r"(sm100::smem_u32(to)), "r"(r));
      asm volatile("st.shared::cluster.u32 [%0], %1;" ::"r"(there), "r"(x) : "memory");
    }
  }
  // op over the team's warps of `x` (the same in a warp's lanes); `before`: over the warps before this one only
  template <typename Op>
  __device__ __forceinline__ int all(int x, int none, Op op, int* before = nullptr) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
    int(&buf)[32] = red[turn];
    if (lane == 0) buf[warp] = x;
    __syncthreads();
    const int mine = lane < warps ? buf[lane] : none;
    int sum = op(mine);
    if (before) *before = op(lane < warp ? mine : none);
    if (size > 1) {
      if (threadIdx.x < size) {
        uint32_t to;
        asm("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(to) : "r"(sm100::smem_u32(&of_rank[turn][rank])), "r"(threadIdx.x));
        asm volatile("st.shared::cluster.s32 [%0], %1;" ::"r"(to), "r"(sum) : "memory");
      }
      meet();
      const int theirs = lane < size ? of_rank[turn][lane] : none;
      if (before) {
        const int lower = op(lane < rank ? theirs : none);
        *before = op(lane == 0 ? *before : lane == 1 ? lower : none);
      }
      sum = op(theirs);
    }
    turn ^= 1;
    return sum;
  }
  __device__ __forceinline__ int sum(int x, int* before = nullptr) {
    return all(x, 0, [](int v) { return __reduce_add_sync(0xffffffffu, v); }, before);
  }
  __device__ __forceinline__ int max(int x) {
    return all(x, INT32_MIN, [](int v) { return __reduce_max_sync(0xffffffffu, v); });
  }
};

// A team (a block, or a cluster of them) per sequence and head.
struct SelectHead {
  const float* w;
  const int32_t* pos;
  float* wo;
  int32_t* po;
  int32_t* count;
  int64_t list;  // where its moves go
  int32_t b, n;

  __device__ __forceinline__ SelectHead(const EvictArgs& a, int32_t b, int32_t h) : b(b) {
    n = a.c.rows(b);
    w = a.weights + b * a.w_b + h * a.w_h;
    pos = a.positions + b * a.p_b + h * a.p_h;
    wo = a.weights_out + b * a.wo_b + h * a.wo_h;
    po = a.positions_out + b * a.po_b + h * a.po_h;
    count = a.counts + (int64_t)b * a.H_kv + h;
    list = ((int64_t)b * a.H_kv + h) * a.most_moves;
  }
  // Whether some of the sequence's rows have no page (every thread of the block calls).
  __device__ __forceinline__ bool lacks_pages(const EvictArgs& a) const {
    const int32_t pages = kb_fastdiv(n - 1, a.c.fd_page) + 1;
    bool lacks = false;
    for (int32_t m = threadIdx.x; m < pages; m += blockDim.x) lacks |= !a.c.has_page(b, m);
    return __syncthreads_or(lacks);
  }
  __device__ __forceinline__ bool has_page(const EvictArgs& a, int32_t row) const { return a.c.has_page(b, kb_fastdiv(row, a.c.fd_page)); }
};

// Keys in registers.  Warp w of the team has the rows [w kWarpRows, (w + 1) kWarpRows), 32 at a time so that ranks within it are ballots.
// The threshold, the least key that stays, is found bit by bit from the top: a count of the keys that reach it with the bit set.  A
// dozen bits leave few keys between what surely stays and what surely goes; once they fit, one per thread, only they are counted.
// Bound by its instructions: 128 heads of 6 000-16 384 rows take 21 us (one block per SM), 256 heads of 2 049 rows 8 us.
__global__ void __launch_bounds__(1024) paged_select_kernel(const EvictArgs a) {
  __shared__ int red[2][32], of_rank[2][8];
  __shared__ uint32_t few[1024];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Team team{red, of_rank, a.cluster, (int)blockIdx.x % a.cluster, 0};
  const SelectHead s(a, blockIdx.y, blockIdx.x / a.cluster);
  const int32_t n = s.n, row0 = (team.rank * warps + warp) * kWarpRows + lane;
  if (a.cluster > 1) team.meet();  // (a block's shared memory may be written once the block has started)

  uint32_t key[kKeys], live = 0;  // live: the rows that count
  int64_t from;                   // positions above it are among the newest
  int32_t rows = n, budget = a.budget;
  {
    float x[kKeys];
    int32_t y[kKeys];
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int i = row0 + j * 32;
      x[j] = i < n ? s.w[i] : 0.f;
      y[j] = i < n ? s.pos[i] : INT32_MIN;
      live |= (uint32_t)(i < n) << j;
    }
    int32_t newest = INT32_MIN;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const int i = row0 + j * 32;
      if (!a.in_place && i < n && i < a.budget) s.wo[i] = x[j], s.po[i] = y[j];
      newest = max(newest, y[j]);
    }
    if (n <= a.budget) {
      if (threadIdx.x == 0 && team.rank == 0) *s.count = 0;
      return;
    }
    newest = team.max(__reduce_max_sync(0xffffffffu, newest));
    from = (int64_t)newest - a.recent;
    if (s.lacks_pages(a)) {
      // those rows hold nothing and can hold nothing: as many of the others stay as there are places with a page
      int places = 0;
#pragma unroll
      for (int j = 0; j < kKeys; ++j) {
        const int i = row0 + j * 32;
        if (i < n && !s.has_page(a, i)) live &= ~(1u << j);
        places += ((live >> j) & 1) && i < a.budget;
      }
      budget = team.sum(__reduce_add_sync(0xffffffffu, places));
      rows = team.sum(__reduce_add_sync(0xffffffffu, __popc(live)));
      if (budget == 0 || budget == rows) {
        if (threadIdx.x == 0 && team.rank == 0) *s.count = 0;
        return;
      }
    }
#pragma unroll
    for (int j = 0; j < kKeys; ++j) key[j] = (live >> j) & 1 ? rank_key(x[j], y[j] > from) : 0u;  // (0: does not count below)
  }
  uint32_t least;
  int reached, over;  // keys that reach `least`, and those above what the bits to come can make of it
  for (bool by_position = false;; by_position = true) {
    uint32_t bit = 0x80000000u;
    least = 0, reached = rows, over = 0;
    for (; bit && reached != budget && reached - over > (int)blockDim.x; bit >>= 1) {
      int reach = 0;
#pragma unroll
      for (int j = 0; j < kKeys; ++j) reach += key[j] >= (least | bit);
      reach = team.sum(__reduce_add_sync(0xffffffffu, reach));
      if (reach >= budget) least |= bit, reached = reach;
      else over = reach;
    }
    if (bit && reached != budget) {
      // every block of the team gets all of them and goes on by itself
      const uint32_t most = least + (bit - 1) + bit;  // (no more than 2^32 - 1)
      const int many = reached - over, others = over;
      uint32_t picked = 0;
#pragma unroll
      for (int j = 0; j < kKeys; ++j) picked |= (uint32_t)(key[j] >= least && key[j] <= most && (live >> j & 1)) << j;
      int at = __popc(picked), before;
#pragma unroll
      for (int x = 1; x < 32; x <<= 1) {
        const int y = __shfl_up_sync(0xffffffffu, at, x);
        if (lane >= x) at += y;
      }
      team.sum(__shfl_sync(0xffffffffu, at, 31), &before);
      at += before - __popc(picked);
#pragma unroll
      for (int j = 0; j < kKeys; ++j)
        if ((picked >> j) & 1) team.tell(&few[at++], key[j]);
      if (team.size > 1) team.meet();
      else __syncthreads();
      const bool here = threadIdx.x < many;
      const uint32_t mine = here ? few[threadIdx.x] : 0u;
      for (; bit && reached != budget; bit >>= 1) {
        const int reach = others + __syncthreads_count(here && mine >= (least | bit));
        if (reach >= budget) least |= bit, reached = reach;
        else over = reach;
      }
    }
    if (by_position || least != 0xffffffffu || reached == budget) break;
    // the newest rows are too many: the newest of them stay
#pragma unroll
    for (int j = 0; j < kKeys; ++j) key[j] = (live >> j) & 1 ? position_key(s.pos[row0 + j * 32], from) : 0u;
  }
  let_next_launch_start();
  // which rows stay; of those that equal the threshold, where there are too many, the lowest
  uint32_t keep = 0;
#pragma unroll
  for (int j = 0; j < kKeys; ++j) keep |= (uint32_t)(key[j] >= least) << j;
  keep &= live;
  if (reached != budget) {
    int equal = 0, before;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) equal += key[j] == least && (live >> j & 1);
    team.sum(__reduce_add_sync(0xffffffffu, equal), &before);
    const int ties = budget - over;
#pragma unroll
    for (int j = 0; j < kKeys; ++j) {
      const bool tie = key[j] == least && (live >> j & 1);
      const uint32_t eq = __ballot_sync(0xffffffffu, tie);
      if (tie && before + __popc(eq & ((1u << lane) - 1)) >= ties) keep &= ~(1u << j);
      before += __popc(eq);
    }
  }
  uint32_t hole = 0, mover = 0;
#pragma unroll
  for (int j = 0; j < kKeys; ++j) {
    const int i = row0 + j * 32;
    const bool stays = (keep >> j) & 1;
    hole |= (uint32_t)(i < a.budget && !stays) << j;
    mover |= (uint32_t)(i >= a.budget && stays) << j;
  }
  hole &= live;
  int hole_at, mover_at;
  team.sum(__reduce_add_sync(0xffffffffu, __popc(hole)), &hole_at);
  const int moves = team.sum(__reduce_add_sync(0xffffffffu, __popc(mover)), &mover_at);
  if (threadIdx.x == 0 && team.rank == 0) *s.count = moves;
  const uint32_t below = (1u << lane) - 1;
#pragma unroll
  for (int j = 0; j < kKeys; ++j) {
    const uint32_t hb = __ballot_sync(0xffffffffu, (hole >> j) & 1), mb = __ballot_sync(0xffffffffu, (mover >> j) & 1);
    if ((hole >> j) & 1) a.dst[s.list + hole_at + __popc(hb & below)] = row0 + j * 32;
    if ((mover >> j) & 1) a.src[s.list + mover_at + __popc(mb & below)] = row0 + j * 32;
    hole_at += __popc(hb), mover_at += __popc(mb);
  }
}

// The same for more rows than a cluster's registers hold: keys are formed again from memory whenever they are needed.
__global__ void __launch_bounds__(1024) paged_select_long_kernel(const EvictArgs a) {
  __shared__ int red[2][32], of_rank[2][8];
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, warps = blockDim.x >> 5;
  Team team{red, of_rank, a.cluster, (int)blockIdx.x % a.cluster, 0};
  const SelectHead s(a, blockIdx.y, blockIdx.x / a.cluster);
  if (a.cluster > 1) team.meet();
  const int per_warp = kb_cdiv_i32(kb_max_i32(s.n, 1), a.cluster * warps * 32) * 32;
  const int begin = kb_min_i32((team.rank * warps + warp) * per_warp, s.n), end = kb_min_i32(begin + per_warp, s.n);
  const uint32_t below = (1u << lane) - 1;
  int32_t newest = INT32_MIN;
  for (int i = begin + lane; i < end; i += 32) {
    if (!a.in_place && i < a.budget) s.wo[i] = s.w[i], s.po[i] = s.pos[i];
    newest = max(newest, s.pos[i]);
  }
  if (s.n <= a.budget) {
    if (threadIdx.x == 0 && team.rank == 0) *s.count = 0;
    return;
  }
  newest = team.max(__reduce_max_sync(0xffffffffu, newest));
  const int64_t from = (int64_t)newest - a.recent;
  const bool lacks = s.lacks_pages(a);
  bool by_position = false;
  // f(key, row, whether there is such a row) for the warp's rows, all lanes together
  auto each = [&](auto f) {
    for (int i0 = begin; i0 < end; i0 += 32) {
      const int i = i0 + lane;
      const bool in = i < end && (!lacks || s.has_page(a, i));
      f(!in ? 0u : by_position ? position_key(s.pos[i], from) : rank_key(s.w[i], s.pos[i] > from), i, in);
    }
  };
  int32_t rows = s.n, budget = a.budget;
  if (lacks) {  // as above
    int places = 0, there = 0;
    each([&](uint32_t, int i, bool in) { places += in && i < a.budget, there += in; });
    budget = team.sum(__reduce_add_sync(0xffffffffu, places));
    rows = team.sum(__reduce_add_sync(0xffffffffu, there));
    if (budget == 0 || budget == rows) {
      if (threadIdx.x == 0 && team.rank == 0) *s.count = 0;
      return;
    }
  }
  uint32_t least;
  int reached, over;
  for (;; by_position = true) {
    least = 0, reached = rows, over = 0;
    for (uint32_t bit = 0x80000000u; bit && reached != budget; bit >>= 1) {
      int reach = 0;
      each([&](uint32_t k, int, bool) { reach += k >= (least | bit); });
      reach = team.sum(__reduce_add_sync(0xffffffffu, reach));
      if (reach >= budget) least |= bit, reached = reach;
      else over = reach;
    }
    if (by_position || least != 0xffffffffu || reached == budget) break;
  }
  int ties = INT32_MAX, equal_before = 0;
  if (reached != budget) {
    int equal = 0;
    each([&](uint32_t k, int, bool in) { equal += in && k == least; });
    team.sum(__reduce_add_sync(0xffffffffu, equal), &equal_before);
    ties = budget - over;
  }
  let_next_launch_start();
  int holes = 0, movers = 0, hole_at = 0, mover_at = 0;
#pragma unroll
  for (int pass = 0; pass < 2; ++pass) {
    int ties_seen = equal_before;
    each([&](uint32_t k, int i, bool in) {
      const uint32_t eq = __ballot_sync(0xffffffffu, in && k == least);
      const bool keep = in && (k > least || (k == least && ties_seen + __popc(eq & below) < ties));
      ties_seen += __popc(eq);
      const bool hole = in && !keep && i < a.budget, mover = keep && i >= a.budget;
      const uint32_t hb = __ballot_sync(0xffffffffu, hole), mb = __ballot_sync(0xffffffffu, mover);
      if (pass) {
        if (hole) a.dst[s.list + hole_at + __popc(hb & below)] = i;
        if (mover) a.src[s.list + mover_at + __popc(mb & below)] = i;
        hole_at += __popc(hb), mover_at += __popc(mb);
      } else {
        holes += __popc(hb), movers += __popc(mb);
      }
    });
    if (pass == 0) {
      team.sum(holes, &hole_at);
      const int moves = team.sum(movers, &mover_at);
      if (threadIdx.x == 0 && team.rank == 0) *s.count = moves;
    }
  }
}

// A warp takes 32 moves at a time: a lane looks up one of them and moves its entries of the bookkeeping, then the lanes copy the rows together.
// HBM-bound: some 314 000 rows of 512 bytes (keys and values) in 60 us, 5.4 TB/s read and written.
template <bool kAligned>
__global__ void __launch_bounds__(kMoveThreads) paged_move_kernel(const EvictArgs a) {
  constexpr int kUnit = kAligned ? 16 : 1, kAtOnce = 4;
  __shared__ longlong2 k_at[kMoveThreads], v_at[kMoveThreads];  // {from, to} in bytes; from -1: no such row
  const int32_t h = blockIdx.y, b = blockIdx.z, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
  const int64_t bh = (int64_t)b * a.H_kv + h;
  const PagedView& c = a.c;
  wait_for_launch_before();
  // (in place, no other block reads the lengths any more: the rows come from the lists)
  if (blockIdx.x == 0 && h == 0 && threadIdx.x == 0) a.lens_out[b * a.lens_out_b] = min(max(c.lens[b * c.lens_b], 0), a.budget);
  const int32_t moves = a.counts[bh];
  const int units = a.D * a.elsize / kUnit;  // of a row: a power of two
  const int shift = __ffs(units) - 1;
  for (int32_t i0 = (blockIdx.x * (kMoveThreads / 32) + warp) * 32; i0 < moves; i0 += gridDim.x * kMoveThreads) {
    const int32_t many = min(32, moves - i0);
    longlong2 k = make_longlong2(-1, 0), v = k;
    if (lane < many) {
      const int32_t src = a.src[bh * a.most_moves + i0 + lane], dst = a.dst[bh * a.most_moves + i0 + lane];
      int32_t sr, dr;
      const int32_t sp = c.locate(b, src, sr), dp = c.locate(b, dst, dr);
      a.weights_out[b * a.wo_b + h * a.wo_h + dst] = a.weights[b * a.w_b + h * a.w_h + src];
      a.positions_out[b * a.po_b + h * a.po_h + dst] = a.positions[b * a.p_b + h * a.p_h + src];
      if (sp >= 0 && dp >= 0) {
        k = make_longlong2((sp * c.k_page + h * c.k_head + sr * c.k_row) * a.elsize, (dp * c.k_page + h * c.k_head + dr * c.k_row) * a.elsize);
        v = make_longlong2((sp * c.v_page + h * c.v_head + sr * c.v_row) * a.elsize, (dp * c.v_page + h * c.v_head + dr * c.v_row) * a.elsize);
        if (c.k_scale) {
          c.k_scale[dp * c.ks_page + h * c.ks_head + dr * c.ks_row] = c.k_scale[sp * c.ks_page + h * c.ks_head + sr * c.ks_row];
          c.v_scale[dp * c.vs_page + h * c.vs_head + dr * c.vs_row] = c.v_scale[sp * c.vs_page + h * c.vs_head + sr * c.vs_row];
        }
      }
    }
    __syncwarp();
    k_at[threadIdx.x] = k, v_at[threadIdx.x] = v;
    __syncwarp();
    using Unit = typename std::conditional<kAligned, uint4, uint8_t>::type;
    for (int u0 = lane; u0 < many << shift; u0 += 32 * kAtOnce) {
      Unit x[kAtOnce], y[kAtOnce];
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int u = u0 + j * 32, r = warp * 32 + (u >> shift), off = (u & (units - 1)) * kUnit;
        if (u < many << shift && k_at[r].x >= 0) {
          x[j] = *reinterpret_cast<const Unit*>(c.k + k_at[r].x + off);
          y[j] = *reinterpret_cast<const Unit*>(c.v + v_at[r].x + off);
        }
      }
#pragma unroll
      for (int j = 0; j < kAtOnce; ++j) {
        const int u = u0 + j * 32, r = warp * 32 + (u >> shift), off = (u & (units - 1)) * kUnit;
        if (u < many << shift && k_at[r].x >= 0) {
          *reinterpret_cast<Unit*>(c.k + k_at[r].y + off) = x[j];
          *reinterpret_cast<Unit*>(c.v + v_at[r].y + off) = y[j];
        }
      }
    }
  }
}

// Rows of a sequence that can move: kept ones behind the budget, into places before it.
int32_t most_moves(const kb_paged_cache& c, int32_t budget) {
  const int64_t capacity = (int64_t)c.M * c.page;
  return (int32_t)(capacity <= budget ? 0 : kb_min_i32(budget, (int32_t)(capacity - budget)));
}

int launch_select(const EvictArgs& in, int32_t heads, int32_t B, cudaStream_t s) {
  EvictArgs a = in;
  const int32_t capacity = kb_max_i32(1, a.c.capacity);
  a.cluster = 1;
  while (a.cluster < kMostCluster && capacity > a.cluster * kBlockRows) a.cluster *= 2;
  const bool held = capacity <= a.cluster * kBlockRows;
  cudaLaunchConfig_t c = {};
  c.blockDim = dim3(held && a.cluster == 1 ? 32 * kb_cdiv_i32(capacity, kWarpRows) : 1024);
  c.gridDim = dim3((unsigned)(heads * a.cluster), (unsigned)B);
  c.stream = s;
  cudaLaunchAttribute at;
  at.id = cudaLaunchAttributeClusterDimension;
  at.val.clusterDim.x = a.cluster, at.val.clusterDim.y = at.val.clusterDim.z = 1;
  c.attrs = &at, c.numAttrs = a.cluster > 1 ? 1 : 0;
  KB_CUDA_TRY(cudaLaunchKernelEx(&c, held ? paged_select_kernel : paged_select_long_kernel, a));
  count_launch();
  return KB_OK;
}

}  // namespace

int paged_write(const kb_paged_write_params& p, cudaStream_t s) {
  const bool f8 = p.cache.dtype == KB_E4M3;
  if (!f8 && p.cache.dtype != p.dtype) return KB_ERR_UNSUPPORTED;
  if ((int64_t)p.cache.B * p.T > (int64_t)1 << 30) return KB_ERR_TOO_LARGE;
  WriteArgs a{};
  a.c = make_paged_view(p.cache);
  const kb_tensor4* x[2] = {&p.k, &p.v};
  const int elsize = dtype_size(p.dtype);
  bool aligned = paged_rows_aligned(p.cache, dtype_size(p.cache.dtype));
  for (int i = 0; i < 2; ++i) {
    a.x[i] = x[i]->data;
    a.sb[i] = x[i]->stride[0], a.sh[i] = x[i]->stride[1], a.st[i] = x[i]->stride[2], a.sd[i] = x[i]->stride[3];
    aligned = aligned && a.sd[i] == 1 && reinterpret_cast<uintptr_t>(a.x[i]) % 16 == 0 && a.sb[i] * elsize % 16 == 0 && a.sh[i] * elsize % 16 == 0 &&
              a.st[i] * elsize % 16 == 0;
  }
  a.new_lens = p.new_lens, a.new_lens_b = p.new_lens_stride;
  a.positions = p.positions, a.pos_b = p.positions_stride[0], a.pos_t = p.positions_stride[1];
  a.weights = p.weights, a.w_b = p.weights_stride[0], a.w_h = p.weights_stride[1];
  a.row_positions = p.row_positions, a.p_b = p.row_positions_stride[0], a.p_h = p.row_positions_stride[1];
  a.B = p.cache.B, a.H_kv = p.cache.H_kv, a.T = p.T, a.D = p.cache.D;
  a.fd_T = kb_fastdiv_make(a.T);
  switch (p.dtype) {
    case KB_F32: return launch_write<float>(a, f8, aligned, s);
    case KB_F16: return launch_write<__half>(a, f8, aligned, s);
    default: return launch_write<__nv_bfloat16>(a, f8, aligned, s);
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
  a.in_place = p.weights == p.weights_out;
  const size_t heads = (size_t)c.B * c.H_kv;
  a.counts = static_cast<int32_t*>(p.workspace);
  a.src = a.counts + heads;
  a.dst = a.src + heads * a.most_moves;
  if (int rc = launch_select(a, c.H_kv, c.B, s)) return rc;
  // 256 moves per block at a time; a few blocks per head are enough where there are many heads
  const int64_t most = ((int64_t)a.most_moves + kMoveThreads - 1) / kMoveThreads, want = kb_max_i32(1, (int32_t)((148 * 8 + heads - 1) / heads));
  const dim3 grid((unsigned)(most < want ? (most < 1 ? 1 : most) : want), (unsigned)c.H_kv, (unsigned)c.B);
  return launch_after(paged_rows_aligned(c, a.elsize) ? paged_move_kernel<true> : paged_move_kernel<false>, grid, kMoveThreads, s, a);
}

}  // namespace kb
