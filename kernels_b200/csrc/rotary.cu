// Rotary position embedding with positions on several axes: pair d (elements d and d + R of a head, d < R) is turned by
// the angle positions[axis(d)][b][t] * inv_freq[d].  The gradient turns by the opposite angle (`inverse`).
//
// The angle is a whole number times a frequency, and only its part below a full turn matters.  So the frequency is
// taken in turns, as a fraction of 2^64, and multiplied by the position modulo 2^64: the multiplication drops whole
// turns exactly, and at position p the angle is off by at most p * 2^-54 turns (the frequency comes with 53 bits),
// where a product in fp32 would be off by p * 2^-24.
//
// HBM-bound: every element is read and written once, past the caches' order of use (__ldcs, __stcs).  A block takes a few tokens and
// forms the cosines and sines of their pairs once, in shared memory; then its threads, each with one vector of pairs of one
// token, walk over the heads, several of them side by side.
// 4 x 8192 tokens, 32 + 8 heads of 128, bf16: 119 us, 5.6 TB/s (0.86 of the measured copy); 8 x 4095 tokens, 16 + 16 heads of 64, f16,
// forward and backward: 121 us; 64 tokens: 3.5 us on the device.
#include "common.cuh"

namespace kb {
namespace {

constexpr int kThreads = 256, kMaxAxes = 8;

struct RotaryArgs {
  const void* x[2];   // q, k
  void* y[2];
  int64_t sb[2], sh[2], st[2], sd[2];
  int32_t heads[2];
  const void* positions;
  int64_t pos_axis, pos_b, pos_t;
  const double* inv_freq;
  int32_t B, T, D, R, axes, pos64, inverse;
  int32_t section_end[kMaxAxes];
  int32_t vecs, tokens;    // vectors of pairs per token, tokens per block: both powers of two
  int32_t heads_per_cta;
  KbFastDiv fd_T, fd_R;
};

template <typename T, int E> struct alignas(E * sizeof(T)) Elems { T v[E]; };

template <typename T, int E>
__device__ __forceinline__ void load_elems(const T* p, int64_t sd, Elems<T, E>& e) {
  if constexpr (E * sizeof(T) == 16) {
    *reinterpret_cast<uint4*>(&e) = __ldcs(reinterpret_cast<const uint4*>(p));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) e.v[i] = p[i * sd];
  }
}
template <typename T, int E>
__device__ __forceinline__ void store_elems(T* p, const Elems<T, E>& e) {
  if constexpr (E * sizeof(T) == 16) {
    __stcs(reinterpret_cast<uint4*>(p), *reinterpret_cast<const uint4*>(&e));
  } else {
#pragma unroll
    for (int i = 0; i < E; ++i) p[i] = e.v[i];
  }
}

constexpr int kMostPairs = 512;  // of a block's tokens

// cos and sin of the angle of pair d of a token
__device__ __forceinline__ float2 turn_of(const RotaryArgs& a, int32_t b, int32_t t, int32_t d) {
  int32_t axis = 0;
  while (axis < a.axes - 1 && d >= a.section_end[axis]) ++axis;
  const int64_t at = axis * a.pos_axis + b * a.pos_b + t * a.pos_t;
  const int64_t pos = a.pos64 ? static_cast<const int64_t*>(a.positions)[at] : static_cast<const int32_t*>(a.positions)[at];
  const double turns = a.inv_freq[d] * 0.15915494309189535;  // 1 / (2 pi)
  const uint64_t frac = (uint64_t)((turns - floor(turns)) * 18446744073709551616.0);
  const int64_t angle = (int64_t)((uint64_t)pos * frac);  // [-1/2, 1/2) turns
  float2 r;
  sincospif((float)angle * 1.0842021724855044e-19f, &r.y, &r.x);  // 2^-63: half turns
  if (a.inverse) r.y = -r.y;
  return r;
}

// E: pairs per thread.  Vectors [0, R / E) hold pairs, the ones behind them what of a head is not rotated, cut in two halves.
template <typename T, int E>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  __shared__ __align__(16) float2 turns[kMostPairs];
  const int64_t token0 = (int64_t)blockIdx.x * a.tokens, all_tokens = (int64_t)a.B * a.T;
  for (int i = threadIdx.x; i < a.tokens * a.R; i += kThreads) {
    const int32_t k = kb_fastdiv(i, a.fd_R), d = i - k * a.R;
    if (token0 + k < all_tokens) {
      const int32_t b = kb_fastdiv((int32_t)(token0 + k), a.fd_T);
      turns[i] = turn_of(a, b, (int32_t)(token0 + k) - b * a.T, d);
    }
  }
  __syncthreads();
  const int vec = threadIdx.x & (a.vecs - 1), rest_of = threadIdx.x / a.vecs, k = rest_of & (a.tokens - 1), head = rest_of / a.tokens;
  const int head_lanes = kThreads / (a.vecs * a.tokens);
  if (token0 + k >= all_tokens) return;
  const int32_t b = kb_fastdiv((int32_t)(token0 + k), a.fd_T), t = (int32_t)(token0 + k) - b * a.T;
  const int32_t rot_vecs = a.R / E;
  const bool turned = vec < rot_vecs;
  const int32_t rest = a.D / 2 - a.R;  // half of what is not rotated
  const int32_t d0 = turned ? vec * E : 2 * a.R + (vec - rot_vecs) * E;
  const int32_t d1 = d0 + (turned ? a.R : rest);
  float c[E], s[E];
  if (turned) {
#pragma unroll
    for (int e = 0; e < E; ++e) {
      const float2 r = turns[k * a.R + d0 + e];
      c[e] = r.x, s[e] = r.y;
    }
  }
  const int32_t all = a.heads[0] + a.heads[1];
  const int32_t h0 = blockIdx.y * a.heads_per_cta, h1 = min(h0 + a.heads_per_cta, all);
#pragma unroll 4
  for (int32_t hh = h0 + head; hh < h1; hh += head_lanes) {
    const int which = hh >= a.heads[0];
    const int32_t h = which ? hh - a.heads[0] : hh;
    const T* x = static_cast<const T*>(a.x[which]) + b * a.sb[which] + h * a.sh[which] + t * a.st[which];
    T* y = static_cast<T*>(a.y[which]) + (((int64_t)b * a.heads[which] + h) * a.T + t) * a.D;
    Elems<T, E> u, w;
    load_elems<T, E>(x + d0 * a.sd[which], a.sd[which], u);
    load_elems<T, E>(x + d1 * a.sd[which], a.sd[which], w);
    if (turned) {
#pragma unroll
      for (int e = 0; e < E; ++e) {
        const float p = to_f32(u.v[e]), r = to_f32(w.v[e]);
        u.v[e] = from_f32<T>(p * c[e] - r * s[e]);
        w.v[e] = from_f32<T>(r * c[e] + p * s[e]);
      }
    }
    store_elems<T, E>(y + d0, u);
    store_elems<T, E>(y + d1, w);
  }
}

bool vectors_ok(const kb_tensor4& x, const void* y, int E) {
  if (!x.data) return true;
  if (x.stride[3] != 1 || reinterpret_cast<uintptr_t>(x.data) % 16 || reinterpret_cast<uintptr_t>(y) % 16) return false;
  return x.stride[0] % E == 0 && x.stride[1] % E == 0 && x.stride[2] % E == 0;
}

template <typename T, int E>
int launch(const RotaryArgs& in, cudaStream_t s) {
  RotaryArgs a = in;
  a.vecs = a.D / 2 / E;
  // a quarter of the block's threads for a head (of 128 pairs at most), so that four heads or more are under way
  a.tokens = a.vecs >= kThreads / 4 ? 1 : kThreads / 4 / a.vecs;
  while (a.tokens * a.R > kMostPairs) a.tokens /= 2;
  a.fd_T = kb_fastdiv_make(a.T), a.fd_R = kb_fastdiv_make(a.R);
  const int64_t ctas = ((int64_t)a.B * a.T + a.tokens - 1) / a.tokens;
  const int32_t all = a.heads[0] + a.heads[1], lanes = kThreads / (a.vecs * a.tokens);
  // few tokens: the heads go to blocks of their own, at the price of the angles formed again in each
  int32_t groups = (int32_t)(ctas >= 148 * 4 ? 1 : (148 * 4 + ctas - 1) / ctas);
  const int32_t most = (all + lanes - 1) / lanes;
  groups = groups > most ? most : groups;
  a.heads_per_cta = ((all + groups - 1) / groups + lanes - 1) / lanes * lanes;
  groups = (all + a.heads_per_cta - 1) / a.heads_per_cta;
  rotary_kernel<T, E><<<dim3((unsigned)ctas, (unsigned)groups), kThreads, 0, s>>>(a);
  KB_LAUNCH_CHECK("rotary_kernel");
  return KB_OK;
}

template <typename T>
int by_alignment(const kb_rotary_params& p, const RotaryArgs& a, cudaStream_t s) {
  constexpr int E = 16 / sizeof(T);
  if (vectors_ok(p.q, p.q_out, E) && vectors_ok(p.k, p.k_out, E) && p.R % E == 0 && (p.D / 2 - p.R) % E == 0) return launch<T, E>(a, s);
  return launch<T, 1>(a, s);
}

}  // namespace

int rotary(const kb_rotary_params& p, cudaStream_t s) {
  RotaryArgs a{};
  const kb_tensor4* x[2] = {&p.q, &p.k};
  void* y[2] = {p.q_out, p.k_out};
  const int32_t heads[2] = {p.H, p.k.data ? p.H_kv : 0};
  for (int i = 0; i < 2; ++i) {
    a.x[i] = x[i]->data, a.y[i] = y[i], a.heads[i] = heads[i];
    a.sb[i] = x[i]->stride[0], a.sh[i] = x[i]->stride[1], a.st[i] = x[i]->stride[2], a.sd[i] = x[i]->stride[3];
  }
  a.positions = p.positions;
  a.pos_axis = p.pos_stride[0], a.pos_b = p.pos_stride[1], a.pos_t = p.pos_stride[2];
  a.inv_freq = p.inv_freq;
  a.B = p.B, a.T = p.T, a.D = p.D, a.R = p.R, a.axes = p.axes, a.pos64 = p.pos64, a.inverse = p.inverse;
  for (int i = 0; i < p.axes; ++i) a.section_end[i] = p.section_end[i];
  switch (p.dtype) {
    case KB_F32: return by_alignment<float>(p, a, s);
    case KB_F16: return by_alignment<__half>(p, a, s);
    default: return by_alignment<__nv_bfloat16>(p, a, s);
  }
}

}  // namespace kb
