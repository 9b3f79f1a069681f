// Rotary position embedding with one to four position axes, forward and (with the sign of the angle turned) backward.
//
// Pair i of a head's first `rot` elements -- (i, i + rot / 2), or (2 i, 2 i + 1) when interleaved -- is turned by
//   angle = pos[axis(i)] * inv_freq[i]:   y0 = x0 cos - x1 sin,   y1 = x1 cos + x0 sin;
// the elements behind `rot` are copied.  A rotation's gradient is the rotation by the opposite angle, so the backward pass
// is this kernel with `inverse` set and nothing is saved but the positions.
//
// The product of a far position and a frequency needs more than 32 bits (a position of 10^6 leaves an angle in fp32 off by
// 0.06): it is formed and reduced to [-pi, pi] in 64 bits, sine and cosine of the rest are taken in 32.  Every element is
// computed in 32 bits and rounded once.
//
// Bound by HBM: each element read once and written once.  A CTA owns `tokens` consecutive tokens of a sequence, computes
// their sines and cosines once into shared memory for all heads of query and key, and walks (head, V pairs) items: two 16-byte
// loads and two 16-byte stores each, neighbouring threads on neighbouring pieces of a row.  2 x 4096 tokens, 32 + 8 heads of 128,
// bf16: 32.2 us, 5.2 TB/s (34.2 without the next item's loads ahead; 46.7 with four items' loads at once, for want of warps).
#include "common.cuh"
#include "debug.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256;

struct RotaryArgs {
  B200RotaryParams p;
  int tokens;       // of one CTA
  int pairs;        // rot / 2
};

// Sine and cosine of `pos * freq`.
__device__ __forceinline__ float2 turn_of(double pos, double freq, bool inverse) {
  constexpr double kTwoPi = 6.283185307179586476925286766559, kPerTurn = 0.15915494309189533576888376337251;
  const double a = pos * freq;
  const float r = static_cast<float>(fma(-rint(a * kPerTurn), kTwoPi, a));
  float s, c;
  sincosf(r, &s, &c);
  return make_float2(c, inverse ? -s : s);
}

template <typename T, int V> struct Piece;   // V elements as one load
template <> struct Piece<float, 4> { using type = uint4; };
template <> struct Piece<__half, 8> { using type = uint4; };
template <> struct Piece<__nv_bfloat16, 8> { using type = uint4; };
template <typename T> struct Piece<T, 1> { using type = T; };

// V > 1: unit inner strides, every row on 16 bytes, pairs and the copied tail in whole pieces.
template <typename T, int V>
__global__ void __launch_bounds__(kThreads) rotary_kernel(const RotaryArgs a) {
  using W = typename Piece<T, V>::type;
  extern __shared__ float2 turns[];   // [tokens][pairs]
  const B200RotaryParams& p = a.p;
  const int b = blockIdx.y, l0 = blockIdx.x * a.tokens;
  const int n_tok = p.L - l0 < a.tokens ? p.L - l0 : a.tokens;
  pdl_wait();
  pdl_launch_dependents();
  const int rot_items = a.pairs / V, items = rot_items + (p.D - p.rot + (V > 1 ? 0 : 1)) / (2 * V);   // of one head
  // The heads of the queries, then of the keys.  A thread's place (token, head, item) moves on by fixed steps: dividing for
  // each item cost as much as the rotation.
  // The next item's pieces travel while one is turned, the first ones while the sines and cosines are made.
  auto walk = [&](const T* x, T* y, const int64_t(&xs)[4], const int64_t(&ys)[4], const int heads, auto before) {
    if (heads == 0) return;
    const int64_t xi = V > 1 ? 1 : xs[3], yi = V > 1 ? 1 : ys[3];
    x += b * xs[0] + l0 * xs[2];
    y += b * ys[0] + l0 * ys[2];
    int it = threadIdx.x % items, h = threadIdx.x / items % heads, t = threadIdx.x / items / heads;
    const int d_it = kThreads % items, d_h = kThreads / items % heads, d_t = kThreads / items / heads;
    __align__(16) T u[V], w[V], next_u[V], next_w[V];
    // the two pieces of an item: the halves of V pairs, or 2 V neighbouring elements (V = 1, an odd number to copy: the last twice)
    auto piece0 = [&](int i) { return i >= rot_items ? p.rot + (i - rot_items) * 2 * V : (p.interleaved ? i * 2 * V : i * V); };
    auto piece1 = [&](int i, int e0) {
      if (i >= rot_items) return V > 1 || e0 + 2 <= p.D ? e0 + V : e0;
      return p.interleaved ? e0 + V : e0 + a.pairs;
    };
    auto fetch = [&](int i, int hd, int tk) {
      if (tk >= n_tok) return;
      const int e0 = piece0(i), e1 = piece1(i, e0);
      const T* from = x + hd * xs[1] + tk * xs[2];
      *reinterpret_cast<W*>(next_u) = *reinterpret_cast<const W*>(from + e0 * xi);
      *reinterpret_cast<W*>(next_w) = *reinterpret_cast<const W*>(from + e1 * xi);
    };
    fetch(it, h, t);
    before();
    while (t < n_tok) {
      const int e0 = piece0(it), e1 = piece1(it, e0);
      const bool tail = it >= rot_items;
      *reinterpret_cast<W*>(u) = *reinterpret_cast<const W*>(next_u);
      *reinterpret_cast<W*>(w) = *reinterpret_cast<const W*>(next_w);
      const int at_it = it, at_h = h, at_t = t;
      it += d_it;
      h += d_h;
      t += d_t;
      if (it >= items) {
        it -= items;
        ++h;
      }
      if (h >= heads) {
        h -= heads;
        ++t;
      }
      fetch(it, h, t);
      if (!tail) {
        const float2* cs = turns + at_t * a.pairs + at_it * V;
        if (p.interleaved && V > 1) {
          // piece u holds pairs 0 .. V/2 - 1, piece w the others
#pragma unroll
          for (int e = 0; e + 1 < V; e += 2) {
            const float2 c0 = cs[e / 2], c1 = cs[V / 2 + e / 2];
            const float u0 = to_f32<T>(u[e]), u1 = to_f32<T>(u[e + 1]), w0 = to_f32<T>(w[e]), w1 = to_f32<T>(w[e + 1]);
            u[e] = from_f32<T>(fmaf(-u1, c0.y, u0 * c0.x));
            u[e + 1] = from_f32<T>(fmaf(u0, c0.y, u1 * c0.x));
            w[e] = from_f32<T>(fmaf(-w1, c1.y, w0 * c1.x));
            w[e + 1] = from_f32<T>(fmaf(w0, c1.y, w1 * c1.x));
          }
        } else {
#pragma unroll
          for (int e = 0; e < V; ++e) {
            const float2 c = cs[e];
            const float x0 = to_f32<T>(u[e]), x1 = to_f32<T>(w[e]);
            u[e] = from_f32<T>(fmaf(-x1, c.y, x0 * c.x));
            w[e] = from_f32<T>(fmaf(x0, c.y, x1 * c.x));
          }
        }
      }
      if (dbg_bhrc(p.status, DBG_ROTARY * 100 + 1, b, p.B, at_h, heads, l0 + at_t, p.L, e0, V, p.D) &&
          dbg_range(p.status, DBG_ROTARY * 100 + 2, e1, V, p.D)) {
        T* to = y + at_h * ys[1] + at_t * ys[2];
        *reinterpret_cast<W*>(to + e0 * yi) = *reinterpret_cast<const W*>(u);
        *reinterpret_cast<W*>(to + e1 * yi) = *reinterpret_cast<const W*>(w);
      }
    }
  };
  auto make_turns = [&]() {
    for (int i = threadIdx.x; i < n_tok * a.pairs; i += kThreads) {
      const int t = i / a.pairs, pair = i - t * a.pairs;
      int axis = 0, end = p.section[0];
      while (axis + 1 < p.axes && pair >= end) end += p.section[++axis];
      const int64_t at = axis * p.pos_stride[0] + b * p.pos_stride[1] + (l0 + t) * p.pos_stride[2];
      const double pos = p.positions_i64 ? static_cast<double>(static_cast<const int64_t*>(p.positions)[at])
                                         : static_cast<double>(static_cast<const int32_t*>(p.positions)[at]);
      const double freq = p.inv_freq_f64 ? static_cast<const double*>(p.inv_freq)[pair]
                                         : static_cast<double>(static_cast<const float*>(p.inv_freq)[pair]);
      turns[i] = turn_of(pos, freq, p.inverse != 0);
    }
    __syncthreads();
  };
  walk(static_cast<const T*>(p.x[0]), static_cast<T*>(p.y[0]), p.x_stride[0], p.y_stride[0], p.heads[0], make_turns);
  walk(static_cast<const T*>(p.x[1]), static_cast<T*>(p.y[1]), p.x_stride[1], p.y_stride[1], p.heads[1], [] {});
}

template <typename T, int V> int launch_typed(const RotaryArgs& a, cudaStream_t stream) {
  const int ctas = (a.p.L + a.tokens - 1) / a.tokens;
  const size_t smem = sizeof(float2) * a.tokens * a.pairs;
  if (!launch_pdl(rotary_kernel<T, V>, dim3(ctas, a.p.B), kThreads, smem, stream, a)) return B200_SDPA_ERR_CUDA;
  count_launch(KID_ROTARY);
  return B200_SDPA_OK;
}

bool pieces_ok(const B200RotaryParams& p, int esize, int v) {
  if ((p.rot / 2) % v != 0 || (p.D - p.rot) % (2 * v) != 0) return false;
  for (int w = 0; w < 2; ++w) {
    if (p.heads[w] == 0) continue;
    if (reinterpret_cast<uintptr_t>(p.x[w]) % 16 || reinterpret_cast<uintptr_t>(p.y[w]) % 16) return false;
    const int n[3] = {p.B, p.heads[w], p.L};
    if (p.x_stride[w][3] != 1 || p.y_stride[w][3] != 1) return false;
    for (int i = 0; i < 3; ++i)
      if (n[i] > 1 && ((p.x_stride[w][i] * esize) % 16 || (p.y_stride[w][i] * esize) % 16)) return false;
  }
  return true;
}

}  // namespace

int launch_rotary(const B200RotaryParams& p, cudaStream_t stream) {
  RotaryArgs a;
  a.p = p;
  a.pairs = p.rot / 2;
  // four tokens share a CTA where that still leaves several CTAs for every SM; else each has its own
  a.tokens = static_cast<int64_t>(p.B) * p.L >= 4 * 4 * 148 ? 4 : 1;
  switch (p.dtype) {
    case B200_SDPA_F32: return pieces_ok(p, 4, 4) ? launch_typed<float, 4>(a, stream) : launch_typed<float, 1>(a, stream);
    case B200_SDPA_F16: return pieces_ok(p, 2, 8) ? launch_typed<__half, 8>(a, stream) : launch_typed<__half, 1>(a, stream);
    case B200_SDPA_BF16:
      return pieces_ok(p, 2, 8) ? launch_typed<__nv_bfloat16, 8>(a, stream) : launch_typed<__nv_bfloat16, 1>(a, stream);
    default: return B200_SDPA_ERR_DTYPE;
  }
}

}  // namespace b200
