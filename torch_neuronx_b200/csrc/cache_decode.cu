// One query row per sequence against a paged cache: the 8-bit cache, and a prefix that the whole batch shares.
//
// With a shared prefix of P keys the softmax runs over P + kv_lens[b] keys, but only the sequence's own keys differ:
//   * prefix: the batch's query rows are the rows of one attention problem (B * group rows for each kv head against P
//     keys, no mask), so its keys are read once for all of them and multiplied by full tensor-core tiles -- the split form
//     of the prefill kernel (prefill_sm100.cu), whose fp32 partials stay in the scratch; probabilities enter its second product as the
//     own keys' do, rounded to the type of a 16-bit cache, as two 16-bit parts for an 8-bit one;
//   * own keys: split-KV decode (decode_mma.cu, decode_fp8.cu), partials beside them;
//   * one merge over both lists, exact in the usual way: o = sum 2^(m_i - m) o_i / sum 2^(m_i - m) l_i.
// Bound by HBM: (P + sum of own lengths) Hkv rows once; the prefix's products by the tensor cores from about 60 sequences
// on (32 / 8 heads).  64 sequences under 16384 + 16..1000 keys: 67 us (bytes and products: 31), of which the prefix's tiles 15, their
// start and end 9.  128 sequences under 8192 + 16..500 keys of an 8-bit cache: 76 us.
#include "common.cuh"
#include "debug.cuh"

namespace b200 {

// cache_rows.cu: rows [0, n) of the table's pages, dense in the rows' dtype (scales null: a copy of 16-bit rows)
// `beside`: the launch before it in the stream is none of its inputs' (it waits for it at its end, so that whoever waits for this one
// waits for both)
int launch_cache_gather(const B200CacheRowsParams& p, bool beside, cudaStream_t stream);

namespace {

constexpr float kLn2 = 0.6931471805599453f;
constexpr int kCombineWarps = 4;

// Rows of partials: o [row][D], ml [row][2]
struct Rows {
  const float* o;
  const float* ml;
};
struct Merge {
  Rows own, prefix;
  int n_prefix;        // of a (query head, sequence)
  int n_own, chunk;    // 16-bit cache: ranges of `chunk` keys, rows (sequence * Hq + head) * n_own + range
  const int2* range;   // 8-bit cache (decode_fp8.cu)
  int heads, units;
  int slots, grid;     // 8-bit cache: slots there are, and the most that one pair has
  int front;           // the prefix's partials are among these too, each sequence's before its own (16-bit: so many of them)
};

// WARPS warps for each (sequence, query head), 4 / WARPS rows in a CTA: the prefix's partials (rows (h * B + b) * n ..) and the own
// ones in use.  Bound by latency: the (maximum, sum) pairs are read at once, one a lane, then the rows eight at a time.  One warp where
// there are rows enough to fill the GPU, four where the ranges are many and the rows few.
template <typename T, int D, int WARPS>
__global__ void __launch_bounds__(kCombineWarps * 32) cache_combine_kernel(const Problem p, const Merge a) {
  constexpr int C = D / 32, kChunk = 32 * WARPS;   // columns per lane, ranges whose weights are held at a time
  __shared__ float sm_w[kCombineWarps / WARPS][kChunk];
  __shared__ float sm_o[WARPS > 1 ? kCombineWarps : 1][D], sm_x[kCombineWarps];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, sub = warp % WARPS, lane_w = sub * 32 + lane;
  const int64_t id = static_cast<int64_t>(blockIdx.x) * (kCombineWarps / WARPS) + warp / WARPS;
  pdl_wait();
  pdl_launch_dependents();
  if (id >= static_cast<int64_t>(p.B) * p.Hq) return;   // (whole warps; with four to a row the grid is exact)
  const int h = static_cast<int>(id % p.Hq), b = static_cast<int>(id / p.Hq);
  // own partials: rows own0 + s * step; the prefix's: rows pre0 + s * pre_step
  int used = 0, step = 1, n_prefix = a.n_prefix, pre_step = 1;
  int64_t own0 = 0, pre0 = (static_cast<int64_t>(h) * p.B + b) * a.n_prefix;
  bool torn = false;   // a wait ran out in the launch before, and a pair's slots were not noted: anything may stand there
  auto slots_ok = [&](int2 r) { return r.x >= 0 && r.x <= r.y && r.y < a.slots && r.y - r.x < a.grid; };
  if (a.range != nullptr) {
    const int in_group = h % p.group, unit = in_group / a.heads * p.Hkv + h / p.group, twice = a.front != 0 ? 1 : 0;
    step = a.heads;
    if (valid_keys(p, b) > 0) {
      const int2 r = a.range[((static_cast<int64_t>(b) << twice) + twice) * a.units + unit];
      torn = !slots_ok(r);
      used = (r.y - r.x + 1) * kFp8Parts;
      own0 = static_cast<int64_t>(r.x) * kFp8Parts * a.heads + in_group % a.heads;
    }
    if (twice) {
      const int2 r = a.range[(static_cast<int64_t>(b) << 1) * a.units + unit];
      torn = torn || !slots_ok(r);
      n_prefix = (r.y - r.x + 1) * kFp8Parts;
      pre_step = a.heads;
      pre0 = static_cast<int64_t>(r.x) * kFp8Parts * a.heads + in_group % a.heads;
    }
  } else if (a.n_own > 0) {
    used = (valid_keys(p, b) + a.chunk - 1) / a.chunk;
    used = used < 1 ? 1 : (used > a.n_own ? a.n_own : used);
    own0 = (static_cast<int64_t>(b) * p.Hq + h) * (a.front + a.n_own);
    if (a.front > 0) {
      pre0 = own0;
      n_prefix = a.front;
      own0 += a.front;
    }
  }
  if (torn) {   // (for all of the row's warps alike) reported by who gave up; the row is not a number
    if (sub == 0) {
      for (int c = 0; c < C; ++c) reinterpret_cast<T*>(p.out)[b * p.os[0] + h * p.os[1] + (lane * C + c) * p.os[3]] = from_f32<T>(CUDART_NAN_F);
      if (p.lse != nullptr && lane == 0) p.lse[b * p.ls[0] + h * p.ls[1]] = CUDART_NAN_F;
    }
    return;
  }
  if (!dbg_bhrc(p.status, DBG_CACHE_DECODE * 100 + 1, b, p.B, h, p.Hq, 0, 1, lane * C, C, p.Dv)) return;
  auto row_of = [&](int s) { return s < n_prefix ? pre0 + static_cast<int64_t>(s) * pre_step : own0 + static_cast<int64_t>(s - n_prefix) * step; };
  const int total = n_prefix + used;
  auto pair_of = [&](int s) { return *reinterpret_cast<const float2*>((s < n_prefix ? a.prefix.ml : a.own.ml) + row_of(s) * 2); };
  auto together = [&]() {
    if constexpr (WARPS > 1) __syncthreads();
    else __syncwarp();
  };
  float mx = -CUDART_INF_F;
  float2 mine = make_float2(-CUDART_INF_F, 0.f);   // of the first chunk
  for (int s = lane_w; s < total; s += kChunk) {
    const float2 ml = pair_of(s);
    if (s == lane_w) mine = ml;
    mx = fmaxf(mx, ml.x);
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
  if constexpr (WARPS > 1) {
    if (lane == 0) sm_x[warp] = mx;
    __syncthreads();
#pragma unroll
    for (int w = 0; w < WARPS; ++w) mx = fmaxf(mx, sm_x[w]);
  }
  const float ms = (mx == -CUDART_INF_F) ? 0.f : mx;
  float acc[C], lsum = 0.f;
#pragma unroll
  for (int c = 0; c < C; ++c) acc[c] = 0.f;
  for (int s0 = 0; s0 < total; s0 += kChunk) {
    if (s0 > 0) {
      together();   // (the weights before have been used)
      mine = s0 + lane_w < total ? pair_of(s0 + lane_w) : make_float2(-CUDART_INF_F, 0.f);
    }
    // a range without a visible key has the sum 0, and nothing else of it may have been written (a NaN sum counts)
    const float wgt = mine.y != 0.f ? exp2f(mine.x - ms) : 0.f;
    lsum += mine.y != 0.f ? wgt * mine.y : 0.f;
    sm_w[warp / WARPS][lane_w] = wgt;
    together();
    const int n = total - s0 < kChunk ? total - s0 : kChunk;
    for (int s1 = sub; s1 < n; s1 += 8 * WARPS) {
      float v[8][C], w[8];
#pragma unroll
      for (int i = 0; i < 8; ++i) {
        const int s = s1 + i * WARPS;
        w[i] = s < n ? sm_w[warp / WARPS][s] : 0.f;
#pragma unroll
        for (int c = 0; c < C; ++c) v[i][c] = 0.f;
        if (w[i] != 0.f) {
          const float* src = (s0 + s < n_prefix ? a.prefix.o : a.own.o) + row_of(s0 + s) * D + lane * C;
          if constexpr (C == 4) *reinterpret_cast<float4*>(v[i]) = *reinterpret_cast<const float4*>(src);
          else *reinterpret_cast<float2*>(v[i]) = *reinterpret_cast<const float2*>(src);
        }
      }
#pragma unroll
      for (int i = 0; i < 8; ++i)
#pragma unroll
        for (int c = 0; c < C; ++c) acc[c] = fmaf(v[i][c], w[i], acc[c]);
    }
  }
#pragma unroll
  for (int o = 16; o > 0; o >>= 1) lsum += __shfl_xor_sync(0xffffffffu, lsum, o);
  if constexpr (WARPS > 1) {
    __syncthreads();   // (sm_x has been read)
#pragma unroll
    for (int c = 0; c < C; ++c) sm_o[warp][lane * C + c] = acc[c];
    if (lane == 0) sm_x[warp] = lsum;
    __syncthreads();
    if (warp != 0) return;
    lsum = 0.f;
#pragma unroll
    for (int w = 0; w < WARPS; ++w) {
      lsum += sm_x[w];
#pragma unroll
      for (int c = 0; c < C; ++c) acc[c] = w == 0 ? sm_o[0][lane * C + c] : acc[c] + sm_o[w][lane * C + c];
    }
  }
  const float inv = lsum != 0.f ? 1.f / lsum : 0.f;
  T* out = reinterpret_cast<T*>(p.out) + b * p.os[0] + h * p.os[1];
  __align__(8) T r[C];
#pragma unroll
  for (int c = 0; c < C; ++c) r[c] = from_f32<T>(acc[c] * inv);
  T* to = out + lane * C;
  if (p.os[3] == 1 && reinterpret_cast<uintptr_t>(to) % (2 * C) == 0) {
    if constexpr (C == 4) *reinterpret_cast<uint2*>(to) = *reinterpret_cast<const uint2*>(r);
    else *reinterpret_cast<uint32_t*>(to) = *reinterpret_cast<const uint32_t*>(r);
  } else {
#pragma unroll
    for (int c = 0; c < C; ++c) out[(lane * C + c) * p.os[3]] = r[c];
  }
  if (p.lse != nullptr && lane == 0) p.lse[b * p.ls[0] + h * p.ls[1]] = lsum == 0.f ? -CUDART_INF_F : fmaf(mx, kLn2, logf(lsum));
}

struct Geometry {
  int chunk, nsplit, n_front; // own keys of a 16-bit cache; nsplit = 0: no table, or an 8-bit cache; n_front: ranges of the prefix before them
  Fp8Geometry fp8;            // own keys of an 8-bit cache
  bool front;                 // the prefix's keys with them, once for each sequence
  PackGeom pack;              // prefix
  uint64_t own_bytes, prefix_bytes, dense_bytes;
  uint64_t total() const { return own_bytes + prefix_bytes + dense_bytes; }
};

uint64_t aligned(uint64_t n) { return (n + 255) / 256 * 256; }

Problem own_problem(const B200CacheDecodeParams& a) {
  Problem p = {};
  p.q = a.q;
  p.k = a.k_pages;
  p.v = a.v_pages;
  p.out = a.out;
  p.lse = a.lse;
  const int64_t qs[4] = {a.q_stride[0], a.q_stride[1], 0, a.q_stride[2]}, os[4] = {a.out_stride[0], a.out_stride[1], 0, a.out_stride[2]};
  for (int i = 0; i < 4; ++i) {
    p.qs[i] = qs[i];
    p.os[i] = os[i];
    p.ks[i] = i < 3 ? a.k_pages_stride[i] : 1;
    p.vs[i] = i < 3 ? a.v_pages_stride[i] : 1;
  }
  p.ls[0] = a.lse_stride[0];
  p.ls[1] = a.lse_stride[1];
  p.B = a.B;
  p.Hq = a.Hq;
  p.Hkv = a.Hkv;
  p.L = 1;
  p.S = a.block_table_stride * a.page_size;
  p.E = p.Dv = a.D;
  p.group = a.Hq / a.Hkv;
  p.scale = a.scale;
  p.kv_lens = a.kv_lens;
  p.status = a.status;
  p.block_table = a.block_table;
  p.table_stride = a.block_table_stride;
  p.n_pages = a.n_pages;
  while ((1 << p.page_shift) < a.page_size) ++p.page_shift;
  return p;
}

// The batch's rows against the prefix: in the pools' pages (k null), or dense rows at `k` and `v` ((Hkv, P, D)).
Problem prefix_problem(const B200CacheDecodeParams& a, const void* k, const void* v) {
  Problem p = own_problem(a);
  p.out = nullptr;
  p.lse = nullptr;
  p.block_table = a.prefix_table;
  if (k != nullptr) {
    p.k = k;
    p.v = v;
    const int64_t kv[4] = {static_cast<int64_t>(a.Hkv) * a.prefix_len * a.D, static_cast<int64_t>(a.prefix_len) * a.D, a.D, 1};
    for (int i = 0; i < 4; ++i) p.ks[i] = p.vs[i] = kv[i];
  }
  p.qs[0] = static_cast<int64_t>(a.B) * a.q_stride[0];
  p.qs[2] = a.q_stride[0];
  p.L = a.B;
  p.B = 1;
  p.S = a.prefix_len;
  p.kv_lens = nullptr;
  return p;
}
// Tensor copies read a 16-bit prefix in its pages; an 8-bit one, or one of smaller pages, is first gathered into dense 16-bit rows.
bool gathered(const B200CacheDecodeParams& a) {
  return a.k_scales != nullptr || !prefix_paged(prefix_problem(a, nullptr, nullptr), a.n_pages);
}

// Keys of one CTA of the 16-bit kernel: enough CTAs for every slot of the GPU, ranges long enough to pay for a CTA's start and end.
int default_chunk(const Problem& p, int keys) {
  const int64_t units = static_cast<int64_t>(p.B) * p.Hkv * ((p.group + 15) / 16);
  int best = 256;
  double best_us = 1e30;
  for (int chunk = 64; chunk <= 2048; chunk += chunk < 512 ? 64 : 256) {
    const int n = (keys - 1) / chunk + 1;
    const double fill = static_cast<double>(units) * n / 444;
    const double rounds = fill < 1.0 ? 1.0 : fill + 0.35;
    const double us = rounds * (3.5 + chunk / 64.0 * (1.1 + 1.6 * (fill < 1.0 ? fill : 1.0))) * (1.0 + 0.002 * n);
    if (us < best_us) {
      best_us = us;
      best = chunk;
    }
    if (chunk >= keys) break;
  }
  return best;
}

}  // namespace

namespace {

// Whether the prefix is read for each sequence, before its own keys, instead of once for all.  For each costs B times its keys, from
// L2 all but once.
// 8-bit: once for all costs two more launches (gathered rows, then tiles of 128 query rows whether there are as many or not).  Both in
// us, fitted to 1 to 128 sequences under 300 to 11008 keys (each against once, with up to 100 own keys): 1 sequence, 8192 keys, 8 kv
// heads of 128: 16.4 against 29.9; 5, 3708, 4: 16.4 against 21.9; 8, 4096, 8: 28.0 against 27.4; 16, 2048, 8: 28.2 against 24.5;
// 128, 2048, 8: 110 against 40; 64, 4096, 2 heads of 64: 29.4 against 21.3.
// 16-bit: one more launch, and the own keys run beside it; so for each only while the elements that its grid covers, prefix and room of
// the table, for all sequences, are few.  (The lengths are the device's to know: a table far wider than its sequences takes the other
// form sooner than it need.)  With up to 100 own keys in a table of 128: 1, 300, 2: 6.9 against 11.0; 5, 1000, 4 heads of 64: 8.2 against 10.3; 2, 2048, 8: 11.0 against 12.3; 4, 2048, 8: 13.7
// against 12.6; 8, 1024, 8: 13.7 against 13.0; 16, 2048, 8: 27.7 against 14.6.
bool in_front(const B200CacheDecodeParams& a) {
  const Problem f = prefix_problem(a, nullptr, nullptr);
  if (a.k_scales == nullptr) {
    const Problem p = own_problem(a);
    const double keys = static_cast<double>(a.B) * a.Hkv * ((p.group + 15) / 16) * (static_cast<double>(a.prefix_len) + p.S);
    return p.S > 0 && keys * a.D < 7.0e6;
  }
  const int heads = f.group <= 8 ? 8 : 16;
  const double blocks = static_cast<double>(a.B) * a.Hkv * ((f.group + heads - 1) / heads) * ((a.prefix_len + 127) / 128);
  const double each = blocks / 148 * (a.D == 128 ? 1.0 : 0.6);
  PackGeom g;
  prefix_geometry(f, &g);
  const double steps = g.dual ? (g.split_tiles + 1) / 2 : g.split_tiles;
  const double rounds = static_cast<double>((g.grid + 147) / 148);
  const double once = 6.5 + 6.0 * a.prefix_len * a.Hkv * a.D / 8.0e6 + rounds * steps * 1.9;
  return each < once;
}

}  // namespace

int cache_decode_served(const B200CacheDecodeParams& a) {
  for (int i = 0; i < 3 && a.k_scales != nullptr; ++i)   // (the kernels multiply page and row by 32 bits)
    if (a.k_scales_stride[i] < 0 || a.k_scales_stride[i] > 0x7fffffffLL || a.v_scales_stride[i] < 0 || a.v_scales_stride[i] > 0x7fffffffLL)
      return B200_SDPA_ERR_UNSUPPORTED;
  if (static_cast<int64_t>(a.B) * a.Hq > 0x7fffffffLL) return B200_SDPA_ERR_UNSUPPORTED;
  if (a.prefix_len == 0) return a.k_scales != nullptr ? B200_SDPA_OK : B200_SDPA_ERR_UNSUPPORTED;
  const Problem f = prefix_problem(a, nullptr, nullptr);
  if (f.group > 128) return B200_SDPA_ERR_UNSUPPORTED;
  return prefix_eligible(f, a.dtype) ? B200_SDPA_OK : B200_SDPA_ERR_ALIGNMENT;
}

namespace {

int geometry(const B200CacheDecodeParams& a, Geometry* g) {
  const int rc = cache_decode_served(a);
  if (rc != B200_SDPA_OK) return rc;
  const Problem p = own_problem(a);
  *g = {};
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq;
  const int kv_chunk = a.kv_chunk < (1 << 30) ? a.kv_chunk : 1 << 30;   // (no table has more)
  g->front = a.prefix_len > 0 && in_front(a);
  if (a.k_scales != nullptr && (p.S > 0 || g->front)) {
    if (!decode_fp8_served(p, a.n_pages) || !decode_fp8_geometry(p, g->front ? a.prefix_len : 0, kv_chunk, &g->fp8)) return B200_SDPA_ERR_UNSUPPORTED;
    g->own_bytes = aligned(g->fp8.bytes);
  } else if (p.S > 0) {
    g->chunk = kv_chunk > 0 ? (kv_chunk + 31) / 32 * 32 : default_chunk(p, p.S + (g->front ? a.prefix_len : 0));
    g->nsplit = (p.S - 1) / g->chunk + 1;
    if (g->front) g->n_front = (a.prefix_len - 1) / g->chunk + 1;
    if (g->nsplit + g->n_front > 65535 || static_cast<int64_t>(p.Hkv) * ((p.group + 15) / 16) > 65535) return B200_SDPA_ERR_UNSUPPORTED;
    g->own_bytes = aligned(static_cast<uint64_t>(rows) * (g->nsplit + g->n_front) * (a.D + 2) * sizeof(float));
  }
  if (a.prefix_len > 0 && !g->front) {
    const Problem f = prefix_problem(a, nullptr, nullptr);
    prefix_geometry(f, &g->pack);
    g->prefix_bytes = aligned(g->pack.ws_bytes);
    if (gathered(a)) g->dense_bytes = 2 * aligned(static_cast<uint64_t>(a.Hkv) * a.prefix_len * a.D * 2);
  }
  return B200_SDPA_OK;
}

template <typename T, int WARPS> int launch_combine_warps(const Problem& p, const Merge& a, cudaStream_t stream) {
  auto kern = p.E == 128 ? cache_combine_kernel<T, 128, WARPS> : cache_combine_kernel<T, 64, WARPS>;
  const unsigned grid = static_cast<unsigned>((static_cast<int64_t>(p.B) * p.Hq * WARPS + kCombineWarps - 1) / kCombineWarps);
  if (!launch_pdl(kern, dim3(grid), kCombineWarps * 32, 0, stream, p, a)) return B200_SDPA_ERR_CUDA;
  count_launch(KID_COMBINE);
  return B200_SDPA_OK;
}
template <typename T> int launch_combine(const Problem& p, const Merge& a, cudaStream_t stream) {
  return static_cast<int64_t>(p.B) * p.Hq >= 1024 ? launch_combine_warps<T, 1>(p, a, stream) : launch_combine_warps<T, 4>(p, a, stream);
}

}  // namespace

int plan_cache_decode(const B200CacheDecodeParams& a, B200SdpaPlan* plan) {
  Geometry g;
  const int rc = geometry(a, &g);
  if (rc != B200_SDPA_OK) return rc;
  const bool fp8 = g.fp8.grid > 0;
  plan->path = B200_SDPA_PATH_DECODE;
  plan->block_m = 1;
  plan->block_n = fp8 ? 128 : g.chunk;
  plan->grid_x = fp8 ? g.fp8.grid : a.Hkv * ((a.Hq / a.Hkv + 15) / 16);
  plan->grid_y = fp8 ? 1 : a.B;
  plan->grid_z = fp8 ? 1 : g.nsplit + g.n_front;
  plan->threads = fp8 ? 192 : 128;
  plan->smem_bytes = 0;
  plan->kv_splits = fp8 ? g.fp8.grid : g.nsplit + g.n_front;
  plan->launches = 1 + (plan->kv_splits > 0 ? 1 : 0) + (a.prefix_len > 0 && !g.front ? (gathered(a) ? 2 : 1) : 0);
  plan->workspace_bytes = g.total();
  return B200_SDPA_OK;
}

int launch_cache_decode(const B200CacheDecodeParams& a, cudaStream_t stream) {
  Geometry g;
  int rc = geometry(a, &g);
  if (rc != B200_SDPA_OK) return rc;
  if (g.total() > 0 && (a.workspace == nullptr || a.workspace_bytes < g.total() || reinterpret_cast<uintptr_t>(a.workspace) % 16))
    return B200_SDPA_ERR_WORKSPACE;
  const Problem p = own_problem(a);
  const int64_t rows = static_cast<int64_t>(a.B) * a.Hq;
  char* ws = static_cast<char*>(a.workspace);
  float* pre_o = reinterpret_cast<float*>(ws + g.own_bytes);
  float* pre_ml = pre_o + rows * g.pack.n_split * a.D;
  Merge m = {};
  m.prefix = {pre_o, pre_ml};
  m.n_prefix = g.front ? 0 : g.pack.n_split;
  // 8-bit: the own keys first; the gathering, which needs nothing of theirs, runs beside them.  16-bit: the prefix first; the
  // own keys run beside it, on the SMs that it leaves or has done with.  (64 sequences under 16384 keys: 70 us one behind the other.)
  if (g.fp8.grid > 0) {
    CacheScales sc = {};
    sc.k = static_cast<const uint8_t*>(a.k_scales);
    sc.v = static_cast<const uint8_t*>(a.v_scales);
    for (int i = 0; i < 3; ++i) {
      sc.ks[i] = a.k_scales_stride[i];
      sc.vs[i] = a.v_scales_stride[i];
    }
    sc.n_pages = a.n_pages;
    OwnPartials part;
    part.slots = g.fp8.slots;
    part.o = reinterpret_cast<float*>(ws);
    part.ml = part.o + g.fp8.slots * kFp8Parts * g.fp8.heads * a.D;
    part.range = reinterpret_cast<int2*>(part.ml + g.fp8.slots * kFp8Parts * g.fp8.heads * 2);
    m.own = {part.o, part.ml};
    m.range = part.range;
    m.heads = g.fp8.heads;
    m.units = g.fp8.units;
    m.slots = static_cast<int>(g.fp8.slots);
    m.grid = g.fp8.grid;
    if (g.front) {
      m.front = 1;
      m.prefix = m.own;
    }
    const FrontKeys front = {a.prefix_table, g.front ? a.prefix_len : 0};
    rc = launch_decode_partial_fp8(p, sc, a.dtype, g.fp8, front, part, stream);
    if (rc != B200_SDPA_OK) return rc;
  }
  if (g.front) {
    // nothing more: the prefix is among the own keys' partials
  } else if (a.prefix_len > 0 && gathered(a)) {
    char* dense = ws + g.own_bytes + g.prefix_bytes;
    B200CacheRowsParams r = {};
    r.dtype = a.dtype;
    r.page_size = a.page_size;
    r.k = dense;
    r.v = dense + g.dense_bytes / 2;
    r.k_pages = const_cast<void*>(a.k_pages);
    r.v_pages = const_cast<void*>(a.v_pages);
    r.k_scales = const_cast<void*>(a.k_scales);
    r.v_scales = const_cast<void*>(a.v_scales);
    for (int i = 0; i < 3; ++i) {
      r.k_pages_stride[i] = a.k_pages_stride[i];
      r.v_pages_stride[i] = a.v_pages_stride[i];
      r.k_scales_stride[i] = a.k_scales_stride[i];
      r.v_scales_stride[i] = a.v_scales_stride[i];
    }
    r.k_stride[1] = r.v_stride[1] = static_cast<int64_t>(a.prefix_len) * a.D;
    r.k_stride[2] = r.v_stride[2] = a.D;
    r.B = 1;
    r.Hkv = a.Hkv;
    r.L = a.prefix_len;
    r.D = a.D;
    r.block_table = a.prefix_table;
    r.block_table_stride = (a.prefix_len + a.page_size - 1) / a.page_size;
    r.n_pages = a.n_pages;
    r.status = a.status;
    rc = launch_cache_gather(r, g.fp8.grid > 0, stream);
    if (rc != B200_SDPA_OK) return rc;
    rc = launch_prefix_partial(prefix_problem(a, r.k, r.v), a.dtype, g.pack, pre_o, pre_ml, stream, 0, a.k_scales != nullptr);
    if (rc != B200_SDPA_OK) return rc;
  } else if (a.prefix_len > 0) {
    rc = launch_prefix_partial(prefix_problem(a, nullptr, nullptr), a.dtype, g.pack, pre_o, pre_ml, stream, a.n_pages, false);
    if (rc != B200_SDPA_OK) return rc;
  }
  if (g.nsplit > 0) {
    float* own_o = reinterpret_cast<float*>(ws);
    const int n = g.nsplit + g.n_front;
    float* own_ml = own_o + rows * n * a.D;
    m.own = {own_o, own_ml};
    if (g.front) {
      m.front = g.n_front;
      m.prefix = m.own;
    }
    m.n_own = g.nsplit;
    m.chunk = g.chunk;
    rc = launch_decode_partial_mma(p, a.dtype, g.chunk, n, own_o, own_ml, stream, true, FrontKeys{a.prefix_table, a.prefix_len}, g.n_front);
    if (rc != B200_SDPA_OK) return rc;
  }
  return a.dtype == B200_SDPA_BF16 ? launch_combine<__nv_bfloat16>(p, m, stream) : launch_combine<__half>(p, m, stream);
}

}  // namespace b200
