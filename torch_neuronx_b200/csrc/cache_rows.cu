// Rows into and out of an 8-bit paged key/value cache.
//
// A cached row (one token, one head, D elements) is D e4m3 values and one power of two 2^e, kept as its biased exponent
// (e8m0, one byte): the least e with amax <= 448 * 2^e, so the largest value uses the format's top binade.  A power of two
// costs a float format nothing (only values 2^-15 below the row's largest lose bits they would keep under a finer scale)
// and makes both directions exact where it matters: x * 2^-e is exact, so a value is rounded once, to e4m3; value * 2^e is
// exact in bf16, so reading back rounds nothing but 2^128, which e4m3 makes of bf16's largest numbers (from 248 * 2^120 on) and
// which reads as an infinity (fp16: once, below 2^-14, and beyond 65504 likewise).  A row of zeros has e = 0; a
// row with a NaN or an infinity has the scale NaN (255) and reads as NaN; e is at least -127.
//
// Bound by HBM.  A row is D / 16 lanes with 16 elements each: 32 bytes on the 16-bit side, 16 on the other; writing, the maximum
// meets over those lanes.  8 heads of 128, bf16: 16 prompts of 512..4096 tokens written in 41 us (5.8 TB/s), 8 sequences of
// 4096..8192 rows read in 66 us (5.7 TB/s).
// A page number outside the pool is reported through the status word, and nothing is read or written there: such rows read as zeros.
// (Gathered rows are page 0's, as in the kernels that read the pages themselves.)
#include "common.cuh"
#include "debug.cuh"
#include "fp8.cuh"

namespace b200 {

namespace {

constexpr int kThreads = 256;

// Pool row (page, row in page) of position `pos` of sequence b; false: outside the table or the pool.
__device__ __forceinline__ bool locate(const B200CacheRowsParams& p, int page_shift, int b, int64_t pos, int64_t* page, int* row) {
  const int64_t slot = pos >> page_shift;
  if (pos < 0 || slot >= p.block_table_stride) return false;
  *page = p.block_table[static_cast<int64_t>(b) * p.block_table_stride + slot];
  *row = static_cast<int>(pos & ((1 << page_shift) - 1));
  return *page >= 0 && *page < p.n_pages;
}

// The larger of two pairs of 16-bit numbers, a NaN where there is one.
template <bool BF16> __device__ __forceinline__ uint32_t max_pair(uint32_t a, uint32_t b) {
  uint32_t r;
  if (BF16) {
    asm("max.NaN.bf16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  } else {
    asm("max.NaN.f16x2 %0, %1, %2;" : "=r"(r) : "r"(a), "r"(b));
  }
  return r;
}

// LPR: lanes of a row, a power of two >= D / 16.  One CTA: `tokens` tokens of the keys or of the values of one sequence.  A thread's place
// (token, head) moves on by fixed steps and offsets are 32 x 32 bits: in the first form, which divided for each row and chose between
// keys and values in the loop, instructions and not bytes were the bound (16 prompts of 512..4096 tokens, 8 heads of 128: 82 us).
template <bool BF16, int LPR>
__global__ void __launch_bounds__(kThreads) cache_write_kernel(const B200CacheRowsParams p, const int page_shift, const int tokens,
                                                               const int rows_16b) {
  constexpr int kRows = kThreads / LPR;
  const int b = blockIdx.y, i0 = blockIdx.x * tokens;
  pdl_wait();
  pdl_launch_dependents();
  int n = p.lens != nullptr ? p.lens[b] : p.L;
  n = n < p.L ? n : p.L;
  const int n_tok = n - i0 < tokens ? n - i0 : tokens;
  if (n_tok <= 0) return;
  const bool is_v = blockIdx.z != 0;
  const uint32_t x_head = static_cast<uint32_t>(is_v ? p.v_stride[1] : p.k_stride[1]), x_row = static_cast<uint32_t>(is_v ? p.v_stride[2] : p.k_stride[2]);
  const uint32_t y_page = static_cast<uint32_t>(is_v ? p.v_pages_stride[0] : p.k_pages_stride[0]);
  const uint32_t y_head = static_cast<uint32_t>(is_v ? p.v_pages_stride[1] : p.k_pages_stride[1]), y_row = static_cast<uint32_t>(is_v ? p.v_pages_stride[2] : p.k_pages_stride[2]);
  const uint32_t s_page = static_cast<uint32_t>(is_v ? p.v_scales_stride[0] : p.k_scales_stride[0]);
  const uint32_t s_head = static_cast<uint32_t>(is_v ? p.v_scales_stride[1] : p.k_scales_stride[1]), s_row = static_cast<uint32_t>(is_v ? p.v_scales_stride[2] : p.k_scales_stride[2]);
  const int lane = threadIdx.x % LPR, c0 = lane * 16;
  const uint16_t* x = static_cast<const uint16_t*>(is_v ? p.v : p.k) + b * (is_v ? p.v_stride[0] : p.k_stride[0]) +
                      static_cast<int64_t>(i0) * x_row + c0;
  uint8_t* pages = static_cast<uint8_t*>(is_v ? p.v_pages : p.k_pages) + c0;
  uint8_t* scales = static_cast<uint8_t*>(is_v ? p.v_scales : p.k_scales);
  const int* table = p.block_table + static_cast<int64_t>(b) * p.block_table_stride;
  const int64_t start = p.start[b];
  const int first = threadIdx.x / LPR, d_h = kRows % p.Hkv, d_t = kRows / p.Hkv;
  int h = first % p.Hkv, t = first / p.Hkv;
  const int rounds = (n_tok * p.Hkv + kRows - 1) / kRows;   // (whole warps walk on together: the maximum meets over a row's lanes)
  __align__(16) uint32_t e[8], next[8];
  int next_entry;
  auto fetch = [&]() {   // the row at (t, h) and its page
#pragma unroll
    for (int k = 0; k < 8; ++k) next[k] = 0u;
    next_entry = -1;
    if (t >= n_tok || c0 >= p.D) return;
    const uint16_t* from = x + static_cast<uint64_t>(static_cast<uint32_t>(h)) * x_head + static_cast<uint64_t>(static_cast<uint32_t>(t)) * x_row;
    if (rows_16b) {
      *reinterpret_cast<uint4*>(next) = ld_stream_16B(from);
      *reinterpret_cast<uint4*>(next + 4) = ld_stream_16B(from + 8);
    } else {
#pragma unroll
      for (int k = 0; k < 8; ++k) next[k] = from[2 * k] | static_cast<uint32_t>(from[2 * k + 1]) << 16;
    }
    const int64_t pos = start + i0 + t;
    if (pos >= 0 && (pos >> page_shift) < p.block_table_stride) next_entry = table[pos >> page_shift];
  };
  fetch();
  for (int i = 0; i < rounds; ++i) {
    const bool on = t < n_tok && c0 < p.D;
    const int64_t pos = start + i0 + t;
    const int entry = next_entry;
    const uint64_t head = static_cast<uint32_t>(h);
#pragma unroll
    for (int k = 0; k < 8; ++k) e[k] = next[k];
    h += d_h;
    t += d_t;
    if (h >= p.Hkv) {
      h -= p.Hkv;
      ++t;
    }
    fetch();   // (the next row travels while this one is rounded)
    uint32_t top2 = e[0] & 0x7fff7fffu;
#pragma unroll
    for (int k = 1; k < 8; ++k) top2 = max_pair<BF16>(top2, e[k] & 0x7fff7fffu);
#pragma unroll
    for (int o = LPR / 2; o > 0; o >>= 1) top2 = max_pair<BF16>(top2, __shfl_xor_sync(0xffffffffu, top2, o));
    if (on) {
      const uint32_t top = top2 >> 16 > (top2 & 0xffffu) ? top2 >> 16 : top2 & 0xffffu;   // (bits order like magnitudes)
      const int code = scale_code(__float_as_uint(half_to_f32<BF16>(static_cast<uint16_t>(top))));
      if (static_cast<unsigned>(entry) < static_cast<unsigned>(p.n_pages)) {
        const float inv = scale_inverse(code);
        uint32_t w[8];
#pragma unroll
        for (int k = 0; k < 8; ++k)
          w[k] = pack_e4m3(half_to_f32<BF16>(static_cast<uint16_t>(e[k])) * inv, half_to_f32<BF16>(static_cast<uint16_t>(e[k] >> 16)) * inv);
        const uint64_t page = static_cast<uint32_t>(entry), row = static_cast<uint32_t>(pos) & ((1u << page_shift) - 1);
        *reinterpret_cast<uint4*>(pages + page * y_page + head * y_head + row * y_row) =
            make_uint4(w[0] | w[1] << 16, w[2] | w[3] << 16, w[4] | w[5] << 16, w[6] | w[7] << 16);
        if (lane == 0) scales[page * s_page + head * s_head + row * s_row] = static_cast<uint8_t>(code);
      } else {
        const bool full = pos >= (static_cast<int64_t>(p.block_table_stride) << page_shift);
        report_page(p.status, full ? B200_SDPA_ERR_CACHE_FULL : B200_SDPA_ERR_PAGE, b, static_cast<int>(pos), p.n_pages);
      }
    }
  }
}

// A gathered row holds nothing beyond its type's largest number, 65504 or 255 * 2^120: e4m3 makes 65536 and 2^128 of it, half a step
// more, and an infinite key or value would stand for a finite one.  NaN stays.
template <bool BF16> __device__ __forceinline__ float within(float x) {
  constexpr float kMost = BF16 ? 255.f * 0x1p120f : 65504.f;
  return fabsf(x) > kMost ? copysignf(kMost, x) : x;
}

// LPR: lanes of a row, a power of two >= D / 16.  QUANT false: the pools hold the rows' own 16-bit type (strides in
// elements).  Without lens every row is there.  GATHERED: rows for this library's own products.
template <bool BF16, int LPR, bool QUANT, bool GATHERED>
__global__ void __launch_bounds__(kThreads) cache_read_kernel(const B200CacheRowsParams p, const int page_shift, const int tokens,
                                                               const int rows_16b, const int beside) {
  constexpr int kRows = kThreads / LPR;
  const int b = blockIdx.y, i0 = blockIdx.x * tokens;
  if (!beside) pdl_wait();
  pdl_launch_dependents();
  int n = p.lens != nullptr ? p.lens[b] : p.L;
  n = n < p.L ? n : p.L;
  const int n_tok = p.L - i0 < tokens ? p.L - i0 : tokens;
  const int lane = threadIdx.x % LPR, c0 = lane * 16;
  const int total = c0 < p.D ? n_tok * 2 * p.Hkv : 0;
  for (int r = threadIdx.x / LPR; r < total; r += kRows) {
    const int hk = r / n_tok, t = r - hk * n_tok;   // neighbouring tokens of a head: neighbouring rows of the result
    const bool is_v = hk >= p.Hkv;
    const int h = hk - (is_v ? p.Hkv : 0);
    const int64_t* xs = is_v ? p.v_stride : p.k_stride;
    uint16_t* x = static_cast<uint16_t*>(const_cast<void*>(is_v ? p.v : p.k)) + b * xs[0] + h * xs[1] + (i0 + t) * xs[2] + c0;
    __align__(16) uint32_t out[8] = {};
    if (i0 + t < n) {
      int64_t page = 0;
      int row = 0;
      bool there = locate(p, page_shift, b, i0 + t, &page, &row);
      if (!there) {
        report_page(p.status, B200_SDPA_ERR_PAGE, GATHERED ? kSharedPrefix : b, (i0 + t) >> page_shift << page_shift, p.n_pages);
        page = 0;
        there = GATHERED;
      }
      if (there) {
        const int64_t* ps = is_v ? p.v_pages_stride : p.k_pages_stride;
        const int64_t at = page * ps[0] + h * ps[1] + row * ps[2] + c0;
        const void* pool = is_v ? p.v_pages : p.k_pages;
        if constexpr (QUANT) {
          const int64_t* ss = is_v ? p.v_scales_stride : p.k_scales_stride;
          const uint4 w = ld_stream_16B(static_cast<const uint8_t*>(pool) + at);
          const int code = static_cast<const uint8_t*>(is_v ? p.v_scales : p.k_scales)[page * ss[0] + h * ss[1] + row * ss[2]];
          const float scale = scale_value(code);
          const bool beyond = GATHERED && code > (BF16 ? 246 : 134);   // (448 times the scale is more than the type's largest)
          const uint32_t in[4] = {w.x, w.y, w.z, w.w};
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            float f[4];
            unpack_e4m3x4(in[i], f);
#pragma unroll
            for (int j = 0; j < 4; ++j) f[j] *= scale;
            if (beyond) {
#pragma unroll
              for (int j = 0; j < 4; ++j) f[j] = within<BF16>(f[j]);
            }
            out[2 * i] = pack16<BF16>(f[0], f[1]);
            out[2 * i + 1] = pack16<BF16>(f[2], f[3]);
          }
        } else {
          *reinterpret_cast<uint4*>(out) = ld_stream_16B(static_cast<const uint16_t*>(pool) + at);
          *reinterpret_cast<uint4*>(out + 4) = ld_stream_16B(static_cast<const uint16_t*>(pool) + at + 8);
        }
      }
    }
    if (rows_16b) {
      *reinterpret_cast<uint4*>(x) = make_uint4(out[0], out[1], out[2], out[3]);
      *reinterpret_cast<uint4*>(x + 8) = make_uint4(out[4], out[5], out[6], out[7]);
    } else {
#pragma unroll
      for (int i = 0; i < 16; ++i) x[i] = static_cast<uint16_t>(out[i / 2] >> (16 * (i & 1)));
    }
  }
  if (beside) pdl_wait();   // (complete no sooner than the launch before)
}

// Tokens of one CTA, `heads` rows each: enough for a few rounds of its threads, fewer where there would not be several CTAs for every SM.
int tokens_per_cta(const B200CacheRowsParams& p, int rows_per_round, int heads) {
  constexpr int kRounds = 4;
  int tokens = (kRounds * rows_per_round + heads - 1) / heads;
  tokens = tokens < 1 ? 1 : tokens;
  while (tokens > 1 && static_cast<int64_t>(p.B) * ((p.L + tokens - 1) / tokens) < 4 * 148) tokens = (tokens + 1) / 2;
  return tokens;
}

int page_shift_of(int page_size) {
  int s = 0;
  while ((1 << s) < page_size) ++s;
  return s;
}

// Whether every dense row starts on 16 bytes.
bool rows_16b(const B200CacheRowsParams& p) {
  if (reinterpret_cast<uintptr_t>(p.k) % 16 || reinterpret_cast<uintptr_t>(p.v) % 16) return false;
  for (int i = 0; i < 3; ++i)
    if (p.k_stride[i] % 8 || p.v_stride[i] % 8) return false;
  return true;
}

enum Direction { WRITE, READ, GATHER, COPY };   // COPY: gathered rows of a 16-bit cache

template <Direction DIR, bool BF16, int LPR> int launch_rows(const B200CacheRowsParams& p, int beside, cudaStream_t stream) {
  const int tokens = tokens_per_cta(p, kThreads / LPR, DIR == WRITE ? p.Hkv : 2 * p.Hkv);
  const dim3 grid((p.L + tokens - 1) / tokens, p.B, DIR == WRITE ? 2 : 1);
  const int shift = page_shift_of(p.page_size);
  bool ok;
  if constexpr (DIR == WRITE) ok = launch_pdl(cache_write_kernel<BF16, LPR>, grid, kThreads, 0, stream, p, shift, tokens, rows_16b(p) ? 1 : 0);
  else ok = launch_pdl(cache_read_kernel<BF16, LPR, DIR != COPY, DIR != READ>, grid, kThreads, 0, stream, p, shift, tokens, rows_16b(p) ? 1 : 0, beside);
  if (!ok) return B200_SDPA_ERR_CUDA;
  count_launch(DIR == WRITE ? KID_CACHE_WRITE : KID_CACHE_READ);
  return B200_SDPA_OK;
}

template <Direction DIR, bool BF16> int launch_lanes(const B200CacheRowsParams& p, cudaStream_t stream, int beside = 0) {
  const int lanes = p.D / 16;
  if (lanes <= 4) return launch_rows<DIR, BF16, 4>(p, beside, stream);
  if (lanes <= 8) return launch_rows<DIR, BF16, 8>(p, beside, stream);
  return launch_rows<DIR, BF16, 16>(p, beside, stream);
}

}  // namespace

int launch_cache_write(const B200CacheRowsParams& p, cudaStream_t stream) {
  return p.dtype == B200_SDPA_BF16 ? launch_lanes<WRITE, true>(p, stream) : launch_lanes<WRITE, false>(p, stream);
}
int launch_cache_read(const B200CacheRowsParams& p, cudaStream_t stream) {
  return p.dtype == B200_SDPA_BF16 ? launch_lanes<READ, true>(p, stream) : launch_lanes<READ, false>(p, stream);
}
int launch_cache_gather(const B200CacheRowsParams& p, bool beside, cudaStream_t stream) {
  if (p.k_scales == nullptr) return launch_lanes<COPY, true>(p, stream, beside);   // (a copy: either 16-bit type)
  return p.dtype == B200_SDPA_BF16 ? launch_lanes<GATHER, true>(p, stream, beside) : launch_lanes<GATHER, false>(p, stream, beside);
}

}  // namespace b200
