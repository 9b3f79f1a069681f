// Split-KV flash decoding against an 8-bit paged cache (cache_rows.cu has the format), products on tensor cores.
//
// The partial kernel of decode_mma.cu with half the bytes: grid (kv head and block of query heads, sequence, key split), the
// cache read once for all query heads of a block, fp32 partials (o, m, l) merged by the same second launch.
// What the format changes:
//   * e4m3 is exact in fp16, so both products are fp16 m16n8k16 MMAs with the bytes expanded in registers: a fragment word
//     of K holds four consecutive elements of one key, and the order inside a k-step is free as long as the query
//     fragments use it too; a transposed fragment word of V holds two keys x two columns, one byte permutation makes it
//     an operand for each column.  (8-bit MMAs would need P and Q in 8 bits.)
//   * scores: s = (q . k8) * 2^e_k, the row's power of two applied to the finished fp32 score.  A query row is brought to
//     a maximum in [2^14, 2^15) by a power of two first (bf16; fp16 keeps its own scale unless it has room above), so
//     fp16 holds it exactly but for elements 2^-28 below the row's largest, which round at 2^-39 of it.
//   * values: o += (p 2^(e_v - r + 9)) v8 with r the largest e_v the warp has met (o is rescaled when it grows), so the
//     probability stays inside fp16; it enters as hi + lo, two fp16 operands: 22 bits, and never coarser than 2^-34 of
//     the largest value row the warp has met.  With up to 8 query heads the low parts ride in the eight rows of the
//     MMA that would be empty; with up to 16 they cost a second MMA.
// Softmax in the exp2 domain on raw scores, statistics fp32, the running maximum raised lazily (2^6).
#include "common.cuh"
#include "debug.cuh"
#include "fp8.cuh"

namespace b200 {

namespace {

constexpr int kWarps = 4;
constexpr int kThreads = kWarps * 32;
constexpr int kBlockKeys = 64;
constexpr int kStages = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRescaleThreshold = 6.0f;
constexpr float kProbShift = 9.0f;   // p <= 2^6, p 2^9 <= 2^15 in fp16

template <int D> struct Geo {
  static constexpr int kRowBytes = D + 16;                     // padded row: conflict-free ldmatrix
  static constexpr int kTileBytes = kBlockKeys * kRowBytes;    // one K or V block
  static constexpr int kStageBytes = 2 * kTileBytes;
  static constexpr int kRingBytes = kStages * kStageBytes;
  static constexpr int kChunksPerRow = D / 16;
  static constexpr int kScaleBytes = 2 * 2 * kBlockKeys * 4;   // [parity][K, V][key]
  static constexpr int kSmemBytes = kRingBytes + kScaleBytes;
};

__device__ __forceinline__ uint32_t smem_addr(const void* p) { return static_cast<uint32_t>(__cvta_generic_to_shared(p)); }
__device__ __forceinline__ void cp_async_16(uint32_t dst, const void* src, bool valid) {
  const int n = valid ? 16 : 0;   // 0 source bytes: the 16 destination bytes are zero-filled
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(n) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() { asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory"); }
__device__ __forceinline__ void ldsm_x4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void ldsm_x4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr));
}
__device__ __forceinline__ void mma_f16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, %3};"
      : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
      : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float ex2f(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// (lo, hi) as an fp16 pair, and what the rounding left over as another.
__device__ __forceinline__ void split_f16(float lo, float hi, uint32_t& head, uint32_t& rest) {
  head = pack16<false>(lo, hi);
  const float2 h = __half22float2(*reinterpret_cast<const __half2*>(&head));
  rest = pack16<false>(lo - h.x, hi - h.y);
}
__device__ __forceinline__ float quad_max(float x) {
  x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 1));
  return fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 2));
}
__device__ __forceinline__ float quad_sum(float x) {
  x += __shfl_xor_sync(0xffffffffu, x, 1);
  return x + __shfl_xor_sync(0xffffffffu, x, 2);
}

// HEADS: query heads of a CTA, 8 or 16.  ROWS = accumulator rows with a query head in them (g, and g + 8 of 16).
template <int D, bool BF16, int HEADS>
__global__ void __launch_bounds__(kThreads, HEADS == 8 ? 3 : 2)
    decode_fp8_kernel(const Problem p, const CacheScales sc, const int chunk, const int nsplit, float* __restrict__ part_o,
                      float* __restrict__ part_ml) {
  using G = Geo<D>;
  constexpr int KS = D / 16;            // k-steps of the first product
  constexpr bool kTwo = HEADS == 16;    // rows g + 8 are heads too (else they carry the low parts of P)
  extern __shared__ __align__(16) uint8_t smem[];

  const int split = blockIdx.z;   // slowest: the launch ends on the last (short or empty) chunks
  const int hk = blockIdx.x % p.Hkv;
  const int gsub = blockIdx.x / p.Hkv;
  const int b = blockIdx.y;
  pdl_wait();
  const int n_keys = valid_keys(p, b);
  const int s0 = split * chunk;
  if (s0 >= n_keys && split != 0) return;   // split 0 still writes an (empty) partial
  const int s1 = (s0 + chunk < n_keys) ? s0 + chunk : n_keys;
  const int n_blocks = s1 > s0 ? (s1 - s0 + kBlockKeys - 1) / kBlockKeys : 0;

  const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
  const int g = lane >> 2, tq = lane & 3;
  const int h0 = hk * p.group + gsub * HEADS;
  const int n_heads = (p.group - gsub * HEADS) < HEADS ? (p.group - gsub * HEADS) : HEADS;

  const uint8_t* kbase = static_cast<const uint8_t*>(p.k) + hk * p.ks[1];
  const uint8_t* vbase = static_cast<const uint8_t*>(p.v) + hk * p.vs[1];
  const int* table = p.block_table + static_cast<int64_t>(b) * p.table_stride;
  const int page_mask = (1 << p.page_shift) - 1;
  const uint32_t smem_base = smem_addr(smem);
  float* scales = reinterpret_cast<float*>(smem + G::kRingBytes);

  // Page of a key position of this chunk; -1 where there is none (behind the end, or a number outside the pool).
  auto page_of = [&](int row) -> int {
    if (row >= s1) return -1;
    const int page = table[row >> p.page_shift];
    if (static_cast<unsigned>(page) < static_cast<unsigned>(sc.n_pages)) return page;
    report_page(p.status, B200_SDPA_ERR_PAGE, b, row, sc.n_pages);
    return -1;
  };
  constexpr int kCopies = kBlockKeys * G::kChunksPerRow / kThreads;
  int pages[kCopies];
  auto fetch_pages = [&](int blk) {
#pragma unroll
    for (int i = 0; i < kCopies; ++i) pages[i] = page_of(s0 + blk * kBlockKeys + (tid + i * kThreads) / G::kChunksPerRow);
  };
  auto load_block = [&](int blk) {
    const uint32_t stage = smem_base + (blk % kStages) * G::kStageBytes;
    const int key0 = s0 + blk * kBlockKeys;
#pragma unroll
    for (int i = 0; i < kCopies; ++i) {
      const int c = tid + i * kThreads;
      const int row = c / G::kChunksPerRow, ch = c % G::kChunksPerRow;
      const bool ok = pages[i] >= 0;
      const int64_t page = ok ? pages[i] : 0;
      const int in_page = (key0 + row) & page_mask;
      cp_async_16(stage + row * G::kRowBytes + ch * 16, kbase + page * p.ks[0] + in_page * p.ks[2] + ch * 16, ok);
      cp_async_16(stage + G::kTileBytes + row * G::kRowBytes + ch * 16, vbase + page * p.vs[0] + in_page * p.vs[2] + ch * 16, ok);
    }
  };
  // Thread t < 64 brings the key scale of key t of a block, thread 64 + t the value scale.
  auto fetch_scale = [&](int blk) -> int {
    const int key = s0 + blk * kBlockKeys + (tid & 63);
    const int page = page_of(key);
    if (page < 0) return -1;
    const int64_t* ss = tid < 64 ? sc.ks : sc.vs;
    return (tid < 64 ? sc.k : sc.v)[page * ss[0] + hk * ss[1] + (key & page_mask) * ss[2]];
  };
  // Keys: the scale itself.  Values: its exponent (NaN for a NaN scale; -inf where there is no key).
  auto store_scale = [&](int blk, int code) {
    float x;
    if (tid < 64) x = code < 0 ? 0.f : scale_value(code);
    else x = code < 0 ? -CUDART_INF_F : (code == 255 ? CUDART_NAN_F : static_cast<float>(code - 127));
    scales[(blk & 1) * 2 * kBlockKeys + tid] = x;
  };

  if (n_blocks > 0) {
    store_scale(0, fetch_scale(0));
#pragma unroll
    for (int i = 0; i < kStages - 1; ++i) {
      if (i < n_blocks) {
        fetch_pages(i);
        load_block(i);
      }
      cp_async_commit();
    }
    if (kStages - 1 < n_blocks) fetch_pages(kStages - 1);
  }

  // ---- query rows: through the last stage as fp16, scaled by a power of two
  uint32_t qf[KS][kTwo ? 4 : 2];
  float sl2[2];   // score to exp2 units, of rows g and g + 8
  {
    const uint16_t* q16 = reinterpret_cast<const uint16_t*>(p.q) + b * p.qs[0];
    constexpr int kPitch = 2 * D + 16;
    uint8_t* stage = smem + (kStages - 1) * G::kStageBytes;
    float* q_scale = reinterpret_cast<float*>(stage + HEADS * kPitch);
    static_assert(HEADS * kPitch + HEADS * 4 <= G::kStageBytes, "the query rows fit in a stage");
    for (int row = warp; row < HEADS; row += kWarps) {
      float x[D / 32];
      uint32_t top = 0;
#pragma unroll
      for (int i = 0; i < D / 32; ++i) {
        x[i] = row < n_heads ? half_to_f32<BF16>(q16[(h0 + row) * p.qs[1] + (lane + 32 * i) * p.qs[3]]) : 0.f;
        const uint32_t m = __float_as_uint(x[i]) & 0x7fffffffu;
        top = m > top ? m : top;
      }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) {
        const uint32_t m = __shfl_xor_sync(0xffffffffu, top, o);
        top = m > top ? m : top;
      }
      // largest element into [2^14, 2^15); zeros, infinities and NaN stay as they are
      int up = top == 0u || top >= 0x7f800000u ? 0 : 127 + 14 - static_cast<int>(top >> 23);
      if (!BF16 && up < 0) up = 0;
      if (up > 126) up = 126;
      const float f = __int_as_float((127 + up) << 23);   // up >= -113
#pragma unroll
      for (int i = 0; i < D / 32; ++i)
        *reinterpret_cast<__half*>(stage + row * kPitch + (lane + 32 * i) * 2) = __float2half_rn(x[i] * f);
      if (lane == 0) q_scale[row] = p.scale * kLog2e * __int_as_float((127 - up) << 23);
    }
    __syncthreads();
    // k-step s of a fragment: elements 16 s + 4 tq .. + 3 of a row, as the bytes of a key's fragment word
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      const uint2 lo = *reinterpret_cast<const uint2*>(stage + g * kPitch + (16 * s + 4 * tq) * 2);
      qf[s][0] = lo.x;
      qf[s][1] = lo.y;
      if constexpr (kTwo) {
        const uint2 hi = *reinterpret_cast<const uint2*>(stage + (g + 8) * kPitch + (16 * s + 4 * tq) * 2);
        qf[s][2] = hi.x;
        qf[s][3] = hi.y;
      }
    }
    sl2[0] = q_scale[g];
    sl2[1] = kTwo ? q_scale[g + 8] : 0.f;
    __syncthreads();
  }

  constexpr int kRows = kTwo ? 2 : 1;
  float o_acc[D / 8][4];   // block 2 j: columns 16 j + 4 tq, + 2; block 2 j + 1: + 1, + 3
#pragma unroll
  for (int n = 0; n < D / 8; ++n)
#pragma unroll
    for (int r = 0; r < 4; ++r) o_acc[n][r] = 0.f;
  float m[kRows], l[kRows], r_exp = -CUDART_INF_F;
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    m[r] = -CUDART_INF_F;
    l[r] = 0.f;
  }

  for (int blk = 0; blk < n_blocks; ++blk) {
    if (blk + kStages - 1 < n_blocks) load_block(blk + kStages - 1);
    cp_async_commit();
    if (blk + kStages < n_blocks) fetch_pages(blk + kStages);
    const int next_scale = blk + 1 < n_blocks ? fetch_scale(blk + 1) : -1;
    cp_async_wait<kStages - 1>();
    __syncthreads();

    const uint32_t kt = smem_base + (blk % kStages) * G::kStageBytes;
    const uint32_t vt = kt + G::kTileBytes;
    const int key_w = s0 + blk * kBlockKeys + warp * 16;   // first key of this warp's 16
    if (key_w < s1) {
      const float* ksc = scales + (blk & 1) * 2 * kBlockKeys + warp * 16;
      const float* vsc = ksc + kBlockKeys;
      // ---- S = Q K^T for 16 keys: two n-blocks of 8 keys
      float sv[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
      {
        // matrices = (keys 0-7, bytes 0-15), (keys 8-15, 0-15), (keys 0-7, 16-31), (keys 8-15, 16-31)
        const uint32_t a0 = kt + (warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * G::kRowBytes + (lane >> 4) * 16;
#pragma unroll
        for (int s = 0; s < KS; s += 2) {
          uint32_t kf[4];
          ldsm_x4(a0 + s * 16, kf);
#pragma unroll
          for (int u = 0; u < 4; ++u) {
            uint32_t b0, b1;
            unpack_e4m3_f16(kf[u], b0, b1);
            const int ks = s + (u >> 1);
            mma_f16(sv[u & 1], qf[ks][0], kTwo ? qf[ks][kTwo ? 2 : 0] : 0u, qf[ks][1], kTwo ? qf[ks][kTwo ? 3 : 0] : 0u, b0, b1);
          }
        }
      }
      float kx[2][2], ev[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n) {
        *reinterpret_cast<float2*>(kx[n]) = *reinterpret_cast<const float2*>(ksc + n * 8 + tq * 2);
        *reinterpret_cast<float2*>(ev[n]) = *reinterpret_cast<const float2*>(vsc + n * 8 + tq * 2);
      }
      const bool tail = key_w + 16 > s1;
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int r = 0; r < 2 * kRows; ++r) {
          sv[n][r] *= kx[n][r & 1];
          if (tail && key_w + n * 8 + tq * 2 + (r & 1) >= s1) sv[n][r] = -CUDART_INF_F;
        }
      // ---- the largest value exponent, and the row maxima; o is rescaled when either reference grows
      const float e_top = quad_max(fmaxf(fmaxf(ev[0][0], ev[0][1]), fmaxf(ev[1][0], ev[1][1])));
      float mn[kRows];
      bool grow = e_top > r_exp;
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        mn[r] = fmaxf(m[r], quad_max(fmaxf(fmaxf(sv[0][2 * r], sv[0][2 * r + 1]), fmaxf(sv[1][2 * r], sv[1][2 * r + 1]))));
        grow |= (mn[r] - m[r]) * sl2[r] > kRescaleThreshold;
      }
      if (__any_sync(0xffffffffu, grow)) {
        const float re = fmaxf(r_exp, e_top);
        const float down = re == r_exp ? 1.f : ex2f(r_exp - re);   // -inf -> 0
        r_exp = re;
        float a[2];
#pragma unroll
        for (int r = 0; r < kRows; ++r) {
          a[r] = mn[r] == m[r] ? 1.f : ex2f((m[r] - mn[r]) * sl2[r]);
          m[r] = mn[r];
          l[r] *= a[r];
          a[r] *= down;
        }
        if (!kTwo) a[1] = a[0];
#pragma unroll
        for (int n = 0; n < D / 8; ++n) {
          o_acc[n][0] *= a[0];
          o_acc[n][1] *= a[0];
          o_acc[n][2] *= a[1];
          o_acc[n][3] *= a[1];
        }
      }
      // ---- probabilities, times the value scale relative to r
      float w[2][2];
#pragma unroll
      for (int n = 0; n < 2; ++n)
#pragma unroll
        for (int e = 0; e < 2; ++e) w[n][e] = ev[n][e] == -CUDART_INF_F ? 0.f : ex2f(ev[n][e] - r_exp + kProbShift);
      uint32_t ph[kRows][2], pl[kRows][2];   // [row][n-block]: hi and lo parts of two keys
#pragma unroll
      for (int r = 0; r < kRows; ++r) {
        const float nm = (m[r] == -CUDART_INF_F) ? 0.f : -m[r] * sl2[r];
        float sum = 0.f;
#pragma unroll
        for (int n = 0; n < 2; ++n) {
          const float p0 = ex2f(fmaf(sv[n][2 * r], sl2[r], nm)), p1 = ex2f(fmaf(sv[n][2 * r + 1], sl2[r], nm));
          sum += p0 + p1;
          split_f16(p0 * w[n][0], p1 * w[n][1], ph[r][n], pl[r][n]);
        }
        l[r] += sum;
      }
      // ---- O += P V: sixteen columns at a time
      {
        // matrices = (keys 0-7, bytes 0-15), (keys 8-15, 0-15), (keys 0-7, 16-31), (keys 8-15, 16-31), transposed
        const uint32_t v0 = vt + (warp * 16 + ((lane >> 3) & 1) * 8 + (lane & 7)) * G::kRowBytes + (lane >> 4) * 16;
#pragma unroll
        for (int j = 0; j < D / 32; ++j) {
          uint32_t vf[4];
          ldsm_x4_trans(v0 + j * 32, vf);
#pragma unroll
          for (int u = 0; u < 2; ++u) {
            uint32_t even0, odd0, even1, odd1;   // keys 0-7 and 8-15 of an even and an odd column
            unpack_e4m3_f16(__byte_perm(vf[2 * u], 0, 0x3120), even0, odd0);
            unpack_e4m3_f16(__byte_perm(vf[2 * u + 1], 0, 0x3120), even1, odd1);
            float(&oe)[4] = o_acc[4 * j + 2 * u];
            float(&oo)[4] = o_acc[4 * j + 2 * u + 1];
            if constexpr (kTwo) {
              mma_f16(oe, ph[0][0], ph[kRows - 1][0], ph[0][1], ph[kRows - 1][1], even0, even1);
              mma_f16(oo, ph[0][0], ph[kRows - 1][0], ph[0][1], ph[kRows - 1][1], odd0, odd1);
              mma_f16(oe, pl[0][0], pl[kRows - 1][0], pl[0][1], pl[kRows - 1][1], even0, even1);
              mma_f16(oo, pl[0][0], pl[kRows - 1][0], pl[0][1], pl[kRows - 1][1], odd0, odd1);
            } else {
              mma_f16(oe, ph[0][0], pl[0][0], ph[0][1], pl[0][1], even0, even1);
              mma_f16(oo, ph[0][0], pl[0][0], ph[0][1], pl[0][1], odd0, odd1);
            }
          }
        }
      }
    }
    store_scale(blk + 1, next_scale);   // the other parity
    __syncthreads();   // the stage may be refilled, and the scales read, from here on
  }
  cp_async_wait<0>();
  pdl_launch_dependents();

  // ---- the four warps' states meet in shared memory
  float* sm_o = reinterpret_cast<float*>(smem);               // [warp][HEADS][D]
  float* sm_ml = sm_o + kWarps * HEADS * D;                   // [warp][HEADS][2] (max in log2 units, sum)
  static_assert(kWarps * HEADS * (D + 2) * 4 <= G::kSmemBytes, "merge buffer must fit");
  __syncthreads();
  const float back = r_exp == -CUDART_INF_F ? 0.f : ex2f(0.5f * (r_exp - kProbShift));   // 2^(r - 9), in two factors
#pragma unroll
  for (int j = 0; j < D / 16; ++j) {
    float(&oe)[4] = o_acc[2 * j];
    float(&oo)[4] = o_acc[2 * j + 1];
    if constexpr (!kTwo) {
#pragma unroll
      for (int r = 0; r < 2; ++r) {
        oe[r] += oe[r + 2];
        oo[r] += oo[r + 2];
      }
    }
#pragma unroll
    for (int r = 0; r < kRows; ++r)
      *reinterpret_cast<float4*>(&sm_o[(warp * HEADS + g + 8 * r) * D + j * 16 + tq * 4]) =
          make_float4(oe[2 * r] * back * back, oo[2 * r] * back * back, oe[2 * r + 1] * back * back, oo[2 * r + 1] * back * back);
  }
#pragma unroll
  for (int r = 0; r < kRows; ++r) {
    const float sum = quad_sum(l[r]);
    if (tq == 0) {
      sm_ml[(warp * HEADS + g + 8 * r) * 2] = m[r] == -CUDART_INF_F ? -CUDART_INF_F : m[r] * sl2[r];
      sm_ml[(warp * HEADS + g + 8 * r) * 2 + 1] = sum;
    }
  }
  __syncthreads();
  for (int idx = tid; idx < n_heads * D; idx += kThreads) {
    const int row = idx / D, d = idx - row * D;
    float mx = -CUDART_INF_F;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) mx = fmaxf(mx, sm_ml[(w * HEADS + row) * 2]);
    const float ms = (mx == -CUDART_INF_F) ? 0.f : mx;
    float o = 0.f, lsum = 0.f;
#pragma unroll
    for (int w = 0; w < kWarps; ++w) {
      const float wgt = ex2f(sm_ml[(w * HEADS + row) * 2] - ms);
      o = fmaf(sm_o[(w * HEADS + row) * D + d], wgt, o);
      lsum = fmaf(sm_ml[(w * HEADS + row) * 2 + 1], wgt, lsum);
    }
    const int64_t slot = (static_cast<int64_t>(b) * p.Hq + (h0 + row)) * nsplit + split;
    if (!dbg_range(p.status, DBG_DECODE_FP8 * 100 + 1, slot, 1, static_cast<int64_t>(p.B) * p.Hq * nsplit) ||
        !dbg_range(p.status, DBG_DECODE_FP8 * 100 + 2, h0 + row, 1, p.Hq))
      continue;
    part_o[slot * D + d] = o;
    if (d == 0) {
      part_ml[slot * 2] = mx;
      part_ml[slot * 2 + 1] = lsum;
    }
  }
}

template <int D, bool BF16, int HEADS>
int launch_one(const Problem& p, const CacheScales& sc, int chunk, int nsplit, float* po, float* pml, cudaStream_t stream) {
  using G = Geo<D>;
  auto kern = decode_fp8_kernel<D, BF16, HEADS>;
  if (cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, G::kSmemBytes) != cudaSuccess) {
    cudaGetLastError();
    return B200_SDPA_ERR_CUDA;
  }
  dim3 grid(p.Hkv * ((p.group + HEADS - 1) / HEADS), p.B, nsplit);
  if (!launch_pdl(kern, grid, kThreads, G::kSmemBytes, stream, p, sc, chunk, nsplit, po, pml)) return B200_SDPA_ERR_CUDA;
  count_launch(KID_DECODE);
  return B200_SDPA_OK;
}

template <int D, bool BF16>
int launch_heads(const Problem& p, const CacheScales& sc, int chunk, int nsplit, float* po, float* pml, cudaStream_t stream) {
  return p.group <= 8 ? launch_one<D, BF16, 8>(p, sc, chunk, nsplit, po, pml, stream)
                      : launch_one<D, BF16, 16>(p, sc, chunk, nsplit, po, pml, stream);
}

}  // namespace

int launch_decode_partial_fp8(const Problem& p, const CacheScales& sc, int dtype, int chunk, int nsplit, float* po, float* pml,
                              cudaStream_t stream) {
  const bool bf16 = dtype == B200_SDPA_BF16;
  if (p.E == 128)
    return bf16 ? launch_heads<128, true>(p, sc, chunk, nsplit, po, pml, stream)
                : launch_heads<128, false>(p, sc, chunk, nsplit, po, pml, stream);
  return bf16 ? launch_heads<64, true>(p, sc, chunk, nsplit, po, pml, stream)
              : launch_heads<64, false>(p, sc, chunk, nsplit, po, pml, stream);
}

}  // namespace b200
