// group4.cu — weights in 4-bit groups: the quantiser, the layout and the
// products y = x W^T (+ b) and down(silu(gate x) * (up x)).
//
//   W[n, k] = scale[n, k / G] * (code[n, k] - zero[n, k / G]),  G = 32, 64, 128,
//   codes 0..15, scales bf16, zero points 0..15 (8 where there are none).
//
// Device layout: blocks of 16 rows x 128 K, [matrix][row tile][chunk], contiguous, so
// that a warp's share of a product is one run of memory that bulk copies bring in:
//   1024 bytes of words: 16 bytes 32 h + 4 g + t hold row 8 h + g's words (h = 0, 1;
//     g = 0..7; t = 0..3), word i (0..3) the chunk's K 32 i + 8 t .. + 7, element
//     2 j + e of a word (e = 0, 1) at bits 16 e + 4 j;
//   32 bytes of bf16 scales for each of the chunk's 128 / G groups: row 8 h + g's at
//     2 g + h;
//   16 bytes of zero points for each group, in the same order (if there are any).
// Rows and K past the matrix have code 8, scale 0 and zero point 8.
#include "common.cuh"
#include "few_stream.cuh"

namespace sb {

__host__ __device__ __forceinline__ int64_t group4_chunks(int64_t K) { return (K + 127) / 128; }
__host__ __device__ __forceinline__ int64_t group4_tiles(int64_t N) { return (N + 15) / 16; }
__host__ __device__ __forceinline__ int group4_block(int gshift, bool zeros) {
  return 1024 + ((zeros ? 48 : 32) << (7 - gshift));
}

// Places inside a block: word m (K 8m .. 8m+7 of the chunk) of row r, scale and zero
// point of row r in group q.
__host__ __device__ __forceinline__ int group4_word_at(int r, int m) {
  return (r >> 3) * 512 + (r & 7) * 64 + (m & 3) * 16 + (m >> 2) * 4;
}
__host__ __device__ __forceinline__ int group4_scale_at(int r, int q) {
  return 1024 + q * 32 + (r & 7) * 4 + (r >> 3) * 2;
}
__host__ __device__ __forceinline__ int group4_zero_at(int r, int q, int gshift) {
  return 1024 + (32 << (7 - gshift)) + q * 16 + (r & 7) * 2 + (r >> 3);
}

// The four codes of K 4h .. 4h+3 (h = 0, 1) of a word, in the word's bit order before a shift by 8h.
__device__ __forceinline__ uint32_t group4_half(uint32_t q0, uint32_t q1, uint32_t q2, uint32_t q3) {
  return q0 | (q1 << 16) | (q2 << 4) | (q3 << 20);
}

// Element e (0..7) of a word.
__device__ __forceinline__ uint32_t group4_code(uint32_t w, int e) { return (w >> (16 * (e & 1) + 4 * (e >> 1))) & 15u; }

// w / s rounded to a whole number, ties to even, as the real quotient rounds (`inv` is
// 1 / s; |w / s| is below 2^20).  The fp32 product is within 2 units of the quotient, so
// its rounding is at most one off; w - q s is exact in one fused multiply-add for such q
// and tells.  Adding and taking away 1.5 x 2^23 rounds.
__device__ __forceinline__ float round_quotient(float w, float s, float inv) {
  float q = __fsub_rn(__fadd_rn(w * inv, 12582912.f), 12582912.f);
  const float r = fmaf(-q, s, w), two = 2.f * fabsf(r), step = copysignf(1.f, r);
  if (two >= s && (two > s || ((int)q & 1))) q += step;
  return q;
}

template <typename TW>
__device__ __forceinline__ float4 load4(const TW* p, int64_t left, bool vec) {
  float4 v = make_float4(0.f, 0.f, 0.f, 0.f);
  if (left <= 0) return v;
  if constexpr (std::is_same<TW, float>::value) {
    if (vec && left >= 4) return __ldg(reinterpret_cast<const float4*>(p));
  } else {
    if (vec && left >= 4) {
      const uint2 u = __ldg(reinterpret_cast<const uint2*>(p));
      return make_float4(__uint_as_float(u.x << 16), __uint_as_float(u.x & 0xFFFF0000u), __uint_as_float(u.y << 16),
                         __uint_as_float(u.y & 0xFFFF0000u));
    }
  }
  v.x = (float)p[0];
  if (left > 1) v.y = (float)p[1];
  if (left > 2) v.z = (float)p[2];
  if (left > 3) v.w = (float)p[3];
  return v;
}

// Quantises `count` matrices W [N, K] (rows `ldw` apart, one matrix after another).
// Symmetric: s = bf16(fp32(absmax / 7)), code = round(w / s) + 8; with zero points
// s = bf16(fp32((hi - lo) / 15)) with 0 in [lo, hi], z = round(-lo / s), code =
// round(w / s) + z; all clamped to 0..15.  s = 0 gives the zero code; a group with a
// non-finite weight (or a span past fp32) gets a NaN scale, so that it cannot pass
// for weights.
//
// Bound by memory and by the quotients' instructions alike: a warp takes 256 K of a row,
// 8 neighbouring weights (a word) per lane, so that a group is 4, 8 or 16 lanes and its
// extremes are 2 to 4 shuffles.
template <typename TW>
__global__ void __launch_bounds__(256) group4_quantize_kernel(const TW* __restrict__ w, int64_t ldw, int64_t count,
                                                              int64_t N, int64_t K, int gshift, bool asym, bool vec,
                                                              bool vec_out, uint8_t* __restrict__ data,
                                                              float* __restrict__ values) {
  const int lane = threadIdx.x & 31;
  const int64_t chunks = group4_chunks(K), pairs = (chunks + 1) / 2, rows = group4_tiles(N) * 16;
  const int span = (1 << gshift) >> 3;  // lanes per group
  const unsigned mask = ((1u << span) - 1u) << (lane & ~(span - 1));
  // (row, pair of chunks) advances by the grid's warps, divided once
  const int64_t stride = ((int64_t)gridDim.x * blockDim.x) >> 5, drow = stride / pairs, dc = stride - drow * pairs;
  const int64_t first = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
  int64_t row = first / pairs, c2 = first - row * pairs;
  for (; row < count * rows; row += drow, c2 += dc) {
    if (c2 >= pairs) {
      c2 -= pairs;
      if (++row >= count * rows) break;
    }
    const int64_t e = count == 1 ? 0 : row / rows, n = row - e * rows, from = e * N + n;
    const int64_t k = c2 * 256 + 8 * lane, left = n < N ? K - k : 0, c = c2 * 2 + (lane >> 4);
    const float4 v0 = load4(w + from * ldw + k, left, vec), v1 = load4(w + from * ldw + k + 4, left - 4, vec);
    const float el[8] = {v0.x, v0.y, v0.z, v0.w, v1.x, v1.y, v1.z, v1.w};
    float hi = 0.f, lo = 0.f;
    bool odd = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      odd |= !isfinite(el[i]);
      hi = fmaxf(hi, el[i]);
      lo = fminf(lo, el[i]);
    }
    for (int o = 1; o < span; o <<= 1) {
      hi = fmaxf(hi, __shfl_xor_sync(0xffffffffu, hi, o));
      lo = fminf(lo, __shfl_xor_sync(0xffffffffu, lo, o));
    }
    const bool bad = (__ballot_sync(0xffffffffu, odd) & mask) != 0;
    const float s32 = asym ? __fdiv_rn(hi - lo, 15.f) : __fdiv_rn(fmaxf(hi, -lo), 7.f);
    __nv_bfloat16 sb = __float2bfloat16_rn(s32);
    const bool off = bad || !isfinite(s32) || __bfloat162float(sb) == 0.f;
    if (bad || !isfinite(s32)) sb = __float2bfloat16_rn(NAN);
    const float s = __bfloat162float(sb);
    // s below 2^-100 (its reciprocal may overflow): both scaled up, exactly
    const float up = s < 0x1p-100f ? 0x1p100f : 1.f, su = s * up, inv = __fdiv_rn(1.f, su);
    const float z = (!asym || off) ? 8.f : fminf(fmaxf(round_quotient(-lo * up, su, inv), 0.f), 15.f);
    float q[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      q[i] = off ? z : fminf(fmaxf(round_quotient(el[i] * up, su, inv) + z, 0.f), 15.f);
      if (i >= left) q[i] = 8.f;
    }
    if (c < chunks) {
      const int r = (int)(n & 15), m = lane & 15;
      uint8_t* block = data + ((e * (rows >> 4) + (n >> 4)) * chunks + c) * group4_block(gshift, asym);
      *reinterpret_cast<uint32_t*>(block + group4_word_at(r, m)) =
          group4_half((uint32_t)q[0], (uint32_t)q[1], (uint32_t)q[2], (uint32_t)q[3]) |
          (group4_half((uint32_t)q[4], (uint32_t)q[5], (uint32_t)q[6], (uint32_t)q[7]) << 8);
      if ((lane & (span - 1)) == 0) {  // (a group past the matrix is all zeros: scale 0, zero point 8)
        const int gq = (8 * m) >> gshift;
        *reinterpret_cast<__nv_bfloat16*>(block + group4_scale_at(r, gq)) = sb;
        if (asym) block[group4_zero_at(r, gq, gshift)] = (uint8_t)z;
      }
    }
    if (values && left > 0) {
      float* d = values + from * K + k;
      if (vec_out && left >= 8) {
        *reinterpret_cast<float4*>(d) = make_float4((q[0] - z) * s, (q[1] - z) * s, (q[2] - z) * s, (q[3] - z) * s);
        *reinterpret_cast<float4*>(d + 4) = make_float4((q[4] - z) * s, (q[5] - z) * s, (q[6] - z) * s, (q[7] - z) * s);
      } else {
#pragma unroll
        for (int i = 0; i < 8; ++i)
          if (i < left) d[i] = (q[i] - z) * s;
      }
    }
  }
}

// codes uint8 [count, N, K], scales bf16 and zeros uint8 (or null) [count, N, ceil(K/G)]
// -> blocks, a thread per word; a code or zero point past 15 is reported and its low
// bits kept
__global__ void group4_pack_kernel(const uint8_t* __restrict__ codes, const __nv_bfloat16* __restrict__ scales,
                                   const uint8_t* __restrict__ zeros, int64_t count, int64_t N, int64_t K, int gshift,
                                   uint8_t* __restrict__ data) {
  const int64_t chunks = group4_chunks(K), rows = group4_tiles(N) * 16, groups = (K + (1 << gshift) - 1) >> gshift;
  const int64_t total = count * rows * chunks * 16;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int m = (int)(i & 15);
    const int64_t row = (i >> 4) / chunks, c = (i >> 4) - row * chunks, e = row / rows, n = row - e * rows;
    const int64_t from = e * N + n, k0 = c * 128 + m * 8;
    uint8_t* block = data + ((e * (rows >> 4) + (n >> 4)) * chunks + c) * group4_block(gshift, zeros != nullptr);
    const int r = (int)(n & 15);
    uint32_t q[8];
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      q[j] = n < N && k0 + j < K ? codes[from * K + k0 + j] : 8u;
      if (q[j] > 15u) set_status(ST_BAD_ARGUMENT);
      q[j] &= 15u;
    }
    *reinterpret_cast<uint32_t*>(block + group4_word_at(r, m)) =
        group4_half(q[0], q[1], q[2], q[3]) | (group4_half(q[4], q[5], q[6], q[7]) << 8);
    if ((k0 & ((1 << gshift) - 1)) == 0) {
      const int64_t g = k0 >> gshift;
      const bool in = n < N && k0 < K;
      const int gq = (m * 8) >> gshift;
      *reinterpret_cast<__nv_bfloat16*>(block + group4_scale_at(r, gq)) =
          in ? scales[from * groups + g] : __float2bfloat16_rn(0.f);
      if (zeros) {
        const uint8_t z = in ? zeros[from * groups + g] : 8u;
        if (z > 15u) set_status(ST_BAD_ARGUMENT);
        block[group4_zero_at(r, gq, gshift)] = z & 15u;
      }
    }
  }
}

// blocks -> values [count * N, ldo] (columns past K: zero), a thread per word
template <typename TO>
__global__ void group4_dequant_kernel(const uint8_t* __restrict__ data, bool asym, int64_t count, int64_t N, int64_t K,
                                      int gshift, TO* __restrict__ out, int64_t ldo, bool vec) {
  const int64_t chunks = group4_chunks(K), tiles = group4_tiles(N), per = (ldo + 7) / 8, total = count * N * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t row = i / per, m = i - row * per, k = m * 8, e = row / N, n = row - e * N;
    float v[8];
    if (k < K) {
      const uint8_t* block = data + ((e * tiles + (n >> 4)) * chunks + (m >> 4)) * group4_block(gshift, asym);
      const int r = (int)(n & 15), mm = (int)(m & 15), gq = (mm * 8) >> gshift;
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(block + group4_word_at(r, mm)));
      const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + group4_scale_at(r, gq)));
      const int z = asym ? block[group4_zero_at(r, gq, gshift)] : 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = k + j < K ? (float)((int)group4_code(w, j) - z) * s : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) v[j] = 0.f;
    }
    TO* d = out + row * ldo + k;
    if constexpr (std::is_same<TO, float>::value) {
      if (vec && k + 8 <= ldo) {
        *reinterpret_cast<float4*>(d) = make_float4(v[0], v[1], v[2], v[3]);
        *reinterpret_cast<float4*>(d + 4) = make_float4(v[4], v[5], v[6], v[7]);
        continue;
      }
    } else {
      if (vec && k + 8 <= ldo) {
        __nv_bfloat162 p[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) p[j] = __floats2bfloat162_rn(v[2 * j], v[2 * j + 1]);
        *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(p);
        continue;
      }
    }
#pragma unroll
    for (int j = 0; j < 8; ++j)
      if (k + j < ldo) d[j] = (TO)v[j];
  }
}

// ---------------------------------------------------------------------------
// tokens as planes
// ---------------------------------------------------------------------------
// Rows of x as T bf16 planes of rows `ldp` long (a multiple of 8, the tail zero):
// fp32 rows in three planes, bf16 rows that the kernels cannot load 16 bytes at a
// time copied as they are.
template <typename TX, int T>
__global__ void few_planes_kernel(const TX* __restrict__ x, int64_t ldx, int64_t M, int K, __nv_bfloat16* planes,
                                  int64_t ldp) {
  few_wait();
  few_trigger();
  const int64_t total = M * ldp, plane = total;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t m = i / ldp, k = i % ldp;
    __nv_bfloat16 p[T];
    split_planes<T>(k < K ? (float)x[m * ldx + k] : 0.f, p);
#pragma unroll
    for (int q = 0; q < T; ++q) planes[q * plane + i] = p[q];
  }
}

// Tokens as the kernels take them (FewX): x itself where its rows can be loaded 16
// bytes at a time, else planes in a workspace (few_planes_bytes of it).
inline int64_t align8(int64_t v) { return (v + 7) / 8 * 8; }

inline bool few_planes_needed(const void* x, int x_dtype, int64_t ldx, int64_t K) {
  return x_dtype != SB_BF16 || (reinterpret_cast<uintptr_t>(x) & 15u) != 0 || ldx % 8 != 0 || K % 8 != 0;
}
inline size_t few_planes_bytes(int x_dtype, int64_t M, int64_t K) {
  return align_up((size_t)(x_dtype == SB_BF16 ? 1 : 3) * M * align8(K) * 2, 256);
}

// ---------------------------------------------------------------------------
// launching the stream
// ---------------------------------------------------------------------------
constexpr int FEW_SMEM = 232448;      // a block's shared memory at most
constexpr int64_t FEW_MAX_K = 16384;  // one staged fp32 token (three planes) is 96 KB, beside rings of 92 KB

// A block's shared memory beside the staged tokens and the work's lists: rings of
// `depth` slots, their barriers and the tails' sums.
template <class W>
int few_fixed_bytes(int nt, int rt, int warps, int depth) {
  return warps * (depth * (rt * W::SLOT + 8) + rt * nt * 512);
}

// A launch whose kernel may begin while the one before it on the stream ends and
// waits itself for that one's results: at once, or, where the one before is of the
// same call, after what does not depend on them.
template <typename... P, typename... A>
int few_launch(void (*kern)(P...), dim3 grid, int threads, size_t smem, cudaStream_t st, A... args) {
  cudaLaunchConfig_t cfg{};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = grid;
  cfg.blockDim = dim3(threads);
  cfg.dynamicSmemBytes = smem;
  cfg.stream = st;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  SB_CUDA_TRY(cudaLaunchKernelEx(&cfg, kern, static_cast<P>(args)...));
  return SB_OK;
}

inline int few_planes(const void* x, int x_dtype, int64_t ldx, int64_t M, int64_t K, void* ws, FewX* out,
                      cudaStream_t st) {
  if (!few_planes_needed(x, x_dtype, ldx, K)) {
    *out = FewX{static_cast<const __nv_bfloat16*>(x), ldx, 0, (int)K};
    return SB_OK;
  }
  const int64_t ldp = align8(K);
  __nv_bfloat16* p = static_cast<__nv_bfloat16*>(ws);
  int64_t blocks = (M * ldp + 255) / 256;
  if (blocks > (int64_t)num_sms() * 16) blocks = (int64_t)num_sms() * 16;
  ProfScope prof("few_planes", st);
  const int rc = x_dtype == SB_BF16
                     ? few_launch(few_planes_kernel<__nv_bfloat16, 1>, dim3((unsigned)blocks), 256, 0, st,
                                  static_cast<const __nv_bfloat16*>(x), ldx, M, (int)K, p, ldp)
                     : few_launch(few_planes_kernel<float, 3>, dim3((unsigned)blocks), 256, 0, st,
                                  static_cast<const float*>(x), ldx, M, (int)K, p, ldp);
  if (rc) return rc;
  *out = FewX{p, ldp, M * ldp, (int)ldp};
  return SB_OK;
}

// A kernel's shared-memory limit, raised once per device.
template <typename K>
int few_allow_smem(PerDevice& once, K kern) {
  int dev = 0;
  SB_CUDA_TRY(cudaGetDevice(&dev));
  return once.once(dev, [&]() -> int {
    SB_CUDA_TRY(cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, FEW_SMEM));
    return SB_OK;
  });
}

template <class W, bool GATEUP, int T, int TH, int NT, int RT, int WARPS, class Work>
int launch_few_stream(const char* name, const W& w0, const W& w1, const FewX& x, const Work& work, int64_t N, int tile,
                      const FewHidden& hidden, const FewRows& rows, bool after, cudaStream_t st) {
  auto kern = few_stream_kernel<W, GATEUP, T, TH, NT, RT, WARPS, Work>;
  static PerDevice attr;
  int rc;
  if ((rc = few_allow_smem(attr, kern))) return rc;
  constexpr int UNIT = (GATEUP ? 1 : RT) * 16;
  FewShape sh{};
  sh.N = (int)N;
  sh.tile_tokens = tile;
  sh.tiles = (int)((N + UNIT - 1) / UNIT);
  sh.early = after;
  sh.tokens_last = after && !work.waits();
  const int64_t groups = work.groups(tile), units = groups * sh.tiles;
  if (units >= (1ll << 26)) return fail(SB_ERR_INVALID, "%s: too many outputs for one call", name);
  sh.groups = (int)groups;
  // as many ring slots as fit, 2 to 8
  const size_t fixed = (size_t)tile * T * few_row_bytes(w0.chunks * W::CHUNK) + work.bytes();
  constexpr size_t ROOM = (size_t)FEW_SMEM / (16 / WARPS) - 1024;
  sh.depth = 2;
  while (sh.depth < 8 && fixed + few_fixed_bytes<W>(NT, RT, WARPS, sh.depth + 1) <= ROOM) ++sh.depth;
  const size_t smem = fixed + few_fixed_bytes<W>(NT, RT, WARPS, sh.depth);
  const int64_t most = (int64_t)num_sms() * (16 / WARPS), blocks = units < most ? units : most;
  // A block that goes on to another group waits for its warps and stages tokens: some 3 to 5
  // units' time.  Counted as 5 / 0 where a block has 2 units: 64 tokens, top 8 of 64 4-bit
  // experts 97.0 / 100.0 us; MLP [1024 x 2048] x 2 + [2048 x 1024] at 300 tokens 32.3 / 38.8, at
  // 100 21.2 / 27.7; [4096 x 2048] at 48 9.9 / 13.7.  (3: 33.8 and 8: 33.4 at 300 tokens.)
  sh.start = groups > 1 && units >= 2 * blocks ? 5 : 0;
  ProfScope prof(name, st);
  return few_launch(kern, dim3((unsigned)blocks), WARPS * 32, smem, st, w0, w1, x, work, sh, hidden, rows);
}

// The kernel for groups of up to `most` tokens, and how many of them a block stages.  Two
// column tiles against one: whole layer 76.7 / 78.8 us at 12 tokens, 78.9 / 82.4 at 16 (64
// experts, top 8), [4096 x 2048] at 128 tokens 18.7 / 26.5.
template <class W, bool GATEUP, int T, int TH, class Work>
int few_stream(const char* name, const W& w0, const W& w1, const FewX& x, const Work& work, int64_t most, int64_t N,
               const FewHidden& hidden, const FewRows& rows, bool after, cudaStream_t st) {
  const int64_t row = (int64_t)T * few_row_bytes(w0.chunks * W::CHUNK);
  constexpr int R1 = GATEUP ? 2 : 1;
  auto fit = [&](int nt, int rt, int warps, int depth) {  // in an SM's share of a block
    const int64_t left =
        FEW_SMEM / (16 / warps) - 1024 - few_fixed_bytes<W>(nt, rt, warps, depth) - (int64_t)work.bytes();
    const int64_t n = most < nt * 8 ? most : nt * 8;
    return (int)(left / row < n ? left / row : n);
  };
  int tile;
  if (most > 8 && (tile = fit(2, 2, 16, 2)) > 8)
    return launch_few_stream<W, GATEUP, T, TH, 2, 2, 16>(name, w0, w1, x, work, N, tile, hidden, rows, after, st);
  if ((tile = fit(1, R1, 8, 8 / R1)) == (most < 8 ? most : 8))
    return launch_few_stream<W, GATEUP, T, TH, 1, R1, 8>(name, w0, w1, x, work, N, tile, hidden, rows, after, st);
  if ((tile = fit(1, R1, 16, 2)) < 1) return fail(SB_ERR_INVALID, "%s: one token does not fit in shared memory", name);
  return launch_few_stream<W, GATEUP, T, TH, 1, R1, 16>(name, w0, w1, x, work, N, tile, hidden, rows, after, st);
}

template <int T, int G>
int few_linear(const char* name, const Group4W<G>& w, const FewX& x, int64_t M, int64_t N, const float* bias, void* y,
               int y_dtype, bool after, cudaStream_t st) {
  return few_stream<Group4W<G>, false, T, 1>(name, w, w, x, FewContiguous{(int)M}, M, N, FewHidden{},
                                             FewRows{y, y_dtype, bias}, after, st);
}

inline int group_shift(int64_t group) { return group == 32 ? 5 : group == 64 ? 6 : group == 128 ? 7 : -1; }

template <int G>
Group4W<G> group4_weights(const sb_group4* m) {
  return Group4W<G>{static_cast<const uint8_t*>(m->data), (int)group4_chunks(m->K), (int)group4_tiles(m->N),
                    group4_block(group_shift(G), m->zeros != 0)};
}

// f(group size as a constant)
template <typename F>
int with_group(int group, F f) {
  if (group == 32) return f(std::integral_constant<int, 32>{});
  if (group == 64) return f(std::integral_constant<int, 64>{});
  return f(std::integral_constant<int, 128>{});
}

inline int check_group4(const sb_group4* m, const char* what) {
  SB_REQUIRE(m, "%s: null matrix", what);
  SB_REQUIRE(m->K > 0 && m->N > 0 && m->count > 0, "%s: shape must be positive (count=%lld N=%lld K=%lld)", what,
             (long long)m->count, (long long)m->N, (long long)m->K);
  SB_REQUIRE(m->K <= FEW_MAX_K && m->N <= (1 << 24) && m->count <= (1 << 20),
             "%s: K is limited to %d, N to 2^24, count to 2^20", what, (int)FEW_MAX_K);
  SB_REQUIRE(group_shift(m->group) > 0, "%s: group %d must be 32, 64 or 128", what, (int)m->group);
  SB_REQUIRE(m->data, "%s: null data", what);
  SB_REQUIRE((reinterpret_cast<uintptr_t>(m->data) & 15u) == 0, "%s: packed data must be 16-byte aligned", what);
  return SB_OK;
}
// A matrix that one product takes
inline int check_group4_one(const sb_group4* m, const char* what) {
  const int rc = check_group4(m, what);
  if (rc) return rc;
  SB_REQUIRE(m->count == 1, "%s: one matrix, got %lld", what, (long long)m->count);
  return SB_OK;
}

inline int check_few_x(const void* x, int x_dtype, int64_t ldx, int64_t M, int64_t K, const char* what) {
  SB_REQUIRE(x_dtype == SB_F32 || x_dtype == SB_BF16, "%s: x dtype must be SB_F32 or SB_BF16", what);
  SB_REQUIRE(M >= 0 && M <= (1 << 20), "%s: %lld tokens (0 to 2^20)", what, (long long)M);
  SB_REQUIRE(M == 0 || x, "%s: x is null", what);
  SB_REQUIRE(ldx >= K || M <= 1, "%s: rows of x overlap (stride %lld, %lld columns)", what, (long long)ldx,
             (long long)K);
  return SB_OK;
}

inline int check_workspace(const void* ws, size_t have, size_t need) {
  if (need && (!ws || have < need))
    return fail(SB_ERR_WORKSPACE, "workspace of %zu bytes is smaller than the %zu needed", have, need);
  SB_REQUIRE((reinterpret_cast<uintptr_t>(ws) & 255u) == 0, "workspace must be 256-byte aligned");
  return SB_OK;
}

// ---------------------------------------------------------------------------
// many tokens
// ---------------------------------------------------------------------------
// From a few hundred tokens on a product is a matrix product, and the tensor cores
// are fed best by the persistent tcgen05 GEMM (gemm_tc.cuh) on weights written out in
// 16 bits once: N x K x 4 bytes, against M x N x K products.  A value has 13
// significant bits (a code's 5 times a scale's 8), so it is two bf16 terms exactly,
// hi + lo, and the sum runs over x lo + x hi: twice the matrix work, where one rounded
// term would add as much error as the output's own rounding.  The accumulator
// truncates every step's sum, so the small terms go first: their steps lose 2^-8 of what
// they would behind the large ones.  What the large ones' K / 16 steps lose is seen in fp32
// outputs alone, off by (normwise; in brackets with the large terms first; the short form
// 0.6 to 1.8e-7) 1.6e-6 (4.3e-6) at K = 2048, 7.7e-6 (2.0e-5) at 8192, 1.6e-5 (4.1e-5) at
// 16384.  (fp32 activations would take six terms: they stay with the stream.)
//
// Which form is the faster one: see long_linear().

// values of a matrix as rows of [hi | lo], kp columns each (zeros past K); row n of the
// matrix goes to row n * step + off
__global__ void group4_terms_kernel(const uint8_t* __restrict__ data, bool asym, int64_t N, int64_t K, int gshift,
                                    int64_t kp, int step, int off, __nv_bfloat16* __restrict__ out) {
  few_wait();
  few_trigger();
  const int64_t chunks = group4_chunks(K), per = kp / 8, total = N * per;
  for (int64_t i = (int64_t)blockIdx.x * blockDim.x + threadIdx.x; i < total; i += (int64_t)gridDim.x * blockDim.x) {
    const int64_t n = i / per, m = i - n * per, k = m * 8;
    __nv_bfloat16 hi[8], lo[8];
    if (k < K) {
      const uint8_t* block = data + ((n >> 4) * chunks + (m >> 4)) * group4_block(gshift, asym);
      const int r = (int)(n & 15), mm = (int)(m & 15), gq = (mm * 8) >> gshift;
      const uint32_t w = __ldg(reinterpret_cast<const uint32_t*>(block + group4_word_at(r, mm)));
      const float s = __bfloat162float(*reinterpret_cast<const __nv_bfloat16*>(block + group4_scale_at(r, gq)));
      const int z = asym ? block[group4_zero_at(r, gq, gshift)] : 8;
#pragma unroll
      for (int j = 0; j < 8; ++j) {
        __nv_bfloat16 p[2];
        split_planes<2>(k + j < K ? (float)((int)group4_code(w, j) - z) * s : 0.f, p);
        hi[j] = p[0];
        lo[j] = p[1];
      }
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) hi[j] = lo[j] = __float2bfloat16_rn(0.f);
    }
    __nv_bfloat16* d = out + (n * step + off) * 2 * kp + k;
    *reinterpret_cast<uint4*>(d) = *reinterpret_cast<const uint4*>(hi);
    *reinterpret_cast<uint4*>(d + kp) = *reinterpret_cast<const uint4*>(lo);
  }
}

// y = x lo + x hi (+ bias): the tokens' K blocks twice
struct EpiGroup4Rows {
  const float* bias;
  void* y;
  int64_t ldo;
  int dtype, N, kb;  // kb: K blocks of a term
  __device__ __forceinline__ int a_block(int i) const { return i < kb ? i : i - kb; }
  __device__ __forceinline__ int b_block(int i) const { return i < kb ? i + kb : i - kb; }
  __device__ __forceinline__ void apply(int64_t row, int col0, const uint32_t (&r)[32]) const {
    if (dtype == SB_BF16 && col0 + 32 <= N && (ldo & 7) == 0 && (reinterpret_cast<uintptr_t>(y) & 15u) == 0) {
      uint32_t p[16];
#pragma unroll
      for (int j = 0; j < 16; ++j) {
        float a = __uint_as_float(r[2 * j]), b = __uint_as_float(r[2 * j + 1]);
        if (bias) {
          a += __ldg(bias + col0 + 2 * j);
          b += __ldg(bias + col0 + 2 * j + 1);
        }
        const __nv_bfloat162 v = __floats2bfloat162_rn(a, b);
        p[j] = *reinterpret_cast<const uint32_t*>(&v);
      }
      uint4* d = reinterpret_cast<uint4*>(static_cast<__nv_bfloat16*>(y) + row * ldo + col0);
#pragma unroll
      for (int j = 0; j < 4; ++j) d[j] = make_uint4(p[4 * j], p[4 * j + 1], p[4 * j + 2], p[4 * j + 3]);
    } else {
#pragma unroll
      for (int j = 0; j < 32; ++j)
        if (col0 + j < N)
          store_out(y, dtype, row * ldo + col0 + j, __uint_as_float(r[j]) + (bias ? __ldg(bias + col0 + j) : 0.f));
    }
  }
  __device__ __forceinline__ void tail(int64_t, const uint32_t (&)[32]) const {}
};

// h = silu(gate) * up from columns gate, up, gate, up, ..., as rows of [hi | lo], ip columns each
struct EpiGroup4Hidden {
  __nv_bfloat16* h;
  int64_t ip;
  int I, kb;
  __device__ __forceinline__ int a_block(int i) const { return i < kb ? i : i - kb; }
  __device__ __forceinline__ int b_block(int i) const { return i < kb ? i + kb : i - kb; }
  __device__ __forceinline__ void apply(int64_t row, int col0, const uint32_t (&r)[32]) const {
    __nv_bfloat16 hi[16], lo[16];
    const int c0 = col0 / 2;
#pragma unroll
    for (int j = 0; j < 16; ++j) {
      const float g = __uint_as_float(r[2 * j]), u = __uint_as_float(r[2 * j + 1]);
      __nv_bfloat16 p[2];
      split_planes<2>(c0 + j < I ? g / (1.f + expf(-g)) * u : 0.f, p);
      hi[j] = p[0];
      lo[j] = p[1];
    }
    __nv_bfloat16* d = h + row * 2 * ip + c0;  // ip is a multiple of 64: whole 16-byte pieces
#pragma unroll
    for (int j = 0; j < 2; ++j)
      if (c0 + 8 * j < ip) {
        reinterpret_cast<uint4*>(d)[j] = reinterpret_cast<const uint4*>(hi)[j];
        reinterpret_cast<uint4*>(d + ip)[j] = reinterpret_cast<const uint4*>(lo)[j];
      }
  }
  __device__ __forceinline__ void tail(int64_t, const uint32_t (&)[32]) const {}
};

// y = h_lo w_hi + h_hi w_lo + h_hi w_hi (what is left out, h_lo w_lo, is 2^-16 of it)
struct EpiGroup4Down : EpiGroup4Rows {
  __device__ __forceinline__ int a_block(int i) const { return i < kb ? i + kb : i < 2 * kb ? i - kb : i - 2 * kb; }
  __device__ __forceinline__ int b_block(int i) const { return i < 2 * kb ? i : i - 2 * kb; }
};

inline int64_t align64(int64_t v) { return (v + 63) / 64 * 64; }

// Tokens that the short form serves with one pass over the weights: as many as it can
// stage (few_stream's choice, for groups of 128) in T planes of K.
inline int64_t few_pass_tokens(int T, int64_t K, int rt) {
  using W = Group4W<128>;
  const int64_t row = (int64_t)T * few_row_bytes((int)group4_chunks(K) * W::CHUNK);
  const int64_t two = (FEW_SMEM - 1024 - few_fixed_bytes<W>(2, 2, 16, 2)) / row;
  if (two > 8) return two < 16 ? two : 16;
  const int64_t one = (FEW_SMEM - 1024 - few_fixed_bytes<W>(1, rt, 16, 2)) / row;
  return one < 8 ? one : 8;
}

// Whether a product takes the long form.  The short one pays for every pass over the N x
// K weights; the long one about 6 passes' time for writing the terms out and then, however
// few the tokens, the steps of a tile along 2 K (as much as a pass over 62500 rows) or
// the terms' way back in (10 passes).  Short / long in us on a B200:
//   K, N          2048, 4096             4096, 14336              14336, 4096
//   tokens        256   25.4 /  32.6     176    97.2 / 134.8      64    92 / 185
//                 320   30.1 /  33.0     256   142.4 / 135.6      128  172 / 184
//                                        512   267   / 190        320  411 / 187
//   K, N          2048, 1024             16384, 1024              72, 48
//                 1024  25.8 /  27.1     256   128 / 157          2048   5.7 / 8.6
//                 2048  46.1 /  28.1     320   152 / 156          4096   8.6 / 8.7
inline bool long_linear(int x_dtype, int64_t M, int64_t K, int64_t N) {
  if (x_dtype != SB_BF16) return false;
  const int64_t tokens = few_pass_tokens(1, K, 1), passes = (M + tokens - 1) / tokens;
  return (passes - 6) * N >= (N > 6250 ? 10 * N : 62500);
}
// The MLP by the same reckoning: gate and up 2 I x H, down H x I with a hidden state of
// two planes (a quarter more for a pass) and, in the long form, over 3 I; a tenth more
// for the long form's other launches.
//   H, I          2048, 1024             4096, 14336              2048, 8192
//   tokens        512   48.0 /  56.2     96   434 / 491           192  181 / 228
//                 704   63.4 /  62.8     128  569 / 490           256  237 / 228
//   H, I          1024, 512              7168, 2048               256, 512
//                 704   29.2 /  32.8     192  142 / 157           2048  32.8 / 26.6
//                 1024  35.3 /  33.3     256  184 / 156           4096  48.4 / 33.2
inline bool long_mlp(int x_dtype, int64_t M, int64_t H, int64_t I) {
  if (x_dtype != SB_BF16) return false;
  const int64_t t1 = few_pass_tokens(1, H, 2), t2 = few_pass_tokens(2, I, 1);
  const double p1 = (double)((M + t1 - 1) / t1), p2 = (double)((M + t2 - 1) / t2), w = (double)H * I;
  const double gateup = 20. * I > 62500. ? 20. * I : 62500., down = 10. * H > 93750. ? 10. * H : 93750.;
  return (2 * p1 + 1.25 * p2) * w >= 1.1 * (18 * w + gateup * H + down * I);
}

inline int group4_terms(const sb_group4* m, int64_t kp, int step, int off, __nv_bfloat16* out, cudaStream_t st) {
  int64_t blocks = (m->N * (kp / 8) + 255) / 256;
  if (blocks > (int64_t)num_sms() * 16) blocks = (int64_t)num_sms() * 16;
  ProfScope prof("group4_terms", st);
  return few_launch(group4_terms_kernel, dim3((unsigned)blocks), 256, 0, st, static_cast<const uint8_t*>(m->data),
                    m->zeros != 0, m->N, m->K, group_shift(m->group), kp, step, off, out);
}

// x [M, ..] (row stride ldx, `ka` columns) times w [rows, 2 kp] over `kb` K blocks, for N
// columns (those past `rows`: zero); the tile's width by how many tiles that leaves for
// the SMs
template <class Epi>
int group4_gemm(const char* name, const __nv_bfloat16* x, int64_t ldx, int64_t ka, int64_t M, const __nv_bfloat16* w,
                int64_t kp, int64_t rows, int64_t N, int kb, const Epi& epi, cudaStream_t st) {
  CUtensorMap ta, tb;
  int rc;
  if ((rc = make_tmap_2d(&ta, x, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)M, (uint64_t)ka, (uint64_t)ldx, 64, 128,
                         CU_TENSOR_MAP_SWIZZLE_128B)))
    return rc;
  const int64_t mt = (M + 127) / 128;
  auto go = [&](auto bn) -> int {
    constexpr int BN = decltype(bn)::value;
    if ((rc = make_tmap_2d(&tb, w, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 2, (uint64_t)rows, (uint64_t)(2 * kp), (uint64_t)(2 * kp),
                           64, BN, CU_TENSOR_MAP_SWIZZLE_128B)))
      return rc;
    // as many stages as fit: a tile's K loop waits on memory
    return launch_gemm_tc<BN, BN == 256 ? 4 : BN == 128 ? 6 : 8>(name, ta, tb, tb, (int)M, (int)N, kb * 64, epi, st);
  };
  // rounds of tiles over the SMs, a tile costing its columns and about 64 more
  auto cost = [&](int64_t bn) { return (mt * ((N + bn - 1) / bn) + num_sms() - 1) / num_sms() * (bn + 64); };
  if (cost(256) <= cost(128) && cost(256) <= cost(64)) return go(std::integral_constant<int, 256>{});
  if (cost(128) <= cost(64)) return go(std::integral_constant<int, 128>{});
  return go(std::integral_constant<int, 64>{});
}

}  // namespace sb

extern "C" size_t sb_group4_matrix_bytes(int64_t K, int64_t N, int32_t group, int zeros) {
  if (K <= 0 || N <= 0 || sb::group_shift(group) < 0) return 0;
  return (size_t)(sb::group4_tiles(N) * sb::group4_chunks(K) * sb::group4_block(sb::group_shift(group), zeros != 0));
}

extern "C" int sb_group4_quantize(const void* w, int w_dtype, int64_t ldw, const sb_group4* out, float* values,
                                  void* stream) {
  using namespace sb;
  int rc;
  if ((rc = check_group4(out, "sb_group4_quantize"))) return rc;
  SB_REQUIRE(w_dtype == SB_F32 || w_dtype == SB_BF16, "sb_group4_quantize: w dtype must be SB_F32 or SB_BF16");
  SB_REQUIRE(w, "sb_group4_quantize: w is null");
  SB_REQUIRE(ldw >= out->K, "sb_group4_quantize: row stride %lld below K=%lld", (long long)ldw, (long long)out->K);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t blocks = (out->count * group4_tiles(out->N) * 16 * ((group4_chunks(out->K) + 1) / 2) + 7) / 8;
  if (blocks > (int64_t)num_sms() * 64) blocks = (int64_t)num_sms() * 64;
  const int sh = group_shift(out->group);
  const bool vec_out = values && out->K % 4 == 0 && (reinterpret_cast<uintptr_t>(values) & 15u) == 0;
  const size_t el = w_dtype == SB_BF16 ? 2 : 4;
  const bool vec = ldw % 4 == 0 && (reinterpret_cast<uintptr_t>(w) & (4 * el - 1)) == 0;
  auto* data = static_cast<uint8_t*>(out->data);
  ProfScope prof("group4_quantize", st);
  if (w_dtype == SB_BF16)
    group4_quantize_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, st>>>(
        static_cast<const __nv_bfloat16*>(w), ldw, out->count, out->N, out->K, sh, out->zeros != 0, vec, vec_out, data,
        values);
  else
    group4_quantize_kernel<float><<<(unsigned)blocks, 256, 0, st>>>(static_cast<const float*>(w), ldw, out->count, out->N,
                                                                    out->K, sh, out->zeros != 0, vec, vec_out, data,
                                                                    values);
  SB_CUDA_TRY(cudaGetLastError());
  return SB_OK;
}

extern "C" int sb_group4_pack(const uint8_t* codes, const void* scales, const uint8_t* zeros, const sb_group4* out,
                              void* stream) {
  using namespace sb;
  int rc;
  if ((rc = check_group4(out, "sb_group4_pack"))) return rc;
  SB_REQUIRE(codes && scales, "sb_group4_pack: null codes or scales");
  SB_REQUIRE(!zeros == !out->zeros, "sb_group4_pack: zero points given for a matrix without, or the reverse");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t blocks = (out->count * group4_tiles(out->N) * group4_chunks(out->K) * 256 + 255) / 256;
  if (blocks > (int64_t)num_sms() * 64) blocks = (int64_t)num_sms() * 64;
  group4_pack_kernel<<<(unsigned)blocks, 256, 0, st>>>(codes, static_cast<const __nv_bfloat16*>(scales), zeros,
                                                       out->count, out->N, out->K, group_shift(out->group),
                                                       static_cast<uint8_t*>(out->data));
  SB_CUDA_TRY(cudaGetLastError());
  return SB_OK;
}

extern "C" int sb_group4_dequantize(const sb_group4* m, void* out, int out_dtype, void* stream) {
  using namespace sb;
  int rc;
  if ((rc = check_group4(m, "sb_group4_dequantize"))) return rc;
  SB_REQUIRE(out, "sb_group4_dequantize: out is null");
  SB_REQUIRE(out_dtype == SB_F32 || out_dtype == SB_BF16, "sb_group4_dequantize: out dtype must be SB_F32 or SB_BF16");
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  int64_t blocks = (m->count * m->N * ((m->K + 7) / 8) + 255) / 256;
  if (blocks > (int64_t)num_sms() * 64) blocks = (int64_t)num_sms() * 64;
  const bool vec = m->K % 8 == 0 && (reinterpret_cast<uintptr_t>(out) & 15u) == 0;
  const auto* data = static_cast<const uint8_t*>(m->data);
  const int sh = group_shift(m->group);
  ProfScope prof("group4_dequant", st);
  if (out_dtype == SB_F32)
    group4_dequant_kernel<float><<<(unsigned)blocks, 256, 0, st>>>(data, m->zeros != 0, m->count, m->N, m->K, sh,
                                                                   static_cast<float*>(out), m->K, vec);
  else
    group4_dequant_kernel<__nv_bfloat16><<<(unsigned)blocks, 256, 0, st>>>(
        data, m->zeros != 0, m->count, m->N, m->K, sh, static_cast<__nv_bfloat16*>(out), m->K, vec);
  SB_CUDA_TRY(cudaGetLastError());
  return SB_OK;
}

extern "C" size_t sb_group4_linear_workspace_bytes(int x_dtype, int64_t M, int64_t K, int64_t N) {
  if (M < 0 || K <= 0 || N <= 0) return 0;
  return sb::few_planes_bytes(x_dtype, M, K) +
         (K <= sb::FEW_MAX_K && sb::long_linear(x_dtype, M, K, N) ? sb::align_up((size_t)(N * sb::align64(K) * 4), 256) : 0);
}

extern "C" int sb_group4_linear(const void* x, int x_dtype, int64_t ldx, int64_t M, const sb_group4* w,
                                const float* bias, void* y, int y_dtype, void* workspace, size_t workspace_bytes,
                                void* stream) {
  using namespace sb;
  int rc;
  if ((rc = check_group4_one(w, "sb_group4_linear")) || (rc = check_few_x(x, x_dtype, ldx, M, w->K, "sb_group4_linear")))
    return rc;
  SB_REQUIRE(y_dtype == SB_F32 || y_dtype == SB_BF16, "sb_group4_linear: y dtype must be SB_F32 or SB_BF16");
  if (M == 0) return SB_OK;
  SB_REQUIRE(y, "sb_group4_linear: y is null");
  // rows that the kernel reads in place need no workspace
  const bool after = few_planes_needed(x, x_dtype, ldx, w->K), many = long_linear(x_dtype, M, w->K, w->N);
  if ((after || many) && (rc = check_workspace(workspace, workspace_bytes,
                                     sb_group4_linear_workspace_bytes(x_dtype, M, w->K, w->N))))
    return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  FewX fx;
  if ((rc = few_planes(x, x_dtype, ldx, M, w->K, workspace, &fx, st))) return rc;
  if (many) {
    auto* terms = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(workspace) + few_planes_bytes(x_dtype, M, w->K));
    const int64_t kp = align64(w->K);
    if ((rc = group4_terms(w, kp, 1, 0, terms, st))) return rc;
    const int kb = (int)(kp / 64);
    return group4_gemm("group4_linear_tc", fx.base, fx.ld, w->K, M, terms, kp, w->N, w->N, 2 * kb,
                       EpiGroup4Rows{bias, y, w->N, y_dtype, (int)w->N, kb}, st);
  }
  return with_group(w->group, [&](auto g) {
    const auto gw = group4_weights<g.value>(w);
    if (x_dtype == SB_BF16) return few_linear<1>("group4_linear", gw, fx, M, w->N, bias, y, y_dtype, after, st);
    return few_linear<3>("group4_linear", gw, fx, M, w->N, bias, y, y_dtype, after, st);
  });
}

extern "C" size_t sb_group4_gated_mlp_workspace_bytes(int x_dtype, int64_t M, int64_t H, int64_t I) {
  if (M < 0 || H <= 0 || I <= 0) return 0;
  // hidden rows [hi | lo] and, one after the other, the terms of gate and up, of down
  if (H <= sb::FEW_MAX_K && I <= sb::FEW_MAX_K && sb::long_mlp(x_dtype, M, H, I))
    return sb::few_planes_bytes(x_dtype, M, H) + sb::align_up((size_t)(M * sb::align64(I) * 4), 256) +
           sb::align_up((size_t)(2 * I * sb::align64(H) * 4), 256) + sb::align_up((size_t)(H * sb::align64(I) * 4), 256);
  return sb::few_planes_bytes(x_dtype, M, H) +
         sb::align_up((size_t)(x_dtype == SB_BF16 ? 2 : 3) * M * sb::align8(I) * 2, 256);
}

extern "C" int sb_group4_gated_mlp(const void* x, int x_dtype, int64_t ldx, int64_t M, const sb_group4* gate,
                                   const sb_group4* up, const sb_group4* down, void* y, int y_dtype, void* workspace,
                                   size_t workspace_bytes, void* stream) {
  using namespace sb;
  int rc;
  if ((rc = check_group4_one(gate, "sb_group4_gated_mlp gate")) || (rc = check_group4_one(up, "sb_group4_gated_mlp up")) ||
      (rc = check_group4_one(down, "sb_group4_gated_mlp down")))
    return rc;
  const int64_t H = gate->K, I = gate->N;
  SB_REQUIRE(up->K == H && up->N == I && up->group == gate->group && !up->zeros == !gate->zeros,
             "sb_group4_gated_mlp: gate and up must have the same shape, group and kind of zero points");
  SB_REQUIRE(down->K == I && down->N == H, "sb_group4_gated_mlp: down must be [%lld, %lld], got [%lld, %lld]",
             (long long)H, (long long)I, (long long)down->N, (long long)down->K);
  if ((rc = check_few_x(x, x_dtype, ldx, M, H, "sb_group4_gated_mlp"))) return rc;
  SB_REQUIRE(y_dtype == SB_F32 || y_dtype == SB_BF16, "sb_group4_gated_mlp: y dtype must be SB_F32 or SB_BF16");
  if (M == 0) return SB_OK;
  SB_REQUIRE(y, "sb_group4_gated_mlp: y is null");
  if ((rc = check_workspace(workspace, workspace_bytes, sb_group4_gated_mlp_workspace_bytes(x_dtype, M, H, I))))
    return rc;
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  FewX fx;
  if ((rc = few_planes(x, x_dtype, ldx, M, H, workspace, &fx, st))) return rc;
  auto* h = reinterpret_cast<__nv_bfloat16*>(static_cast<uint8_t*>(workspace) + few_planes_bytes(x_dtype, M, H));
  if (long_mlp(x_dtype, M, H, I)) {
    const int64_t hp = align64(H), ip = align64(I);
    auto* wgu = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<uint8_t*>(h) + align_up((size_t)(M * ip * 4), 256));
    auto* wd = reinterpret_cast<__nv_bfloat16*>(reinterpret_cast<uint8_t*>(wgu) + align_up((size_t)(2 * I * hp * 4), 256));
    if ((rc = group4_terms(gate, hp, 2, 0, wgu, st)) || (rc = group4_terms(up, hp, 2, 1, wgu, st)) ||
        (rc = group4_terms(down, ip, 1, 0, wd, st)))
      return rc;
    const int hb = (int)(hp / 64), ib = (int)(ip / 64);
    if ((rc = group4_gemm("group4_gateup_tc", fx.base, fx.ld, H, M, wgu, hp, 2 * I, 2 * ip, 2 * hb,
                          EpiGroup4Hidden{h, ip, (int)I, hb}, st)))
      return rc;
    EpiGroup4Down epi;
    static_cast<EpiGroup4Rows&>(epi) = EpiGroup4Rows{nullptr, y, H, y_dtype, (int)H, ib};
    return group4_gemm("group4_down_tc", h, 2 * ip, 2 * ip, M, wd, ip, H, H, 3 * ib, epi, st);
  }
  const int64_t ldh = align8(I);
  const bool after = few_planes_needed(x, x_dtype, ldx, H);
  const FewHidden hidden{h, ldh, M * ldh};
  const FewX hx{h, ldh, M * ldh, (int)ldh};
  rc = with_group(gate->group, [&](auto g) {
    using W = Group4W<g.value>;
    const W wg = group4_weights<g.value>(gate), wu = group4_weights<g.value>(up);
    if (x_dtype == SB_BF16)
      return few_stream<W, true, 1, 2>("group4_gateup", wg, wu, fx, FewContiguous{(int)M}, M, I, hidden, FewRows{}, after,
                                       st);
    return few_stream<W, true, 3, 3>("group4_gateup", wg, wu, fx, FewContiguous{(int)M}, M, I, hidden, FewRows{}, after,
                                     st);
  });
  if (rc) return rc;
  return with_group(down->group, [&](auto g) {
    const auto wd = group4_weights<g.value>(down);
    if (x_dtype == SB_BF16) return few_linear<2>("group4_down", wd, hx, M, H, nullptr, y, y_dtype, true, st);
    return few_linear<3>("group4_down", wd, hx, M, H, nullptr, y, y_dtype, true, st);
  });
}
