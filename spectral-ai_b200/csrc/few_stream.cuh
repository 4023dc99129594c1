// few_stream.cuh — products of packed weights with a few tokens: the weights
// stream from memory through shared memory into registers, become
// matrix-instruction operands there and meet up to 8 * NT tokens.
//
//   acc[r, c] = sum_k value(r, k) * x_c[k]      16 weight rows r, 8 * NT tokens c
//
// With a few tokens such a product is a weight stream: 2 or 4 bits are read per
// weight and the arithmetic must keep up with HBM.  One thread per product is
// too slow for that (a decode and a multiply-add per weight and token), and a
// tcgen05 tile needs 128 rows in tensor memory, filled by a store and a
// hand-off between warps for every 64 columns, which a warp with 16 rows and no
// shared weight tile does not pay.  So a warp decodes 16 rows x 16 K straight into
// the A fragment of an m16n8k16 instruction and the tokens are its 8 columns:
// one instruction per 256 weights and 8 tokens, the same for 1 token as for 8.
//
// Fragment layout: lane (g = lane / 4, t = lane % 4) holds 4 K of rows g and
// g + 8 and 4 K of token g.  The sum does not care which K those are as long as
// weights and tokens agree, so each lane takes K that lie together in memory:
// 16 bytes per row and chunk, no shuffles.
//
//   4-bit groups: chunk of 128 K; lane t's 16 bytes hold the words i = 0..3, word i
//     the K  32 i + 8 t .. + 7  of the chunk, so that the four lanes together cover
//     32 K of ONE group at each word and the fp32 sums of a group are scaled once,
//     after its last word.
//   ternary: chunk of 256 K; lane t's words hold the K 64 t + 16 i .. + 15; the
//     row's scale is applied by the caller.
//
// Tokens are bf16 in T planes (x = sum of the planes): 1 for bf16 activations,
// 3 for fp32 ones (8 bits each: 24 bits, fp32's mantissa), 2 or 3 for the hidden
// state between two products.  Weights (2^-12 times code - zero, -15..15, or -1..1) and
// the planes are exact in bf16, products exact, sums fp32.
//
// What shaped it (B200, warm, per kernel of a 1-token layer; the cycles are those of
// the first version, before the change that the line names):
//  * Code that is run through once is fetched slower than it is executed: with the
//    chunk loop unrolled over 8 chunks held in registers a 1-token call spent most
//    of its time waiting for instructions.  The loop is one small body; weights in
//    flight live in a ring in shared memory.
//  * Sixteen-byte loads by lane touch 8 rows, 8 cache lines, each: issuing them took
//    1800 of a kernel's 5000 cycles.  4-bit weights lie in blocks of 16 rows x 128 K
//    with their scales and zero points, in lane order: one bulk copy each.
//  * Successive instructions into one accumulator wait for each other (a chunk of
//    one row tile and one column tile took 900 cycles): a tile's sums run in up to 4
//    accumulators.
//
// A block keeps its tokens in shared memory in the order in which the lanes read
// them (16-byte units; the four lanes of a row 64 bytes together, rows 64 bytes
// out of step, so that no two lanes of a load meet in a bank).  Columns past the
// last token read another token's values: a column's sums depend on nothing else.
#pragma once

#include "sm100.cuh"
#include "few_ring.cuh"
#include "gemm_tc.cuh"
#include "ternary_gemm.cuh"

namespace sb {

// (a & b) | c in one instruction
__device__ __forceinline__ uint32_t and_or(uint32_t a, uint32_t b, uint32_t c) {
  uint32_t d;
  asm("lop3.b32 %0, %1, %2, %3, 0xEA;" : "=r"(d) : "r"(a), "r"(b), "r"(c));
  return d;
}

__device__ __forceinline__ void mma_bf16(float (&d)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                         uint32_t b0, uint32_t b1, bool first) {
  if (first)  // (known at compile time: the sum starts here)
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%10,%10,%10,%10};"
        : "=f"(d[0]), "=f"(d[1]), "=f"(d[2]), "=f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1), "f"(0.f));
  else
    asm("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ uint32_t word_of(const uint4& v, int i) {
  return i == 0 ? v.x : i == 1 ? v.y : i == 2 ? v.z : v.w;
}

// Kernels follow each other without a gap: the next one of a call is launched early
// (`few_trigger`) and waits for this one's results where it needs them (`few_wait`;
// nothing to wait for returns at once).  The first kernel of a call waits before it
// triggers, so that whatever came before the call has ended when a later kernel of
// the call runs: weights, and a routing that was given, need no wait there.
__device__ __forceinline__ void few_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }
__device__ __forceinline__ void few_trigger() { asm volatile("griddepcontrol.launch_dependents;"); }

// 16 bytes global -> shared, asynchronously; `valid` false reads nothing and writes zeros
__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, bool valid) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(valid ? 16 : 0) : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;" ::: "memory"); }
// an arrival on `bar` when this thread's copies so far have landed
__device__ __forceinline__ void cp_async_arrive(uint64_t* bar) {
  asm volatile("cp.async.mbarrier.arrive.noinc.shared::cta.b64 [%0];" ::"r"(smem_u32(bar)) : "memory");
}
// `bytes` (a multiple of 16, both addresses 16-byte aligned) global -> shared, counted on `bar`
__device__ __forceinline__ void bulk_copy(uint32_t dst, const void* src, uint32_t bytes, uint64_t* bar) {
  asm volatile("cp.async.bulk.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1], %2, [%3];" ::"r"(dst),
               "l"(src), "r"(bytes), "r"(smem_u32(bar))
               : "memory");
}

__device__ __forceinline__ uint4 ld_shared16(uint32_t a) {
  uint4 v;
  asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t ld_shared4(uint32_t a) {
  uint32_t v;
  asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a));
  return v;
}
__device__ __forceinline__ uint32_t ld_shared2(uint32_t a) {
  uint16_t v;
  asm volatile("ld.shared.u16 %0, [%1];" : "=h"(v) : "r"(a));
  return v;
}

// The tokens in global memory: rows `ld` apart, planes `plane` apart (elements),
// 16-byte aligned rows, `K` valid elements, a multiple of 8 (the tail up to there
// is zero).
struct FewX {
  const __nv_bfloat16* base;
  int64_t ld, plane;
  int K;
};

// Bytes of one plane of one staged token.
__host__ __device__ __forceinline__ int few_row_bytes(int padded_k) { return padded_k * 2 + 64; }

// Stages `n` tokens (row(i) their rows) as [token][plane] rows of `chunks` chunks, a
// warp per row.
template <class W, int T, typename RowFn>
__device__ __forceinline__ void few_stage(uint32_t smem, const FewX& x, int n, int chunks, RowFn row) {
  const int units = chunks * (W::CHUNK / 8), bytes = few_row_bytes(chunks * W::CHUNK), have = x.K / 8;
  const int lane = threadIdx.x & 31;
  for (int j = threadIdx.x >> 5; j < n * T; j += blockDim.x >> 5) {
    const int i = T == 1 ? j : j / T, p = T == 1 ? 0 : j % T;
    const __nv_bfloat16* src = x.base + row(i) * x.ld + p * x.plane + lane * 8;
    const uint32_t dst = smem + j * bytes;
#pragma unroll 4
    for (int u = lane; u < units; u += 32, src += 256) cp_async16(dst + W::slot(u) * 16, u < have ? src : x.base, u < have);
  }
}

// A lane's view of the staged tokens: column n * 8 + g, its plane p at + p * bytes.
template <int T, int NT>
struct FewTokens {
  uint32_t at[NT];
  int bytes;
  __device__ __forceinline__ FewTokens(uint32_t smem, int n, int row_bytes, int g, int t) : bytes(row_bytes) {
#pragma unroll
    for (int i = 0; i < NT; ++i) at[i] = smem + (i * 8 + g < n ? (i * 8 + g) * T * row_bytes : 0) + t * 16;
  }
  // unit `slot4` (of four lanes' units) of column-tile n, plane p
  __device__ __forceinline__ uint4 get(int n, int p, int slot4) const {
    return ld_shared16(at[n] + p * bytes + slot4 * 64);
  }
};

// Accumulators per row tile and column tile: enough that RT x LIVE of them make four
// chains.  fp32 tokens (three planes) have the last one for their two low planes: the
// matrix instruction truncates its sum, and the low products, 2^-8 of the high ones,
// would truncate the high sum twice more per K block.
template <int LIVE, int RT, int T>
struct FewChains {
  static constexpr int SPREAD = RT * LIVE >= 4 ? 1 : RT * LIVE >= 2 ? 2 : 4;
  static constexpr int COUNT = T == 3 ? (SPREAD > 1 ? SPREAD : 2) : SPREAD;
  // the chain of product `half` (of `halves`) of plane p in K block i, and whether it is its first
  static __device__ __forceinline__ constexpr int of(int i, int p, int half, int halves) {
    return T == 3 ? (p ? COUNT - 1 : (i * halves + half) % (COUNT - 1)) : ((i * T + p) * halves + half) % COUNT;
  }
  static __device__ __forceinline__ constexpr bool first(int i, int p, int half, int halves) {
    return T == 3 ? (p ? i == 0 && p == 1 && half == 0 : i * halves + half < COUNT - 1)
                  : (i * T + p) * halves + half < COUNT;
  }
  // whether `products` products of a plane reach chain c at all
  static __device__ __forceinline__ constexpr bool used(int c, int products) {
    return T == 3 ? c == COUNT - 1 || c < products : c < products * T;
  }
};

// ---------------------------------------------------------------------------
// 4-bit weights in groups
// ---------------------------------------------------------------------------
// Blocks of 16 rows x 128 K, [matrix][row tile][chunk]: 1024 bytes of words (rows
// g, then rows g + 8: 16 bytes a lane), then for each of the chunk's 128 / G groups
// the 16 rows' scales (bf16), then their zero points (if any), rows g and g + 8
// side by side.
template <int G>
struct Group4W {
  static constexpr int CHUNK = 128;
  static constexpr bool ROW_SCALES = false;
  static constexpr bool BULK = true;     // rings are filled by bulk copies
  static constexpr int ARRIVALS = 1;     // on a ring slot's barrier
  static constexpr int PER = 128 / G;    // groups per chunk
  static constexpr int BLOCKS = G / 32;  // 32-K blocks per group
  static constexpr int SLOT = 1024 + 48 * PER;  // shared memory of a block
  // Sums are in units of 2^12: weights enter as 2^-12 (code - zero), so that a group's sum
  // before its scale, up to 15 x 128 tokens' values, overflows for no finite ones.
  static constexpr float UNIT = 4096.f;
  const uint8_t* data;
  int chunks, tiles;  // per matrix: chunks of a row, row tiles
  int block;          // bytes of a block: 1024 + 32 PER, with zero points 1024 + 48 PER

  static __device__ __forceinline__ int slot(int u) { return u; }

  // row tile `tile` of matrix e
  struct Tile {
    const uint8_t* p;
  };
  __device__ __forceinline__ Tile tile(int e, int tile, int, int) const {
    return Tile{data + ((int64_t)e * tiles + tile) * chunks * block};
  }
  // chunk c of RT row tiles on its way to a ring slot; the whole warp calls it
  template <int RT>
  __device__ __forceinline__ void fetch(uint32_t dst, uint64_t* bar, const Tile (&t)[RT], int c, int lane) const {
    if (lane == 0) {
      mbar_arrive_expect_tx(bar, RT * block);
#pragma unroll
      for (int r = 0; r < RT; ++r) bulk_copy(dst + r * SLOT, t[r].p + (int64_t)c * block, block, bar);
    }
  }

  // Pair j of a word (elements 2j, 2j + 1 in its halves) minus the zero point, over UNIT:
  // OR-ing 2^-5's exponent over the code gives 2^-12 (128 + code), exact in bf16, and
  // `sub` holds 2^-12 (128 + zero) twice.
  static __device__ __forceinline__ uint32_t pair(uint32_t w, int j, uint32_t sub) {
    const uint32_t v = and_or(w >> (4 * j), 0x000F000Fu, 0x3D003D00u);
    const __nv_bfloat162 d =
        __hsub2(*reinterpret_cast<const __nv_bfloat162*>(&v), *reinterpret_cast<const __nv_bfloat162*>(&sub));
    return *reinterpret_cast<const uint32_t*>(&d);
  }

  // a lane's share of a ring slot: words, scales and zero points of rows g and g + 8
  template <int RT>
  struct Part {
    uint4 w[RT][2];
    uint32_t s[RT][PER], z[RT][PER];
  };
  template <int RT>
  __device__ __forceinline__ void read(Part<RT>& p, uint32_t slot, int lane) const {
    const bool zeros = block == SLOT;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      p.w[r][0] = ld_shared16(slot + r * SLOT + lane * 16);
      p.w[r][1] = ld_shared16(slot + r * SLOT + 512 + lane * 16);
#pragma unroll
      for (int q = 0; q < PER; ++q) {
        p.s[r][q] = ld_shared4(slot + r * SLOT + 1024 + (lane >> 2) * 4 + q * 32);
        p.z[r][q] = zeros ? ld_shared2(slot + r * SLOT + 1024 + 32 * PER + q * 16 + (lane >> 2) * 2) : 0x0808u;
      }
    }
  }

  // acc += (chunk c) x (the first LIVE column tiles)
  template <int LIVE, int RT, int T, int NT>
  __device__ __forceinline__ void chunk(const Part<RT>& part, int c, const FewTokens<T, NT>& x,
                                        float (&acc)[RT][NT][4]) const {
    using Chains = FewChains<LIVE, RT, T>;
#pragma unroll
    for (int q = 0; q < PER; ++q) {
      float raw[RT][LIVE][Chains::COUNT][4];
      uint32_t sub[RT][2];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        sub[r][0] = __byte_perm(part.z[r][q], 0x3Du, 0x4040u);  // bytes z, 0x3D, z, 0x3D
        sub[r][1] = __byte_perm(part.z[r][q], 0x3Du, 0x4141u);
      }
#pragma unroll
      for (int i = 0; i < BLOCKS; ++i) {
        uint32_t a[RT][8];
#pragma unroll
        for (int r = 0; r < RT; ++r) {
          const uint32_t wa = word_of(part.w[r][0], q * BLOCKS + i), wb = word_of(part.w[r][1], q * BLOCKS + i);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            a[r][2 * j] = pair(wa, j, sub[r][0]);
            a[r][2 * j + 1] = pair(wb, j, sub[r][1]);
          }
        }
#pragma unroll
        for (int n = 0; n < LIVE; ++n) {
#pragma unroll
          for (int p = 0; p < T; ++p) {
            const uint4 v = x.get(n, p, c * 4 + q * BLOCKS + i);
#pragma unroll
            for (int r = 0; r < RT; ++r) {
              mma_bf16(raw[r][n][Chains::of(i, p, 0, 2)], a[r][0], a[r][1], a[r][2], a[r][3], v.x, v.y,
                       Chains::first(i, p, 0, 2));
              mma_bf16(raw[r][n][Chains::of(i, p, 1, 2)], a[r][4], a[r][5], a[r][6], a[r][7], v.z, v.w,
                       Chains::first(i, p, 1, 2));
            }
          }
        }
      }
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        const float sa = __uint_as_float(part.s[r][q] << 16), sb = __uint_as_float(part.s[r][q] & 0xFFFF0000u);
#pragma unroll
        for (int n = 0; n < LIVE; ++n) {
#pragma unroll
          for (int k = 0; k < 4; ++k) {
            float v = raw[r][n][0][k];
#pragma unroll
            for (int s = 1; s < Chains::COUNT; ++s)
              if (Chains::used(s, BLOCKS * 2)) v += raw[r][n][s][k];
            acc[r][n][k] = fmaf(k < 2 ? sa : sb, v, acc[r][n][k]);
          }
        }
      }
    }
  }
};

// ---------------------------------------------------------------------------
// ternary weights
// ---------------------------------------------------------------------------
// Rows of `blocks` 16-byte blocks (64 K each) and one fp32 scale per row; N rows per
// matrix.  The rows keep the layout of the tile kernels (ternary.cu), so a chunk is
// copied 16 bytes a lane, each lane reading back what it copied itself.
struct TernaryW {
  static constexpr int CHUNK = 256;
  static constexpr bool ROW_SCALES = true;
  static constexpr bool BULK = false;
  static constexpr int ARRIVALS = 32;
  static constexpr int SLOT = 1024;
  static constexpr float UNIT = 1.f;  // of the sums
  const uint32_t* words;
  const float* scales;
  int chunks, blocks;

  // unit 8t + 2i + v of a chunk (lane t's word i, half v) among its four lanes' units
  static __device__ __forceinline__ int slot(int u) { return (u & ~31) | ((u & 7) << 2) | ((u >> 3) & 3); }

  struct Tile {
    const uint32_t *a, *b;  // the lane's rows g and g + 8; past the matrix: its last one
  };
  __device__ __forceinline__ Tile tile(int e, int tile, int N, int lane) const {
    const int g = lane >> 2, r0 = tile * 16;
    const uint32_t* p = words + (((int64_t)e * N + r0) * blocks + (lane & 3)) * 4;
    return Tile{p + (uint32_t)(min(g, N - 1 - r0) * blocks) * 4u, p + (uint32_t)(min(g + 8, N - 1 - r0) * blocks) * 4u};
  }
  // a block past the row's end has no words: zeros, its tokens' values are zero
  template <int RT>
  __device__ __forceinline__ void fetch(uint32_t dst, uint64_t* bar, const Tile (&t)[RT], int c, int lane) const {
    const bool in = c * 4 + (lane & 3) < blocks;
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      cp_async16(dst + r * SLOT + lane * 16, t[r].a + c * 16, in);
      cp_async16(dst + r * SLOT + 512 + lane * 16, t[r].b + c * 16, in);
    }
    cp_async_arrive(bar);
  }

  template <int RT>
  struct Part {
    uint4 w[RT][2];
  };
  template <int RT>
  __device__ __forceinline__ void read(Part<RT>& p, uint32_t slot, int lane) const {
#pragma unroll
    for (int r = 0; r < RT; ++r) {
      p.w[r][0] = ld_shared16(slot + r * SLOT + lane * 16);
      p.w[r][1] = ld_shared16(slot + r * SLOT + 512 + lane * 16);
    }
  }

  template <int LIVE, int RT, int T, int NT>
  __device__ __forceinline__ void chunk(const Part<RT>& part, int c, const FewTokens<T, NT>& x,
                                        float (&acc)[RT][NT][4]) const {
    // sums of 256 K, added up in fp32: the matrix instruction's own accumulation
    // rounds towards zero, which stays small over 16 of its steps
    using Chains = FewChains<LIVE, RT, T>;
    float raw[RT][LIVE][Chains::COUNT][4];
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      uint32_t a[RT][8], b[RT][8];
#pragma unroll
      for (int r = 0; r < RT; ++r) {
        tern_word<1>(word_of(part.w[r][0], i), a[r]);
        tern_word<1>(word_of(part.w[r][1], i), b[r]);
      }
#pragma unroll
      for (int n = 0; n < LIVE; ++n) {
#pragma unroll
        for (int p = 0; p < T; ++p) {
          const uint4 v = x.get(n, p, c * 8 + i * 2), u = x.get(n, p, c * 8 + i * 2 + 1);
#pragma unroll
          for (int r = 0; r < RT; ++r) {
#pragma unroll
            for (int j = 0; j < 4; ++j)
              mma_bf16(raw[r][n][Chains::of(i, p, j, 4)], a[r][2 * j], b[r][2 * j], a[r][2 * j + 1], b[r][2 * j + 1],
                       j == 0 ? v.x : j == 1 ? v.z : j == 2 ? u.x : u.z, j == 0 ? v.y : j == 1 ? v.w : j == 2 ? u.y : u.w,
                       Chains::first(i, p, j, 4));
          }
        }
      }
    }
#pragma unroll
    for (int r = 0; r < RT; ++r)
#pragma unroll
      for (int n = 0; n < LIVE; ++n)
#pragma unroll
        for (int k = 0; k < 4; ++k)
#pragma unroll
          for (int s = 0; s < Chains::COUNT; ++s) acc[r][n][k] += raw[r][n][s][k];
  }
  __device__ __forceinline__ float out_scale(int64_t r) const { return __ldg(scales + r); }
};

// Waits for the next slot of a warp's ring.  Where the wait runs out (and is reported), the
// copies on their way, one for each slot at most and in the slots' order, get the same time
// once more, so that none lands in shared memory that the block has left.  (A call: as part
// of the kernels' own code it takes registers from the chunks' arithmetic, 97.4 us for
// 64 tokens over 4-bit experts against 96.1; without it 94.9.)
__device__ __noinline__ bool few_ring_wait(uint64_t* bars, FewSlots slots) {
  if (mbar_wait_warp(bars + slots.out, slots.parity, ST_TIMEOUT_PRODUCER)) return true;
  const uint64_t t0 = globaltimer();
#pragma unroll 1
  for (int i = 0; i < slots.depth; ++i) {
    uint32_t phase;
    const uint32_t bar = smem_u32(bars + slots.ahead(i, &phase));
    while (!mbar_test_wait(bar, phase) && globaltimer() - t0 <= SB_WAIT_LIMIT_NS) __nanosleep(1000);
  }
  return false;
}

// A warp's ring: `depth` slots of RT blocks and a barrier each, filled and used in turn.
template <class W, int RT>
struct FewRing {
  uint32_t base;
  uint64_t* bars;
  FewSlots slots;
  bool lost;  // a wait ran out: no more waits, no more copies
  static __host__ __device__ constexpr int slot_bytes() { return RT * W::SLOT; }

  __device__ __forceinline__ FewRing(uint8_t* smem, uint64_t* bars_, int warp, int depth)
      : base(smem_u32(smem) + warp * depth * slot_bytes()), bars(bars_ + warp * depth), slots(depth), lost(false) {}
  __device__ __forceinline__ void fetch(int slot, const W& w, const typename W::Tile (&t)[RT], int c, int lane) {
    if (!lost) w.template fetch<RT>(base + slot * slot_bytes(), bars + slot, t, c, lane);
  }
  // reads the next slot once it has been filled; returns it, free to be filled again
  __device__ __forceinline__ int take(const W& w, typename W::template Part<RT>& p, int lane) {
    if (!__all_sync(0xffffffffu, mbar_test_wait(smem_u32(bars + slots.out), slots.parity)) && !lost)
      lost = !few_ring_wait(bars, slots);
    const int slot = slots.out;
    w.read(p, base + slot * slot_bytes(), lane);
    __syncwarp();
    slots.taken();
    return slot;
  }
};

// The barriers of a block's rings, `n` of them, ready for use after the next barrier.
template <class W>
__device__ __forceinline__ void few_bars_init(uint64_t* bars, int n) {
  for (int i = threadIdx.x; i < n; i += blockDim.x) mbar_init(bars + i, W::ARRIVALS);
  fence_barrier_init();
}

// v as planes: bf16(v), bf16 of what that leaves, and so on.  A finite v that bf16 would
// round to infinity (from 3.39e38 on) has its first plane rounded towards zero, which
// leaves the others no more than they hold; an infinite v is its first plane alone.
template <int T>
__device__ __forceinline__ void split_planes(float v, __nv_bfloat16 (&p)[T]) {
  p[0] = __float2bfloat16_rn(v);
  if (T > 1 && isinf(__bfloat162float(p[0]))) {
    if (isinf(v))
      v = 0.f;
    else
      v -= __bfloat162float(p[0] = __float2bfloat16_rz(v));
  } else {
    v -= __bfloat162float(p[0]);
  }
#pragma unroll
  for (int i = 1; i < T; ++i) {
    p[i] = __float2bfloat16_rn(v);
    v -= __bfloat162float(p[i]);
  }
}

// h = silu(gate) * up, as planes
template <int TH>
__device__ __forceinline__ void store_hidden(__nv_bfloat16* h, int64_t plane, float gate, float up) {
  __nv_bfloat16 p[TH];
  split_planes<TH>(gate / (1.f + expf(-gate)) * up, p);
#pragma unroll
  for (int i = 0; i < TH; ++i) h[i * plane] = p[i];
}

__device__ __forceinline__ void store_out(void* y, int dtype, int64_t at, float v) {
  if (dtype == SB_BF16)
    static_cast<__nv_bfloat16*>(y)[at] = __float2bfloat16_rn(v);
  else
    static_cast<float*>(y)[at] = v;
}

// ---------------------------------------------------------------------------
// the grouped stream
// ---------------------------------------------------------------------------
// Where a block's work comes from.  Group gi: `n` tokens of expert `e`, whose
// rows start at entry `first`; entry i's token is row(first + i) of x.  The blocks
// share out the groups' cost (cost() times a group's units and `start` more, what it costs
// a block to begin with it): locate() gives the first unit, `run` of group `gi`, that
// starts at or after a point of it.  (The host keeps groups x units below 2^26.)
struct FewGroup {
  int e, n, first;
};

// Contiguous tokens of one matrix, `tile` to a group.
struct FewContiguous {
  int M;
  struct View {
    int M, tile, count;
    __device__ __forceinline__ uint32_t cost() const { return (uint32_t)count; }
    __device__ __forceinline__ void locate(uint32_t at, int runs, int start, int* gi, int* run) const {
      *gi = (int)(at / (uint32_t)(runs + start));
      *run = max(0, (int)at - *gi * (runs + start) - start);
    }
    __device__ __forceinline__ FewGroup group(int gi) const { return FewGroup{0, min(tile, M - gi * tile), gi * tile}; }
    __device__ __forceinline__ int row(int entry) const { return entry; }
  };
  size_t bytes() const { return 0; }
  bool waits() const { return false; }
  int64_t groups(int tile) const { return (M + (int64_t)tile - 1) / tile; }
  template <int T>
  __device__ __forceinline__ View view(uint8_t*, int tile, int most) const { return View{M, tile, most}; }
};

// What becomes of the sums: hidden rows (gate and up) or output rows.
struct FewHidden {
  __nv_bfloat16* h;   // [plane][entry][ld]
  int64_t ld, plane;  // ld: I rounded up to 8
};
struct FewRows {
  void* y;  // [entry][N]
  int dtype;
  const float* bias;
};

struct FewShape {
  int N;            // rows (channels) of an expert
  int tile_tokens;  // tokens of a group at most
  int tiles;        // units of an expert
  int groups;       // at most
  int tokens_last;  // the first weights are asked for before the first tokens, which may be late
  int start;        // units that beginning with a group costs a block
  int depth;        // slots of a warp's ring
  int early;        // weights and routing may be read before the kernel before this one has ended
};

// A warp's share of the units [0, n) of `chunks` chunks each that a block has of a
// group, cut evenly among the warps chunk by chunk.  It begins inside unit `head`, has
// whole units and ends inside unit `tail` (-1: at a unit's border).  The parts run in
// the order tail, whole units, head: the tail's sums are left in shared memory for the
// warp that has the end of that unit, which adds them to its own, the head's.
template <int WARPS>
struct FewSpan {
  int tail, tail_lo, tail_hi, whole, whole_end, head, head_lo;
  // a warp's first chunk of the n * chunks
  static __device__ __forceinline__ int from(int n, int chunks, int warp) {
    return (int)((uint32_t)(n * chunks * warp) / WARPS);
  }
  __device__ __forceinline__ FewSpan(int n, int chunks, int warp) {
    const int a = from(n, chunks, warp), b = from(n, chunks, warp + 1);
    const int au = (int)((uint32_t)a / (uint32_t)chunks), ac = a - au * chunks;
    const int bu = b - au * chunks < chunks ? au : (int)((uint32_t)b / (uint32_t)chunks), bc = b - bu * chunks;
    tail = a < b && bc ? bu : -1;
    tail_lo = au == bu ? ac : 0;
    tail_hi = bc;
    whole = au + (ac ? 1 : 0);
    whole_end = bu;
    head = ac && au < bu ? au : -1;
    head_lo = ac;
  }
  // part p: its unit and chunks; false: there are no more
  __device__ __forceinline__ bool part(int p, int chunks, int* unit, int* lo, int* hi) const {
    if (tail >= 0) {
      if (p == 0) {
        *unit = tail;
        *lo = tail_lo;
        *hi = tail_hi;
        return true;
      }
      --p;
    }
    *lo = 0;
    *hi = chunks;
    *unit = whole + p;
    if (*unit < whole_end) return true;
    if (head >= 0 && p == max(0, whole_end - whole)) {
      *unit = head;
      *lo = head_lo;
      return true;
    }
    return false;
  }
};

// A persistent block takes a run of units, a unit being RT row tiles of one group, a
// group's units at a time; its warps share them out evenly (FewSpan).  Units of a group
// share its staged tokens; every warp's ring runs ahead of it through its parts and
// groups, so the first weights are on their way before the tokens are waited for.  Tokens
// that are there already are asked for before the first weights, whose bulk copies take
// longer to set out (64 tokens over 4-bit experts 95.5 us against 97.0, MLP at 300 31.4
// against 32.2; ternary rings, filled by the lanes' own copies, lose by it: 87.6 against 86.0).
//
// GATEUP: the unit's two row tiles are a tile of the gate and the same tile of the
// up matrix, so that a lane holds both halves of its channels (N counts channels).
//
// Up to 8 tokens a group: one column tile, and two blocks of 8 warps an SM where both
// fit, so that one works while the other stages tokens or waits at a barrier; else one
// block of 16.  Above 8: two column tiles, and units of two row tiles that share the
// token fragments; the staged tokens leave room for one block of 16 warps.  (Two blocks
// of 8 with 12 tokens a group: 24 tokens of a ternary layer 86 us against 91, but 64 of a
// 4-bit one 103.5 against 100.7 and [4096 x 2048] at 32 tokens 10.6 against 8.8.  Four
// column tiles leave registers for 8 warps, too few to hide a chunk's latency: [4096 x
// 2048] at 128 tokens 18.5 us against 15.3 for two, which decode the weights twice as
// often; both with whole units to the warps.)
//
// Shared memory: [tile_tokens][T] staged rows | the warps' rings | their tails' sums |
// the rings' barriers | the work's lists.
template <class W, bool GATEUP, int T, int TH, int NT, int RT, int WARPS, class Work>
__global__ void __launch_bounds__(WARPS * 32, 16 / WARPS)
    few_stream_kernel(W w0, W w1, FewX x, Work work, FewShape sh, FewHidden hidden, FewRows rows) {
  extern __shared__ __align__(128) uint8_t few_smem[];
  static_assert(!GATEUP || RT == 2, "a gate tile and an up tile");
  constexpr int UT = GATEUP ? 1 : RT;  // row tiles of a matrix in a unit
  using Ring = FewRing<W, RT>;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int chunks = w0.chunks, row_bytes = few_row_bytes(chunks * W::CHUNK), N = sh.N;
  const uint32_t sx = smem_u32(few_smem);
  if (!sh.early) few_wait();
  uint8_t* rings = few_smem + (size_t)sh.tile_tokens * T * row_bytes;
  float* sums = reinterpret_cast<float*>(rings + WARPS * sh.depth * Ring::slot_bytes());  // [warp][RT * NT * 4][32]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sums + WARPS * RT * NT * 128);
  few_bars_init<W>(bars, WARPS * sh.depth);
  const auto view = work.template view<T>(reinterpret_cast<uint8_t*>(bars + WARPS * sh.depth), sh.tile_tokens, sh.groups);
  few_trigger();
  __syncthreads();
  const uint32_t cost = view.cost() * (uint32_t)(sh.tiles + sh.start), each = cost / gridDim.x, rest = cost - each * gridDim.x;
  const uint32_t p0 = each * blockIdx.x + min(blockIdx.x, rest), p1 = p0 + each + (blockIdx.x < rest ? 1u : 0u);
  int gi, first_unit, end_gi, end_unit;
  view.locate(p0, sh.tiles, sh.start, &gi, &first_unit);
  view.locate(p1, sh.tiles, sh.start, &end_gi, &end_unit);
  // this block's units of a group: [units_from(i), units_to(i))
  const int gi0 = gi, last_gi = end_unit ? end_gi : end_gi - 1;
  auto units_from = [&](int i) { return i == gi0 ? first_unit : 0; };
  auto units_to = [&](int i) { return i == end_gi ? end_unit : sh.tiles; };
  if (gi > last_gi) {
    few_wait();  // no kernel ends before the one it followed
    return;
  }

  // the ring's front: chunk fc (to fhi) of part fp of group fg
  Ring ring(rings, bars, warp, sh.depth);
  typename W::Tile front[RT];
  FewSpan<WARPS> span(units_to(gi) - units_from(gi), chunks, warp), fspan = span;
  int fg = gi, fp = 0, fc = 0, fhi = 0;
  auto ahead = [&](int slot) {
    if (fc == fhi) {
      int unit;
      while (fg <= last_gi && !fspan.part(fp, chunks, &unit, &fc, &fhi)) {
        fp = 0;
        if (++fg <= last_gi) fspan = FewSpan<WARPS>(units_to(fg) - units_from(fg), chunks, warp);
      }
      if (fg > last_gi) {
        fc = fhi = 0;
        return;
      }
      ++fp;
      const int e = view.group(fg).e, tile = (units_from(fg) + unit) * UT;
      if constexpr (GATEUP) {
        front[0] = w0.tile(e, tile, N, lane);
        front[1] = w1.tile(e, tile, N, lane);
      } else {
#pragma unroll
        for (int r = 0; r < RT; ++r) front[r] = w0.tile(e, min(tile + r, (N - 1) >> 4), N, lane);
      }
    }
    ring.fetch(slot, w0, front, fc++, lane);
  };
  auto fill = [&] {
#pragma unroll 1
    for (int d = 0; d < sh.depth; ++d) ahead(d);
  };
  if constexpr (!W::BULK) fill();

  float acc[RT][NT][4];
  for (; gi <= last_gi; ++gi) {
    const FewGroup grp = view.group(gi);
    __syncthreads();  // the last group's tokens and sums have been read
    auto stage = [&] {
      few_wait();
      few_stage<W, T>(sx, x, grp.n, chunks, [&](int i) { return view.row(grp.first + i); });
    };
    if constexpr (W::BULK) {
#pragma unroll 1
      for (int s = 0; s < 2; ++s) {  // (in a loop: each once in the code)
        if (s == sh.tokens_last)
          stage();
        else if (gi == gi0)
          fill();
      }
    } else {
      stage();
    }
    cp_async_wait_all();
    __syncthreads();
    const FewTokens<T, NT> tok(sx, grp.n, row_bytes, g, t);
    const int u0 = units_from(gi), n = units_to(gi) - u0;
    if (gi != gi0) span = FewSpan<WARPS>(n, chunks, warp);

    auto finish = [&](int unit) {  // the whole sums of a unit are in acc
      const int c0 = (u0 + unit) * UT * 16;
#pragma unroll
      for (int i = 0; i < NT; ++i) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
          const int col = i * 8 + 2 * t + q;
          if (col >= grp.n) continue;
          const int64_t line = (int64_t)(grp.first + col) * (GATEUP ? hidden.ld : N), base = (int64_t)grp.e * N;
#pragma unroll
          for (int r = 0; r < UT * 2; ++r) {  // the lane's rows c0 + g + 8 r
            const int ch = c0 + g + 8 * r, at = min(ch, N - 1);
            float a = acc[GATEUP ? 0 : r / 2][i][q + (r & 1) * 2] * W::UNIT;
            if constexpr (W::ROW_SCALES) a *= w0.out_scale(base + at);
            if constexpr (GATEUP) {
              float b = acc[1][i][q + (r & 1) * 2] * W::UNIT;
              if constexpr (W::ROW_SCALES) b *= w1.out_scale(base + at);
              if (ch < hidden.ld)  // columns N .. ld: zero
                store_hidden<TH>(hidden.h + line + ch, hidden.plane, ch < N ? a : 0.f, ch < N ? b : 0.f);
            } else {
              if (ch < N) store_out(rows.y, rows.dtype, line + ch, rows.bias ? a + __ldg(rows.bias + ch) : a);
            }
          }
        }
      }
    };

    int unit = 0, lo, hi;
#pragma unroll 1
    for (int p = 0; span.part(p, chunks, &unit, &lo, &hi); ++p) {
#pragma unroll
      for (int r = 0; r < RT; ++r)
#pragma unroll
        for (int i = 0; i < NT; ++i) acc[r][i][0] = acc[r][i][1] = acc[r][i][2] = acc[r][i][3] = 0.f;
      typename W::template Part<RT> part;
      auto run_chunks = [&](auto live) {
        [[maybe_unused]] int slot = 0;
        if constexpr (NT == 1) slot = ring.take(w0, part, lane);
#pragma unroll 1
        for (int c = lo; c < hi; ++c) {
          if constexpr (NT == 1) {  // read a chunk ahead of the arithmetic
            const typename W::template Part<RT> now = part;
            const int used = slot;
            if (c + 1 < hi) slot = ring.take(w0, part, lane);
            ahead(used);
            w0.template chunk<1>(now, c, tok, acc);
          } else {
            ahead(ring.take(w0, part, lane));
            w0.template chunk<decltype(live)::value>(part, c, tok, acc);
          }
        }
      };
      if (NT > 1 && grp.n > 8)
        run_chunks(std::integral_constant<int, NT>{});
      else
        run_chunks(std::integral_constant<int, 1>{});
      if (unit == span.tail) {
        float* mine = sums + warp * RT * NT * 128 + lane;
#pragma unroll
        for (int i = 0; i < RT * NT * 4; ++i) mine[i * 32] = acc[i / (NT * 4)][i / 4 % NT][i % 4];
      } else if (unit != span.head) {
        finish(unit);
      }
    }
    __syncthreads();
    if (span.head >= 0) {  // the warps before this one that ended in its first unit, in order
      for (int v = 0; v < warp; ++v) {
        const int a = FewSpan<WARPS>::from(n, chunks, v), b = FewSpan<WARPS>::from(n, chunks, v + 1);
        if (a < b && b > span.head * chunks) {
          const float* theirs = sums + v * RT * NT * 128 + lane;
#pragma unroll
          for (int i = 0; i < RT * NT * 4; ++i) acc[i / (NT * 4)][i / 4 % NT][i % 4] += theirs[i * 32];
        }
      }
      finish(span.head);
    }
  }
}

}  // namespace sb
