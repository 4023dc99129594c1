// moe_few.cu — a whole mixture-of-experts layer for a few tokens:
//
//   logits[t, e] = x[t] . Wg[e]              (optional: the routing may be given)
//   p = softmax(logits), ids = the k largest, w = p[ids] (or divided by their sum)
//   out[t] = sum_j w[t, j] * down_e(silu(gate_e x[t]) * (up_e x[t])),  e = ids[t, j]
//
// over ternary experts or experts in 4-bit groups.  The grouped layer of
// ternary.cu is built for thousands of tokens: it plans in one kernel, copies
// every token once per expert, runs 256-channel tiles and adds the slots'
// outputs in another kernel.  For a few tokens the layer is the stream of the
// touched experts' weights (few_stream.cuh), and what costs is everything around
// it: launches, copies, intermediate rows.  Here:
//
//   moe_few_logits  the gate's scores
//   moe_few_topk    softmax and top k, a warp per token; up to 2 tokens the kernels
//                   below do it for themselves instead
//   moe_few_gateup  every block groups the entries by expert for itself (cheaper
//                   than a launch and a wait), streams gate and up rows, writes the
//                   hidden rows
//   moe_few_sum     a block owns 16 output channels, stages every hidden row and adds
//                   all experts' shares of its channels
//   moe_few_down, moe_few_combine
//                   (where the hidden rows do not fit in one block) the down products
//                   by expert, then each token's sum
//
// An entry is one (expert, token): a token that names an expert twice has its
// weights added.  Ids outside [0, E) are dropped and reported.  The order of every
// sum is set by the shapes and the routing alone.
#include "common.cuh"
#include "few_stream.cuh"

namespace sb {

constexpr int FEW_MAX_ENTRIES = 2048;  // tokens x k
constexpr int FEW_MAX_TOKENS = 256;
constexpr int FEW_MAX_EXPERTS = 512;
constexpr int FEW_MAX_TOPK = 32;
constexpr int64_t FEW_MAX_WIDTH = 8192;  // H and I: a staged fp32 token (48 KB) beside the longest lists (60 KB) and the rings

// ---------------------------------------------------------------------------
// gate
// ---------------------------------------------------------------------------
constexpr int GATE_TOKENS = 2;    // tokens per block (4: 0.2 us slower at 1 token, 1.8 at 4, 0.6 at 64, 1.2 faster at 256)
constexpr int GATE_WARPS = 16;
// Tokens up to which every block picks the experts itself.  64 experts, top 8, the whole
// layer, own against a kernel's: 22.5 / 23.1 us at 1 token, 32.9 / 33.4 at 2, 45.6 / 45.2 at
// 3, 53.0 / 52.2 at 4 (more warps reach the picking's code at once).
constexpr int FEW_OWN_TOPK = 2;

// Eight neighbouring values as fp32; `n` of them exist, `vec`: aligned to be loaded together.
template <typename TX>
__device__ __forceinline__ void load8(const TX* p, int n, bool vec, float (&v)[8]) {
  if (vec && n >= 8) {
    if constexpr (std::is_same<TX, float>::value) {
      const float4 a = __ldg(reinterpret_cast<const float4*>(p)), b = __ldg(reinterpret_cast<const float4*>(p) + 1);
      v[0] = a.x, v[1] = a.y, v[2] = a.z, v[3] = a.w, v[4] = b.x, v[5] = b.y, v[6] = b.z, v[7] = b.w;
    } else {
      const uint4 u = __ldg(reinterpret_cast<const uint4*>(p));
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        v[2 * i] = __uint_as_float(word_of(u, i) << 16);
        v[2 * i + 1] = __uint_as_float(word_of(u, i) & 0xFFFF0000u);
      }
    }
  } else {
#pragma unroll
    for (int i = 0; i < 8; ++i) v[i] = i < n ? (float)p[i] : 0.f;
  }
}

// A float's place in ascending order as an unsigned number; -0 as 0, NaN as -inf.
__device__ __forceinline__ uint32_t order_of(float v) {
  const uint32_t u = __float_as_uint(v != v ? -INFINITY : v + 0.f);
  return (u >> 31) ? ~u : (u | 0x80000000u);
}

// Softmax of a token's logits and its k largest by one warp, V of them to a lane:
// lower index first among equals, NaN ranked as -inf (its softmax is NaN, and so are
// all the token's weights).
template <int V>
__device__ __forceinline__ void warp_topk(const float* lg, int E, int k, bool norm, int lane, int* ids, float* w) {
  float v[V];
  uint32_t key[V];  // 0: no expert, or taken
  bool nan = false;
  uint32_t best = 0;
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int e = lane + 32 * i;
    v[i] = e < E ? __ldcg(lg + e) : -INFINITY;
    nan |= v[i] != v[i];
    key[i] = e < E ? order_of(v[i]) : 0u;
    best = max(best, key[i]);
  }
  float m = 0.f, sum = 0.f, mine = 0.f, picked = 0.f;
  int my_id = 0;
#pragma unroll 1
  for (int j = 0; j < k; ++j) {
    const uint32_t top = __reduce_max_sync(0xffffffffu, best);
    const float value = __uint_as_float((top >> 31) ? top & 0x7FFFFFFFu : ~top);
    if (j == 0) {  // the largest: the softmax's sum
      m = value;
#pragma unroll
      for (int i = 0; i < V; ++i) sum += lane + 32 * i < E ? expf(v[i] - m) : 0.f;
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, o);
      if (__any_sync(0xffffffffu, nan)) sum = NAN;
    }
    int at = -1;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const unsigned has = __ballot_sync(0xffffffffu, key[i] == top);
      if (at < 0 && has) at = 32 * i + __ffs(has) - 1;
    }
    best = 0;
#pragma unroll
    for (int i = 0; i < V; ++i) {
      if (at == lane + 32 * i) key[i] = 0;
      best = max(best, key[i]);
    }
    const float p = expf(value - m) / sum;
    picked += p;
    if (j == lane) {
      mine = p;
      my_id = at;
    }
  }
  if (lane < k) {
    ids[lane] = my_id;
    w[lane] = norm ? mine / picked : mine;
  }
}

__device__ __forceinline__ void few_topk(const float* lg, int E, int k, bool norm, int lane, int* ids, float* w) {
  if (E <= 64)
    warp_topk<2>(lg, E, k, norm, lane, ids, w);
  else
    warp_topk<FEW_MAX_EXPERTS / 32>(lg, E, k, norm, lane, ids, w);
}

__global__ void __launch_bounds__(256) moe_few_topk_kernel(const float* logits, int B, int E, int k, int norm,
                                                           int32_t* ids, float* weights) {
  few_wait();
  few_trigger();
  const int t = blockIdx.x * 8 + (threadIdx.x >> 5), lane = threadIdx.x & 31;
  if (t < B)
    few_topk(logits + (int64_t)t * E, E, k, norm != 0, lane, ids + (int64_t)t * k, weights + (int64_t)t * k);
}

// a sum in two floats, s + c: about 48 bits
struct Sum2 {
  float s = 0.f, c = 0.f;
  // adds p + e exactly to s, what that rounds off to c
  __device__ __forceinline__ void add(float p, float e) {
    const float n = __fadd_rn(s, p), v = __fsub_rn(n, s);  // (never fused with the product)
    c += __fadd_rn(__fsub_rn(s, __fsub_rn(n, v)), __fsub_rn(p, v)) + e;
    s = n;
  }
  __device__ __forceinline__ float value() const { return isfinite(s) ? s + c : s; }
};

// The sums run in two floats and are rounded once, so that the order of two experts
// is that of their real logits, however the sum is cut (an fp32 sum's error is of
// the size of the gaps that a large batch shows).  A block has 16 / wpe experts, each
// with wpe warps over K, and 2 tokens; its loops stay rolled (see few_stream.cuh).
template <typename TX, typename TG>
__global__ void __launch_bounds__(GATE_WARPS * 32)
    moe_few_logits_kernel(const TX* __restrict__ x, int64_t ldx, int B, int H, int E, const TG* __restrict__ wg, bool vecx,
                          bool vecg, int wpe, float* __restrict__ logits) {
  constexpr bool SPLIT = std::is_same<TX, float>::value || std::is_same<TG, float>::value;  // products round
  __shared__ float2 part[GATE_TOKENS][GATE_WARPS];
  few_wait();
  few_trigger();
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const int t0 = blockIdx.y * GATE_TOKENS, nt = min(GATE_TOKENS, B - t0);
  const int per = GATE_WARPS / wpe, e0 = blockIdx.x * per, e = e0 + warp / wpe, sl = warp % wpe;
  Sum2 acc[GATE_TOKENS];
  if (e < E) {
    const TG* wr = wg + (int64_t)e * H;
#pragma unroll 1
    for (int k0 = (sl * 32 + lane) * 8; k0 < H; k0 += wpe * 256) {
      float w[8], v[GATE_TOKENS][8];
      load8(wr + k0, H - k0, vecg, w);
#pragma unroll
      for (int i = 0; i < GATE_TOKENS; ++i)
        if (i < nt) load8(x + (t0 + i) * ldx + k0, H - k0, vecx, v[i]);
#pragma unroll
      for (int i = 0; i < GATE_TOKENS; ++i)
        if (i < nt)
#pragma unroll
          for (int q = 0; q < 8; ++q) {
            const float p = __fmul_rn(v[i][q], w[q]);
            acc[i].add(p, SPLIT ? fmaf(v[i][q], w[q], -p) : 0.f);
          }
    }
  }
#pragma unroll
  for (int i = 0; i < GATE_TOKENS; ++i) {
    if (i < nt) {
#pragma unroll 1
      for (int o = 16; o > 0; o >>= 1) {
        const float s = __shfl_xor_sync(0xffffffffu, acc[i].s, o), c = __shfl_xor_sync(0xffffffffu, acc[i].c, o);
        acc[i].add(s, c);
      }
      if (lane == 0) part[i][warp] = make_float2(acc[i].s, acc[i].c);
    }
  }
  __syncthreads();
  if (threadIdx.x < per * GATE_TOKENS) {
    const int i = threadIdx.x / per, u = threadIdx.x % per;
    if (i < nt && e0 + u < E) {
      Sum2 a;
#pragma unroll 1
      for (int s = 0; s < wpe; ++s) a.add(part[i][u * wpe + s].x, part[i][u * wpe + s].y);
      logits[(int64_t)(t0 + i) * E + e0 + u] = a.value();
    }
  }
}

// ---------------------------------------------------------------------------
// entries by expert, by every block for itself
// ---------------------------------------------------------------------------
// Lists of R = B * k entries at most, in shared memory.
struct FewPlan {
  int* ids;          // [R] routed ids (-1: dropped)
  float* w;          // [R] their weights
  uint16_t* tok;     // [R] entry's token
  uint16_t* gexp;    // [R] group's expert
  uint16_t* gstart;  // [R] group's first entry
  uint16_t* gsize;   // [R] group's entries
  uint32_t* gcost;   // [R] cost of the groups up to and with this one
  int* count;        // groups, entries
};

// The routing of a call.
struct FewRouting {
  const float* logits;  // [B, E]: every block picks the experts itself; null: ids and weights are there
  int32_t* ids;         // [B, k]
  float* weights;       // [B, k]
  int B, k, E, norm;
  int32_t* pos;  // [B, k] entry of each slot (-1: dropped, or added to an earlier slot); written by gateup
  float* pw;     // [B, k] weight of each slot with a pos
  size_t bytes() const {
    return (size_t)B * k * 20 + 16 + (B == 1 ? 0 : (size_t)(E + 1) * 8 + (size_t)E * ((B + 31) / 32) * 4);
  }
};

// What a unit of a group of n tokens of T planes takes: the weights' decoding and, per
// column tile and plane, the products.  Cycles a unit of up to 8 and of 9 to 16 tokens:
// 4-bit gate and up 1970 / 2370, down (two planes) 1170 / 1640; ternary 1830 / 2185, 1180 / 1760.
template <int T>
__device__ __forceinline__ uint32_t group_cost(int n) {
  return 5u + T * (uint32_t)((n - 1) >> 3);
}

// Expert by expert, each expert's tokens ascending, cut into groups of `tile`.
// `first`: the block that writes pos and pw (and ids and weights, if it picked them) and
// reports dropped ids.  Reads logits, ids and weights past L1: with a gate they were
// written while this kernel waited to start.
template <int T>
__device__ __forceinline__ FewPlan few_group(const FewRouting& r, uint8_t* smem, int tile, bool first) {
  const int R = r.B * r.k, E = r.E;
  FewPlan p;
  p.ids = reinterpret_cast<int*>(smem);
  p.w = reinterpret_cast<float*>(p.ids + R);
  p.tok = reinterpret_cast<uint16_t*>(p.w + R);
  p.gexp = p.tok + R;
  p.gstart = p.gexp + R;
  p.gsize = p.gstart + R;
  p.gcost = reinterpret_cast<uint32_t*>(p.gsize + R);
  p.count = reinterpret_cast<int*>(p.gcost + R);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (r.logits != nullptr) {
    if (warp < r.B) few_topk(r.logits + warp * E, E, r.k, r.norm != 0, lane, p.ids + warp * r.k, p.w + warp * r.k);
  } else {
    for (int i = threadIdx.x; i < R; i += blockDim.x) {
      const int e = __ldcg(r.ids + i);
      const bool ok = e >= 0 && e < E;
      p.ids[i] = ok ? e : -1;
      p.w[i] = __ldcg(r.weights + i);
      if (!ok && first) set_status(ST_BAD_ARGUMENT);
    }
  }
  if (r.B == 1) {  // one token: a group for each of its experts, in slot order, by one warp
    if (warp == 0) {
      __syncwarp();
      const int e = lane < r.k ? p.ids[lane] : -1;
      const unsigned same = __match_any_sync(0xffffffffu, e >= 0 ? e : -1 - lane);
      const bool lead = e >= 0 && (same & ((1u << lane) - 1u)) == 0;
      const unsigned leads = __ballot_sync(0xffffffffu, lead);
      const int at = __popc(leads & ((1u << lane) - 1u));
      if (lead) {
        p.tok[at] = 0;
        p.gexp[at] = (uint16_t)e;
        p.gstart[at] = (uint16_t)at;
        p.gsize[at] = 1;
        p.gcost[at] = (uint32_t)(at + 1);  // all alike
      }
      if (first && lane < r.k) {
        float sum = 0.f;
        for (int j = 0; j < r.k; ++j)
          if ((same >> j) & 1u) sum += p.w[j];
        r.pos[lane] = lead ? at : -1;
        r.pw[lane] = sum;
        if (r.logits != nullptr) {
          r.ids[lane] = e;
          r.weights[lane] = p.w[lane];
        }
      }
      if (lane == 0) p.count[0] = p.count[1] = __popc(leads);
    }
    __syncthreads();
    return p;
  }
  const int words = (r.B + 31) / 32;
  int* off = p.count + 4;                                       // [E + 1] first entry of each expert
  int* goff = off + E + 1;                                      // [E + 1] first group of each expert
  uint32_t* mask = reinterpret_cast<uint32_t*>(goff + E + 1);   // [E][words] an expert's tokens
  for (int i = threadIdx.x; i < E * words; i += blockDim.x) mask[i] = 0u;
  __syncthreads();
  for (int i = threadIdx.x; i < R; i += blockDim.x) {
    const int e = p.ids[i], t = i / r.k;
    if (e >= 0) atomicOr(&mask[e * words + (t >> 5)], 1u << (t & 31));
    if (first && r.logits != nullptr) {
      r.ids[i] = e;
      r.weights[i] = p.w[i];
    }
  }
  __syncthreads();
  if (warp == 0) {
    int base = 0, gbase = 0;
    for (int e0 = 0; e0 < E; e0 += 32) {
      const int e = e0 + lane;
      int n = 0;
      if (e < E)
        for (int q = 0; q < words; ++q) n += __popc(mask[e * words + q]);
      const int gn = (n + tile - 1) / tile;
      int s = n | (gn << 16);  // both at most FEW_MAX_ENTRIES
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      if (e < E) {
        off[e] = base + (s & 0xffff) - n;
        goff[e] = gbase + (s >> 16) - gn;
      }
      s = __shfl_sync(0xffffffffu, s, 31);
      base += s & 0xffff;
      gbase += s >> 16;
    }
    if (lane == 0) {
      off[E] = base;
      goff[E] = gbase;
      p.count[0] = gbase;
      p.count[1] = base;
    }
  }
  __syncthreads();
  for (int i = threadIdx.x; i < R; i += blockDim.x) {
    const int e = p.ids[i], t = i / r.k, j = i - t * r.k;
    const int* slots = p.ids + t * r.k;
    bool again = e < 0;
    for (int q = 0; q < j; ++q) again |= slots[q] == e;
    int at = -1;
    if (!again) {
      at = off[e] + __popc(mask[e * words + (t >> 5)] & ((1u << (t & 31)) - 1u));
      for (int q = 0; q < (t >> 5); ++q) at += __popc(mask[e * words + q]);
      p.tok[at] = (uint16_t)t;
    }
    if (first) {
      float w = 0.f;
      for (int q = j; q < r.k; ++q)
        if (slots[q] == e) w += p.w[t * r.k + q];
      r.pos[i] = at;
      r.pw[i] = w;
    }
  }
  for (int e = threadIdx.x; e < E; e += blockDim.x)
    for (int gi = goff[e], at = off[e]; gi < goff[e + 1]; ++gi, at += tile) {
      p.gexp[gi] = (uint16_t)e;
      p.gstart[gi] = (uint16_t)at;
      p.gsize[gi] = (uint16_t)min(tile, off[e + 1] - at);
    }
  __syncthreads();
  if (warp == 0) {
    uint32_t base = 0;
    for (int g0 = 0; g0 < p.count[0]; g0 += 32) {
      const int gi = g0 + lane;
      uint32_t s = gi < p.count[0] ? group_cost<T>(p.gsize[gi]) : 0u;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const uint32_t a = __shfl_up_sync(0xffffffffu, s, o);
        if (lane >= o) s += a;
      }
      if (gi < p.count[0]) p.gcost[gi] = base + s;
      base += __shfl_sync(0xffffffffu, s, 31);
    }
  }
  __syncthreads();
  return p;
}

// The stream's work: the groups of a routing.  Tokens are x's rows (gate and up,
// `by_token`) or the entries' own (down).
struct FewRouted {
  FewRouting r;
  int by_token;
  int wait;  // the logits or ids come from the kernel before this one
  struct View {
    FewPlan p;
    int by_token;
    __device__ __forceinline__ uint32_t cost() const { return p.count[0] ? p.gcost[p.count[0] - 1] : 0u; }
    __device__ __forceinline__ void locate(uint32_t at, int runs, int start, int* gi, int* run) const {
      int lo = 0, hi = p.count[0];  // the first group that ends after `at`
      while (lo < hi) {
        const int mid = (lo + hi) >> 1;
        if (p.gcost[mid] * (uint32_t)(runs + start) > at)
          hi = mid;
        else
          lo = mid + 1;
      }
      *gi = lo;
      *run = 0;
      if (lo == p.count[0]) return;
      const uint32_t before = lo ? p.gcost[lo - 1] : 0u, one = p.gcost[lo] - before;
      *run = max(0, (int)((at - before * (uint32_t)(runs + start) + one - 1) / one) - start);
      if (*run == runs) {
        *run = 0;
        ++*gi;
      }
    }
    __device__ __forceinline__ FewGroup group(int gi) const { return FewGroup{p.gexp[gi], p.gsize[gi], p.gstart[gi]}; }
    __device__ __forceinline__ int row(int entry) const { return by_token ? p.tok[entry] : entry; }
  };
  size_t bytes() const { return r.bytes(); }
  bool waits() const { return wait != 0; }
  // the most groups that the entries can make: a group per touched expert and one per full tile
  int64_t groups(int tile) const {
    const int64_t R = (int64_t)r.B * r.k, most = (R < r.E ? R : r.E) + R / tile;
    return R < most ? R : most;
  }
  template <int T>
  __device__ __forceinline__ View view(uint8_t* smem, int tile, int) const {
    if (wait) few_wait();
    return View{few_group<T>(r, smem, tile, by_token && blockIdx.x == 0), by_token};
  }
};

// ---------------------------------------------------------------------------
// down and the sum over experts: few entries
// ---------------------------------------------------------------------------
// A block per 16 output channels.  Its warps share out the (group, chunk) items in
// order, each with its own sums [B, 16], added in warp order at the end.  The
// weights do not depend on the hidden rows, so every warp's ring is full before the
// wait for them.
constexpr int SUM_WARPS = 16, SUM_DEPTH = 4;

template <class W, int TH>
__global__ void __launch_bounds__(SUM_WARPS * 32, 1) moe_few_sum_kernel(W wd, FewX h, FewRouting route, int H, void* out,
                                                                        int out_dtype) {
  extern __shared__ __align__(128) uint8_t few_smem[];
  using Ring = FewRing<W, 1>;
  const int B = route.B, R = B * route.k;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31, g = lane >> 2, t = lane & 3;
  const int row_bytes = few_row_bytes(wd.chunks * W::CHUNK), chunks = wd.chunks;
  const uint32_t sx = smem_u32(few_smem);
  uint8_t* rings = few_smem + (size_t)R * TH * row_bytes;
  float* sums = reinterpret_cast<float*>(rings + SUM_WARPS * SUM_DEPTH * Ring::slot_bytes());  // [warp][B][16]
  uint64_t* bars = reinterpret_cast<uint64_t*>(sums + SUM_WARPS * B * 16);
  few_bars_init<W>(bars, SUM_WARPS * SUM_DEPTH);
  const FewPlan p = few_group<TH>(route, reinterpret_cast<uint8_t*>(bars + SUM_WARPS * SUM_DEPTH), 8, false);
  const int r0 = blockIdx.x * 16;
  float* mine = sums + (size_t)warp * B * 16;
  for (int i = lane; i < B * 16; i += 32) mine[i] = 0.f;
  const int items = p.count[0] * chunks;
  int item = items * warp / SUM_WARPS;
  const int end = items * (warp + 1) / SUM_WARPS;
  int gi = item / chunks, c = item - gi * chunks, fi = item, fg = gi, fc = c;
  Ring ring(rings, bars, warp, SUM_DEPTH);
  typename W::Tile front[1];
  if (item < end) front[0] = wd.tile(p.gexp[fg], blockIdx.x, H, lane);
  auto ahead = [&](int slot) {
    if (fi >= end) return;
    ring.fetch(slot, wd, front, fc, lane);
    ++fi;
    if (++fc == chunks) {
      fc = 0;
      if (fi < end) front[0] = wd.tile(p.gexp[++fg], blockIdx.x, H, lane);
    }
  };
#pragma unroll 1
  for (int d = 0; d < SUM_DEPTH; ++d) ahead(d);
  few_wait();
  few_stage<W, TH>(sx, h, p.count[1], chunks, [](int i) { return i; });
  cp_async_wait_all();
  __syncthreads();
  float acc[1][1][4] = {};
  typename W::template Part<1> part_ahead;
  int slot = 0;
  if (item < end) slot = ring.take(wd, part_ahead, lane);
#pragma unroll 1
  for (; item < end; ++item) {
    const int e = p.gexp[gi], first = p.gstart[gi], n = p.gsize[gi];
    const typename W::template Part<1> now = part_ahead;
    const int used = slot;
    if (item + 1 < end) slot = ring.take(wd, part_ahead, lane);
    ahead(used);
    wd.template chunk<1>(now, c, FewTokens<TH, 1>(sx + first * TH * row_bytes, n, row_bytes, g, t), acc);
    const bool last = c + 1 == chunks;
    if (last || item + 1 == end) {
      float sa = W::UNIT, sb = W::UNIT;
      if constexpr (W::ROW_SCALES) {
        sa = wd.out_scale((int64_t)e * H + min(r0 + g, H - 1));
        sb = wd.out_scale((int64_t)e * H + min(r0 + 8 + g, H - 1));
      }
#pragma unroll
      for (int q = 0; q < 2; ++q) {
        const int col = 2 * t + q;
        if (col < n) {  // tokens of a group differ: no two lanes add to one sum
          const int tok = p.tok[first + col], *slots = p.ids + tok * route.k;
          float wt = 0.f;
          for (int j = 0; j < route.k; ++j)
            if (slots[j] == e) wt += p.w[tok * route.k + j];
          float* s = mine + tok * 16 + g;
          s[0] = fmaf(wt, acc[0][0][q] * sa, s[0]);
          s[8] = fmaf(wt, acc[0][0][q + 2] * sb, s[8]);
        }
        acc[0][0][q] = acc[0][0][q + 2] = 0.f;
      }
      __syncwarp();
    }
    c = last ? 0 : c + 1;
    gi += last;
  }
  __syncthreads();
  for (int i = threadIdx.x; i < B * 16; i += SUM_WARPS * 32) {
    const int r = r0 + (i & 15);
    if (r >= H) continue;
    float v = 0.f;
#pragma unroll
    for (int q = 0; q < SUM_WARPS; ++q) v += sums[q * B * 16 + i];
    if (!isfinite(v)) set_status(ST_RANGE);
    store_out(out, out_dtype, (int64_t)(i >> 4) * H + r, v);
  }
}

constexpr int COMBINE_THREADS = 256;

// out[t] = sum_j pw[t, j] * y[pos[t, j]], slots ascending; a block per token and 256 channels
__global__ void __launch_bounds__(COMBINE_THREADS) moe_few_combine_kernel(const float* y, FewRouting r, int H, void* out,
                                                                      int out_dtype) {
  few_wait();
  const int t = blockIdx.y, c = blockIdx.x * COMBINE_THREADS + threadIdx.x;
  if (c >= H) return;
  float v = 0.f;
#pragma unroll 8
  for (int j = 0; j < r.k; ++j) {
    const int at = __ldcg(r.pos + t * r.k + j);
    if (at >= 0) v = fmaf(__ldcg(r.pw + t * r.k + j), __ldcg(y + (int64_t)at * H + c), v);
  }
  if (!isfinite(v)) set_status(ST_RANGE);
  store_out(out, out_dtype, (int64_t)t * H + c, v);
}

// ---------------------------------------------------------------------------
// host
// ---------------------------------------------------------------------------
struct FewLayout {
  size_t logits, pos, pw, h, y, total;  // the tokens' planes come first
};
inline FewLayout few_layout(int x_dtype, int64_t B, int64_t H, int64_t I, int E, int k) {
  FewLayout L;
  L.logits = few_planes_bytes(x_dtype, B, H);
  L.pos = L.logits + align_up((size_t)B * E * 4, 256);
  L.pw = L.pos + align_up((size_t)B * k * 4, 256);
  L.h = L.pw + align_up((size_t)B * k * 4, 256);
  L.y = L.h + align_up((size_t)(x_dtype == SB_BF16 ? 2 : 3) * B * k * align8(I) * 2, 256);
  L.total = L.y + align_up((size_t)B * k * H * 4, 256);
  return L;
}

// The one-kernel sum stages all hidden rows of the call in every block, where they fit:
// against products by expert and a combine, 18.5 / 24.0 us at 1 token, 28.2 / 33.3 at 2,
// 33.2 / 39.4 at 3, 38.3 / 45.4 at 4 (given routing, 64 experts, top 8, H 2048, I 1024).
template <class W, int T, int TH>
int moe_few(const W& gate, const W& up, const W& down, int64_t H, int64_t I, const FewX& x, const FewRouting& r,
            __nv_bfloat16* h, float* y, void* out, int out_dtype, bool routed, bool after, cudaStream_t st) {
  const int64_t R = (int64_t)r.B * r.k, ldh = align8(I);
  int rc;
  if ((rc = few_stream<W, true, T, TH>("moe_few_gateup", gate, up, x, FewRouted{r, 1, routed ? 1 : 0}, r.B, I,
                                       FewHidden{h, ldh, R * ldh}, FewRows{}, after, st)))
    return rc;
  const FewX hx{h, ldh, R * ldh, (int)ldh};
  const size_t rows = (size_t)R * TH * few_row_bytes(down.chunks * W::CHUNK);
  const size_t sum_smem =
      rows + SUM_WARPS * (SUM_DEPTH * (FewRing<W, 1>::slot_bytes() + 8) + (size_t)r.B * 64) + r.bytes();
  if (sum_smem + 1024 <= (size_t)FEW_SMEM) {
    auto kern = moe_few_sum_kernel<W, TH>;
    static PerDevice attr;
    if ((rc = few_allow_smem(attr, kern))) return rc;
    ProfScope prof("moe_few_sum", st);
    return few_launch(kern, dim3((unsigned)((H + 15) / 16)), SUM_WARPS * 32, sum_smem, st, down, hx, r, (int)H, out, out_dtype);
  }
  if ((rc = few_stream<W, false, TH, 1>("moe_few_down", down, down, hx, FewRouted{r, 0, 0}, r.B, H, FewHidden{},
                                        FewRows{y, SB_F32, nullptr}, true, st)))
    return rc;
  ProfScope prof("moe_few_combine", st);
  return few_launch(moe_few_combine_kernel, dim3((unsigned)((H + COMBINE_THREADS - 1) / COMBINE_THREADS), (unsigned)r.B),
                    COMBINE_THREADS, 0, st, y, r, (int)H, out, out_dtype);
}

template <class W>
int moe_few_dtype(int x_dtype, const W& gate, const W& up, const W& down, int64_t H, int64_t I, const FewX& x,
                  const FewRouting& r, __nv_bfloat16* h, float* y, void* out, int out_dtype, bool routed, bool after,
                  cudaStream_t st) {
  if (x_dtype == SB_BF16)
    return moe_few<W, 1, 2>(gate, up, down, H, I, x, r, h, y, out, out_dtype, routed, after, st);
  return moe_few<W, 3, 3>(gate, up, down, H, I, x, r, h, y, out, out_dtype, routed, after, st);
}

template <typename TX, typename TG>
int few_logits(const TX* x, int64_t ldx, int64_t B, int64_t H, int E, const TG* wg, float* logits, cudaStream_t st) {
  ProfScope prof("moe_few_logits", st);
  const bool vecx = (reinterpret_cast<uintptr_t>(x) & 15u) == 0 && ldx % (16 / sizeof(TX)) == 0;
  const bool vecg = (reinterpret_cast<uintptr_t>(wg) & 15u) == 0 && H % (16 / sizeof(TG)) == 0;
  const int64_t rows = (B + GATE_TOKENS - 1) / GATE_TOKENS;
  int wpe = GATE_WARPS;  // warps per expert: fewer where there are blocks enough
  while (wpe > 1 && rows * ((E + GATE_WARPS / wpe - 1) / (GATE_WARPS / wpe)) > 2 * num_sms()) wpe /= 2;
  const int per = GATE_WARPS / wpe;
  return few_launch(moe_few_logits_kernel<TX, TG>, dim3((unsigned)((E + per - 1) / per), (unsigned)rows), GATE_WARPS * 32,
                    0, st, x, ldx, (int)B, (int)H, E, wg, vecx, vecg, wpe, logits);
}

}  // namespace sb

extern "C" int sb_moe_few_max_tokens(int32_t top_k) {
  if (top_k < 1 || top_k > sb::FEW_MAX_TOPK) return 0;
  const int t = sb::FEW_MAX_ENTRIES / top_k;
  return t < sb::FEW_MAX_TOKENS ? t : sb::FEW_MAX_TOKENS;
}

extern "C" size_t sb_moe_few_workspace_bytes(int x_dtype, int64_t B, int64_t H, int64_t I, int32_t n_experts,
                                             int32_t top_k) {
  if (B < 0 || H <= 0 || I <= 0 || n_experts <= 0 || top_k <= 0) return 0;
  return sb::few_layout(x_dtype, B, H, I, n_experts, top_k).total;
}

extern "C" int sb_moe_few(const sb_experts* ex, const void* x, int x_dtype, int64_t ldx, int64_t B, int32_t top_k,
                          const void* gate_w, int gate_dtype, int norm_topk, int32_t* ids, float* weights, void* out,
                          int out_dtype, void* workspace, size_t workspace_bytes, void* stream) {
  using namespace sb;
  SB_REQUIRE(ex, "sb_moe_few: null experts");
  const int64_t H = ex->hidden, I = ex->intermediate;
  const int E = ex->n_experts;
  SB_REQUIRE(H > 0 && I > 0 && H <= FEW_MAX_WIDTH && I <= FEW_MAX_WIDTH, "sb_moe_few: H=%lld, I=%lld (1 to %d)",
             (long long)H, (long long)I, (int)FEW_MAX_WIDTH);
  SB_REQUIRE(E >= 1 && E <= FEW_MAX_EXPERTS, "sb_moe_few: %d experts (1 to %d)", E, FEW_MAX_EXPERTS);
  SB_REQUIRE(top_k >= 1 && top_k <= FEW_MAX_TOPK, "sb_moe_few: top_k %d (1 to %d)", (int)top_k, FEW_MAX_TOPK);
  SB_REQUIRE(!gate_w || top_k <= E, "sb_moe_few: top_k %d of %d experts", (int)top_k, E);
  SB_REQUIRE(B >= 0 && B <= sb_moe_few_max_tokens(top_k), "sb_moe_few: %lld tokens; at most %d for top_k %d",
             (long long)B, sb_moe_few_max_tokens(top_k), (int)top_k);
  SB_REQUIRE(ex->kind == SB_EXPERTS_TERNARY || ex->kind == SB_EXPERTS_GROUP4, "sb_moe_few: unknown kind of experts %d",
             (int)ex->kind);
  int rc;
  if ((rc = check_few_x(x, x_dtype, ldx, B, H, "sb_moe_few"))) return rc;
  SB_REQUIRE(!gate_w || gate_dtype == SB_F32 || gate_dtype == SB_BF16, "sb_moe_few: gate dtype must be SB_F32 or SB_BF16");
  SB_REQUIRE(out_dtype == SB_F32 || out_dtype == SB_BF16, "sb_moe_few: out dtype must be SB_F32 or SB_BF16");
  const bool g4 = ex->kind == SB_EXPERTS_GROUP4;
  SB_REQUIRE(ex->gate && ex->up && ex->down && (g4 || (ex->gate_scale && ex->up_scale && ex->down_scale)),
             "sb_moe_few: null expert weights");
  SB_REQUIRE(((reinterpret_cast<uintptr_t>(ex->gate) | reinterpret_cast<uintptr_t>(ex->up) |
               reinterpret_cast<uintptr_t>(ex->down)) & 15u) == 0,
             "sb_moe_few: packed weights must be 16-byte aligned");
  SB_REQUIRE(!g4 || group_shift(ex->group) > 0, "sb_moe_few: group %d must be 32, 64 or 128", (int)ex->group);
  if (B == 0) return SB_OK;
  SB_REQUIRE(ids && weights && out, "sb_moe_few: null ids, weights or out");
  const FewLayout L = few_layout(x_dtype, B, H, I, E, top_k);
  if ((rc = check_workspace(workspace, workspace_bytes, L.total))) return rc;
  uint8_t* ws = static_cast<uint8_t*>(workspace);
  const cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
  FewX fx;
  if ((rc = few_planes(x, x_dtype, ldx, B, H, ws, &fx, st))) return rc;
  bool after = few_planes_needed(x, x_dtype, ldx, H);
  FewRouting r{nullptr, ids, weights, (int)B, top_k, E, norm_topk, reinterpret_cast<int32_t*>(ws + L.pos),
               reinterpret_cast<float*>(ws + L.pw)};
  if (gate_w) {
    auto* logits = reinterpret_cast<float*>(ws + L.logits);
    const auto* xb = static_cast<const __nv_bfloat16*>(x);
    const auto* xf = static_cast<const float*>(x);
    const auto* gb = static_cast<const __nv_bfloat16*>(gate_w);
    const auto* gf = static_cast<const float*>(gate_w);
    if (x_dtype == SB_BF16)
      rc = gate_dtype == SB_BF16 ? few_logits(xb, ldx, B, H, E, gb, logits, st) : few_logits(xb, ldx, B, H, E, gf, logits, st);
    else
      rc = gate_dtype == SB_BF16 ? few_logits(xf, ldx, B, H, E, gb, logits, st) : few_logits(xf, ldx, B, H, E, gf, logits, st);
    if (rc) return rc;
    after = true;
    if (B <= FEW_OWN_TOPK) {
      r.logits = logits;
    } else {
      ProfScope prof("moe_few_topk", st);
      if ((rc = few_launch(moe_few_topk_kernel, dim3((unsigned)((B + 7) / 8)), 256, 0, st, (const float*)logits, (int)B, E,
                           (int)top_k, norm_topk, ids, weights)))
        return rc;
    }
  }
  auto* h = reinterpret_cast<__nv_bfloat16*>(ws + L.h);
  auto* y = reinterpret_cast<float*>(ws + L.y);
  const bool routed = gate_w != nullptr;
  if (g4)
    return with_group(ex->group, [&](auto gs) {
      auto matrix = [&](const void* data, int64_t K, int64_t N) {
        const sb_group4 m{const_cast<void*>(data), K, N, E, ex->group, ex->zeros};
        return group4_weights<gs.value>(&m);
      };
      return moe_few_dtype(x_dtype, matrix(ex->gate, H, I), matrix(ex->up, H, I), matrix(ex->down, I, H), H, I, fx, r, h,
                           y, out, out_dtype, routed, after, st);
    });
  auto matrix = [&](const void* w, const float* s, int64_t K) {
    return TernaryW{static_cast<const uint32_t*>(w), s, (int)((K + 255) / 256), (int)((K + 63) / 64)};
  };
  return moe_few_dtype(x_dtype, matrix(ex->gate, ex->gate_scale, H), matrix(ex->up, ex->up_scale, H),
                       matrix(ex->down, ex->down_scale, I), H, I, fx, r, h, y, out, out_dtype, routed, after, st);
}
