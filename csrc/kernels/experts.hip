// Expert routing and exchange: the gate's top-k choice with the stable order of the (token, choice)
// slots by expert, and the rows' way into that order and back with the weights applied.
//
//   route      S_t = the top_k experts of l[t, :], by value, ties to the lowest index
//              w_ti = exp(l_ti - m) / sum_j exp(l_tj - m), j over S_t (renormalized) or all experts
//              slot s = t k + j sorted stably by expert: pos[s] its place, src[place] = s, offs[e]
//              the first place of expert e (offs[E] = live slots)
//   route_bwd  dl_i = w_i (g_i - sum_S w g) on S_t, or p_i ([i in S_t] g_i - sum_S p g) on all
//   dispatch   xs[pos[t, j]] = x[t]                     its gradient: dx[t] = sum_j dxs[pos[t, j]]
//   combine    y[t] = sum_j w[t, j] ys[pos[t, j]]       dys[pos] = w dy[t], dw = <dy[t], ys[pos]>
//
// A logit that is -inf or NaN closes its expert (never chosen, no weight), +inf counts as the
// largest finite number; a token with fewer open experts than top_k has empty slots (expert -1,
// weight 0, pos -1), a token that is not valid has only such.  All sums are fp32 in a fixed order
// (no atomics): the same inputs give the same bits.
#include "common.h"

#define RT_MAXE 1024     // experts
#define RT_MAXK 16
#define RT_WAVES 8       // waves of a block (LDS histograms: 8 waves x 1024 x 4 B, or 16 x 512 x 4 B)
#define RT_CHUNK 256     // slots a wave keeps between its two phases
#define RT_MAXBLK 256

struct RouteArgs {
  const void* logits;      // [T, E] fp32 or bf16, row stride ld
  const uint8_t* valid;    // [T] or null
  int* expert;             // [T, k]
  float* weight;           // [T, k]
  int* pos;                // [T, k]
  int* src;                // [T k]
  int* offs;               // [E + 1]
  int* bh;                 // workspace [nblk + 1, E]: a block's slots per expert, then those of the blocks
                           // before it; all slots per expert
  int* wpre;               // workspace [nblk, waves, E]: slots of the block's waves before this one
  long ld;
  int T, E, k, renorm, bf, nblk, tpb;   // tpb: tokens per block
};

// Workgroups of 256 threads in x and y: a launch has less than 2^32 threads in x.
static dim3 wide_grid(long n) {
  const long row = 1l << 23;
  return dim3((unsigned)(n < row ? n : row), (unsigned)((n + row - 1) / row));
}

struct RouteBwdArgs {
  const void* logits;
  const int* expert;
  const float* weight;
  const float* dweight;    // [T, k]
  void* dlogits;           // [T, E], row stride ldo
  long ld, ldo;
  int T, E, k, renorm, bf;
};

__device__ __forceinline__ float gate_of(float v) {
  if (!(v == v)) v = -INFINITY;
  return fminf(v, 3.402823466e38f);
}
// A logit as an integer of the same order, and back (-0 made +0 before: they are equal).
constexpr int GATE_CLOSED = (int)(0xFF800000u ^ 0x7FFFFFFFu);       // -inf
__device__ __forceinline__ int gate_key(float v) {
  const int b = __float_as_int(v + 0.f);
  return b ^ ((b >> 31) & 0x7FFFFFFF);
}
__device__ __forceinline__ float key_gate(int b) { return __int_as_float(b ^ ((b >> 31) & 0x7FFFFFFF)); }

// Maximum or sum over each group of G lanes (G a power of two), in all of its lanes, by lane swaps
// in the vector unit: a shuffle through LDS takes over 100 cycles, and a choice needs one for each of
// log2 G steps (16384 x 64, top 2: 26 us with shuffles, 11 with these).
template <int G, typename T, typename F>
__device__ __forceinline__ T group_all(T x, F op) {
#define HFM_DPP(ctrl) __builtin_bit_cast(T, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), ctrl, 0xF, 0xF, true))
  if (G >= 2) x = op(x, HFM_DPP(0xB1));        // quad: 1 0 3 2
  if (G >= 4) x = op(x, HFM_DPP(0x4E));        // quad: 2 3 0 1
  if (G >= 8) x = op(x, HFM_DPP(0x141));       // half row mirrored (quads are uniform by now)
  if (G >= 16) x = op(x, HFM_DPP(0x140));      // row mirrored
#undef HFM_DPP
  if (G >= 32) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane16_swap(u, u, false, false);
    x = op(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
  }
  if (G >= 64) {
    const uint32_t u = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
    x = op(__builtin_bit_cast(T, (uint32_t)r[0]), __builtin_bit_cast(T, (uint32_t)r[1]));
  }
  return x;
}

// The top_k experts of one token by a group of G lanes (lane gl of the group holds experts gl + G q).
// Lane j of the group ends with choice j (expert, weight; -1, 0 if none).  Bound by its instructions: values
// are compared as integers (a float maximum comes with two instructions that quiet NaNs), and a lane's
// own values are put in order first (the k largest, equal ones by index), so that a choice compares one value a
// lane and its lane moves its list up (20011 x 256 bf16, top 8: 36 us with all float values compared in each choice
// and 8 waves a block, 25 so).
template <int G, int V>
__device__ __forceinline__ void route_token(const float (&o)[V], int k, int renorm, int lane, int& my_e, float& my_w) {
  static_assert(V == 1 || G == 64, "several values a lane: the whole wave has one token");
  const int gl = lane & (G - 1);
  auto larger = [](int a, int b) { return max(a, b); };
  int v[V], id[V], top = GATE_CLOSED, my_v = GATE_CLOSED;
  my_e = -1;
#pragma unroll
  for (int q = 0; q < V; ++q) {
    v[q] = gate_key(o[q]);
    id[q] = gl + G * q;
  }
  if constexpr (G == 64) {
#pragma unroll
    for (int p = 0; p < V - 1; ++p) {
      if (p >= k) break;
#pragma unroll
      for (int q = V - 1; q > p; --q) {
        const bool up = v[q] > v[q - 1];
        const int a = max(v[q], v[q - 1]), b = min(v[q], v[q - 1]), c = id[q], d = id[q - 1];
        v[q - 1] = a;
        v[q] = b;
        id[q - 1] = up ? c : d;
        id[q] = up ? d : c;
      }
    }
    for (int j = 0; j < k; ++j) {
      const int m = __builtin_amdgcn_readfirstlane(group_all<G>(v[0], larger));
      if (m == GATE_CLOSED) break;             // (no open one is left)
      if (j == 0) top = m;
      const unsigned long long has = __ballot(v[0] == m);
      int at = __builtin_amdgcn_readlane(id[0], __ffsll(has) - 1);       // the lowest index among equals
      for (unsigned long long more = has & (has - 1); more; more &= more - 1)
        at = min(at, __builtin_amdgcn_readlane(id[0], __ffsll(more) - 1));
      my_e = gl == j ? at : my_e;
      my_v = gl == j ? m : my_v;
      // (by masks: of a choice between neighbours the compiler makes an index, and of that 600 instructions)
      const int won = at == id[0] ? -1 : 0;
#pragma unroll
      for (int q = 0; q < V; ++q) {
        v[q] = (v[q] & ~won) | ((q + 1 < V ? v[q + 1] : GATE_CLOSED) & won);
        if (V > 1) id[q] = (id[q] & ~won) | ((q + 1 < V ? id[q + 1] : RT_MAXE) & won);
      }
    }
  } else {
    const unsigned long long mine = ((1ull << G) - 1) << (lane & ~(G - 1));
    for (int j = 0; j < k; ++j) {
      const int m = group_all<G>(v[0], larger);
      if (j == 0) top = m;
      const int at = (__ffsll(__ballot(v[0] == m) & mine) - 1) & (G - 1);
      if (gl == j) {
        my_e = m == GATE_CLOSED ? -1 : at;
        my_v = m;
      }
      if (at == gl) v[0] = GATE_CLOSED;
    }
  }
  const float ex = my_e >= 0 ? expf(key_gate(my_v) - key_gate(top)) : 0.f;
  float den = ex;
  if (!renorm) {
    den = 0.f;
#pragma unroll
    for (int q = 0; q < V; ++q) den += o[q] == -INFINITY ? 0.f : expf(o[q] - key_gate(top));
  }
  den = group_all<G>(den, [](float a, float b) { return a + b; });
  my_w = den > 0.f ? ex / den : 0.f;
}

// Places of a block's slots: `before` the expert's slots in earlier blocks, `all` its slots.
template <int W>
__device__ __forceinline__ void route_place(const RouteArgs& a, int b, int* base, int* scan, const int* before,
                                            const int* all, const int* wpre) {
  constexpr int THREADS = 64 * W;
  const int tid = threadIdx.x;
  int* tot = base + RT_MAXE;
  for (int e = tid; e < a.E; e += THREADS) {
    base[e] = before ? before[e] : 0;
    tot[e] = all[e];
  }
  __syncthreads();
  // exclusive scan of tot over the experts, by wave 0
  if (tid < 64) {
    int run = 0;
    for (int e0 = 0; e0 < a.E; e0 += 64) {
      const int c = e0 + tid < a.E ? tot[e0 + tid] : 0;
      int inc = c;
      for (int d = 1; d < 64; d <<= 1) {
        const int u = __shfl_up(inc, d);
        if (tid >= d) inc += u;
      }
      if (e0 + tid < a.E) {
        base[e0 + tid] += run + inc - c;
        if (b == 0) a.offs[e0 + tid] = run + inc - c;
      }
      run += __shfl(inc, 63);
    }
    if (tid == 0) {
      *scan = run;
      if (b == 0) a.offs[a.E] = run;
    }
  }
  __syncthreads();
  const int wave = tid >> 6, lane = tid & 63;
  const int t0 = b * a.tpb, t1 = min(a.T, t0 + a.tpb);
  const int per = (a.tpb + W - 1) / W;
  const int s0 = min(t1, t0 + wave * per) * a.k, s1 = min(t1, t0 + (wave + 1) * per) * a.k;
  for (int s = s0 + lane; s < s1; s += 64) {
    const int e = a.expert[s];
    if (e >= 0) {
      const int p = base[e] + wpre[wave * a.E + e] + a.pos[s];
      a.pos[s] = p;
      a.src[p] = s;
    }
  }
  const int live = *scan, n = a.T * a.k;    // places behind the last live slot
  for (int p = live + b * THREADS + tid; p < n; p += a.nblk * THREADS) a.src[p] = -1;
}

// grid nblk.  A wave takes a contiguous run of its block's tokens: choices first (a group of G lanes
// per token), then the rank of each slot among the wave's earlier slots of its expert (64 slots at a
// time: the lanes with the same expert by one ballot per index bit).  One block (few tokens) places
// its slots at once, several leave it to route_place_kernel.
template <int G, int V, int W>
__global__ void __launch_bounds__(64 * W) route_kernel(RouteArgs a) {
  constexpr int THREADS = 64 * W;
  extern __shared__ int lds[];
  int* wh = lds;                                                // [waves, E]
  short* se = reinterpret_cast<short*>(lds + W * a.E);   // [waves, RT_CHUNK]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int i = tid; i < W * a.E; i += THREADS) wh[i] = 0;
  __syncthreads();
  int* hist = wh + wave * a.E;
  short* es = se + wave * RT_CHUNK;
  const int b = blockIdx.x;
  const int t0 = b * a.tpb, t1 = min(a.T, t0 + a.tpb);
  const int per = (a.tpb + W - 1) / W;
  const int w0 = min(t1, t0 + wave * per), w1 = min(t1, t0 + (wave + 1) * per);
  const int gl = lane & (G - 1), gi = lane / G;
  constexpr int NG = 64 / G;                                     // tokens at a time
  const int ct = RT_CHUNK / a.k / NG * NG;                       // tokens per chunk
  int bits = 0;
  while ((1 << bits) < a.E) ++bits;
  // The next tokens' logits, under way: as loaded, from rows and columns that exist, with nothing between
  // the loads (a condition or a conversion there makes them wait for one another: 100000 x 128 bf16, top 4: 64
  // us, 55 so)
  uint32_t raw[V];
  uint32_t live = 0;
  auto fetch = [&](int t) {
    t = min(t, a.T - 1);
    live = a.valid ? a.valid[t] : 1;
    if (a.bf) {
      const uint16_t* l = reinterpret_cast<const uint16_t*>(a.logits) + (size_t)t * a.ld;
#pragma unroll
      for (int q = 0; q < V; ++q) raw[q] = l[min(gl + G * q, a.E - 1)];
    } else {
      const uint32_t* l = reinterpret_cast<const uint32_t*>(a.logits) + (size_t)t * a.ld;
#pragma unroll
      for (int q = 0; q < V; ++q) raw[q] = l[min(gl + G * q, a.E - 1)];
    }
  };
  if (w0 < w1) fetch(w0 + gi);
  for (int c0 = w0; c0 < w1; c0 += ct) {
    const int c1 = min(w1, c0 + ct);
    for (int t = c0 + gi; t - gi < c1; t += NG) {
      float v[V];
#pragma unroll
      for (int q = 0; q < V; ++q)
        v[q] = live && t < w1 && gl + G * q < a.E ? gate_of(__uint_as_float(a.bf ? raw[q] << 16 : raw[q])) : -INFINITY;
      fetch(t + NG);
      int e;
      float w;
      route_token<G, V>(v, a.k, a.renorm, lane, e, w);
      if (t < c1 && gl < a.k) {
        a.expert[(size_t)t * a.k + gl] = e;
        a.weight[(size_t)t * a.k + gl] = w;
        es[(t - c0) * a.k + gl] = (short)e;
      }
    }
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
    const int n = (c1 - c0) * a.k;
    for (int i0 = 0; i0 < n; i0 += 64) {
      const int i = i0 + lane;
      const int e = i < n ? es[i] : -1;
      unsigned long long same = __ballot(e >= 0);
      for (int q = 0; q < bits; ++q) {
        const unsigned long long m = __ballot((e >> q) & 1);
        same &= ((e >> q) & 1) ? m : ~m;
      }
      const int rank = __popcll(same & ((1ull << lane) - 1));
      int at = 0;
      if (e >= 0) at = hist[e];
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (e >= 0 && rank == 0) hist[e] = at + __popcll(same);
      __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");
      if (i < n) a.pos[(size_t)c0 * a.k + i] = e >= 0 ? at + rank : -1;
    }
  }
  __syncthreads();
  // slots of the block's earlier waves (in place), the block's histogram
  int* base = reinterpret_cast<int*>(se + W * RT_CHUNK);
  int* pre = gridDim.x == 1 ? wh : a.wpre + (size_t)b * W * a.E;
  int* own = gridDim.x == 1 ? base + 2 * RT_MAXE + 1 : a.bh + (size_t)b * a.E;
  for (int e = tid; e < a.E; e += THREADS) {
    int run = 0;
    for (int w = 0; w < W; ++w) {
      const int c = wh[w * a.E + e];
      pre[w * a.E + e] = run;
      run += c;
    }
    own[e] = run;
  }
  if (gridDim.x != 1) return;
  __threadfence_block();
  __syncthreads();
  route_place<W>(a, 0, base, base + 2 * RT_MAXE, nullptr, own, wh);
}

// Slots of the blocks before each block, per expert, and of all: 16 experts a workgroup, 16 runs of
// blocks each.  (Every placing block summing what it needs by itself: 20011 x 256: 37 us in all, 35
// so; 4096 x 1024: 104, 95.)
__global__ void __launch_bounds__(256) route_scan_kernel(RouteArgs a) {
  __shared__ int sum[16][17];
  constexpr int RUN = RT_MAXBLK / 16;
  const int c = threadIdx.x & 15, q = threadIdx.x >> 4, e = blockIdx.x * 16 + c;
  int n[RUN], run = 0;
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int b = q * RUN + i;
    n[i] = b < a.nblk && e < a.E ? a.bh[(size_t)b * a.E + e] : 0;
  }
#pragma unroll
  for (int i = 0; i < RUN; ++i) run += n[i];
  sum[q][c] = run;
  __syncthreads();
  int before = 0, all = 0;
#pragma unroll
  for (int i = 0; i < 16; ++i) {
    before += i < q ? sum[i][c] : 0;
    all += sum[i][c];
  }
  if (e >= a.E) return;
#pragma unroll
  for (int i = 0; i < RUN; ++i) {
    const int b = q * RUN + i;
    if (b < a.nblk) a.bh[(size_t)b * a.E + e] = before;
    before += n[i];
  }
  if (q == 0) a.bh[(size_t)a.nblk * a.E + e] = all;
}

// SCAN: after route_scan_kernel; without it (up to 64 experts) a block sums what it needs by itself.
template <int W, bool SCAN>
__global__ void __launch_bounds__(64 * W) route_place_kernel(RouteArgs a) {
  __shared__ int base[2 * RT_MAXE + 1], sums[128];
  const int b = blockIdx.x;
  const int *before = a.bh + (size_t)b * a.E, *all = a.bh + (size_t)a.nblk * a.E;
  if (!SCAN) {
    const int e = threadIdx.x & 63;
    if (threadIdx.x < 128) sums[threadIdx.x] = 0;
    __syncthreads();
    if (e < a.E) {
      int n = 0, m = 0;
#pragma unroll 16
      for (int r = threadIdx.x >> 6; r < a.nblk; r += W) {
        const int c = a.bh[(size_t)r * a.E + e];
        m += c;
        n += r < b ? c : 0;
      }
      atomicAdd(&sums[e], n);                // (integers: the order does not matter)
      atomicAdd(&sums[64 + e], m);
    }
    __syncthreads();
    before = sums;
    all = sums + 64;
  }
  route_place<W>(a, b, base, base + 2 * RT_MAXE, before, all, a.wpre + (size_t)b * W * a.E);
}

static int route_group(int E) {
  int G = 1;
  while (G < E && G < 64) G <<= 1;
  return G;
}

// Blocks of a call: one while a block's 8 waves take at most 4 rounds of tokens (one launch instead of
// three; 60 x 64, 8 rounds: 12.8 us so, 9.9 with blocks), else a round each, at most 256 (1000 x 1024: 33 us,
// with 4 rounds each 82).
HFM_API int hfm_route_blocks(int T, int E) {
  const int round = RT_WAVES * (64 / route_group(E));
  if (T <= 4 * round) return 1;
  const int n = (T + round - 1) / round;
  return n < RT_MAXBLK ? n : RT_MAXBLK;
}
// Waves of a block: 16 where a token takes a whole wave and their histograms fit the 64 KB, else 8 (both
// with one value a lane and more in us: 16384 x 64: 13.7, 15.0; 100000 x 128: 65, 92; 20011 x 256: 38, 48; 4096 x
// 1024: 90, 85; one block: 500 x 16: 12.9, 9.2).
static int route_waves(int T, int E) { return hfm_route_blocks(T, E) > 1 && E > 32 && E <= 512 ? 16 : RT_WAVES; }
HFM_API int hfm_route_ws_ints(int T, int E) {
  const int n = hfm_route_blocks(T, E);
  return n == 1 ? 0 : (n + 1) * E + n * E * route_waves(T, E);      // (one block keeps its counts in LDS)
}

HFM_API int hfm_route(const RouteArgs* ap, hipStream_t st) {
  RouteArgs a = *ap;
  if (a.T < 0 || a.E < 1 || a.E > RT_MAXE || a.k < 1 || a.k > RT_MAXK || a.k > a.E ||
      (long)a.T * a.k > (1l << 30))
    return (int)hipErrorInvalidValue;
  const int G = route_group(a.E);
  a.nblk = hfm_route_blocks(a.T, a.E);
  a.tpb = a.T > 0 ? (a.T + a.nblk - 1) / a.nblk : 1;
  a.wpre = a.bh + (size_t)(a.nblk + 1) * a.E;
  const int W = route_waves(a.T, a.E);
  size_t lds = (size_t)W * a.E * 4 + W * RT_CHUNK * 2;
  if (a.nblk == 1) lds += (3 * RT_MAXE + 1) * 4;
  const dim3 grid(a.nblk), blk(W * 64);
#define HFM_ROUTE(G, V, W) hipLaunchKernelGGL((route_kernel<G, V, W>), grid, blk, lds, st, a)
  switch (G) {
    case 1: HFM_ROUTE(1, 1, 8); break;
    case 2: HFM_ROUTE(2, 1, 8); break;
    case 4: HFM_ROUTE(4, 1, 8); break;
    case 8: HFM_ROUTE(8, 1, 8); break;
    case 16: HFM_ROUTE(16, 1, 8); break;
    case 32: HFM_ROUTE(32, 1, 8); break;
    default:
      if (a.E > 512) HFM_ROUTE(64, 16, 8);
      else if (W == 8) {                         // (one block)
        if (a.E <= 64) HFM_ROUTE(64, 1, 8);
        else if (a.E <= 128) HFM_ROUTE(64, 2, 8);
        else if (a.E <= 256) HFM_ROUTE(64, 4, 8);
        else HFM_ROUTE(64, 8, 8);
      } else {
        if (a.E <= 64) HFM_ROUTE(64, 1, 16);
        else if (a.E <= 128) HFM_ROUTE(64, 2, 16);
        else if (a.E <= 256) HFM_ROUTE(64, 4, 16);
        else HFM_ROUTE(64, 8, 16);
      }
  }
#undef HFM_ROUTE
  if (a.nblk > 1) {
    // (16384 x 64 with its gradient, from Python: 32 us with the scan's launch, 29 so)
    if (a.E > 64) hipLaunchKernelGGL(route_scan_kernel, dim3((a.E + 15) / 16), dim3(256), 0, st, a);
    if (a.E > 64 && W == 8) hipLaunchKernelGGL((route_place_kernel<8, true>), grid, blk, 0, st, a);
    else if (a.E > 64) hipLaunchKernelGGL((route_place_kernel<16, true>), grid, blk, 0, st, a);
    else if (W == 8) hipLaunchKernelGGL((route_place_kernel<8, false>), grid, blk, 0, st, a);
    else hipLaunchKernelGGL((route_place_kernel<16, false>), grid, blk, 0, st, a);
  }
  HFM_LAUNCH_CHECK();
}

// A group of G lanes per token: lane j has choice j, and 16 bytes of the row a turn.  The row is written as
// if no expert were chosen (zeros, or -p dot), then the chosen ones over it.  p_i needs no second
// softmax: the first choice has the largest logit m and the weight exp(0) / den, so p_i = exp(l_i - m) w_0.
// (20011 x 256 bf16, top 8, renormalized: 18 us with every element compared with every choice, 7 so.)
template <typename T, int G>
__global__ void __launch_bounds__(256) route_bwd_kernel(RouteBwdArgs a) {
  constexpr int V = 16 / sizeof(T);
  typedef T vec __attribute__((ext_vector_type(V), aligned(sizeof(T))));
  const int gl = threadIdx.x & (G - 1);
  const long t = ((long)blockIdx.y * gridDim.x + blockIdx.x) * (256 / G) + threadIdx.x / G;
  if (t >= a.T) return;
  const size_t o = (size_t)t * a.k + gl;
  const int e = gl < a.k ? a.expert[o] : -1;
  const float w = e >= 0 ? a.weight[o] : 0.f, g = e >= 0 ? a.dweight[o] : 0.f;
  const float dot = group_all<G>(e >= 0 ? w * g : 0.f, [](float x, float y) { return x + y; });
  const T* l = reinterpret_cast<const T*>(a.logits) + (size_t)t * a.ld;
  T* d = reinterpret_cast<T*>(a.dlogits) + (size_t)t * a.ldo;
  const int e0 = __shfl(e, 0, G);
  const bool soft = !a.renorm && e0 >= 0 && e0 < a.E;
  const float m = soft ? gate_of((float)l[e0]) : 0.f, c = -__shfl(w, 0, G) * dot;
  for (int i = gl * V; i < a.E; i += G * V) {
    vec v = {};
    if (i + V <= a.E) {
      if (soft) {
        const vec x = *reinterpret_cast<const vec*>(l + i);
#pragma unroll
        for (int q = 0; q < V; ++q) v[q] = (T)(c * expf(gate_of((float)x[q]) - m));
      }
      *reinterpret_cast<vec*>(d + i) = v;
    } else {
      for (int q = i; q < a.E; ++q) d[q] = soft ? (T)(c * expf(gate_of((float)l[q]) - m)) : (T)0.f;
    }
  }
  __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "wavefront");       // (the wave's stores stay in order)
  if (e >= 0 && e < a.E) d[e] = (T)(w * (g - dot));
}

template <typename T>
static void route_bwd(const RouteBwdArgs& a, hipStream_t st) {
  const int lanes = (a.E * (int)sizeof(T) + 15) / 16;          // (and one for each choice)
  const int G = lanes <= 16 ? 16 : lanes <= 32 ? 32 : 64;
  const dim3 grid = wide_grid((a.T + 256l / G - 1) / (256 / G)), blk(256);
  if (G == 16) hipLaunchKernelGGL((route_bwd_kernel<T, 16>), grid, blk, 0, st, a);
  else if (G == 32) hipLaunchKernelGGL((route_bwd_kernel<T, 32>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((route_bwd_kernel<T, 64>), grid, blk, 0, st, a);
}

HFM_API int hfm_route_bwd(const RouteBwdArgs* ap, hipStream_t st) {
  const RouteBwdArgs& a = *ap;
  if (a.T < 0 || a.E < 1 || a.E > RT_MAXE || a.k < 1 || a.k > RT_MAXK) return (int)hipErrorInvalidValue;
  if (a.T == 0) return 0;
  if (a.bf) route_bwd<bf16>(a, st);
  else route_bwd<float>(a, st);
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_route_args_bytes() { return (int)sizeof(RouteArgs); }
HFM_API int hfm_route_bwd_args_bytes() { return (int)sizeof(RouteBwdArgs); }

// ------------------------------------------------------------------ exchange
// One wave per token, 16 bytes per lane and turn, a row's last elements (fewer than 16 bytes) one by one;
// a token's row is read once for all its slots (dispatch, combine_bwd), or its slots' rows summed in
// order (combine, dispatch_bwd).  Bound by the rows' bytes.  A 16-byte access of global memory may start at
// any element: rows of an odd width take the same accesses as aligned ones.  The four exchanges together: 10007
// rows of 313 floats with 4 slots 77 us, 3.3 TB/s (with single elements 95; with one turn's loads at a time 87);
// 16384 rows of 1248 bf16 with 2 slots 112 us, 4.4 TB/s (one turn's: 118).
struct ExchArgs {
  const void* a;           // x / dxs / ys / dy
  const void* b;           // combine_bwd: ys
  void* out;               // xs / dx / y / dys
  const int* pos;          // [T, k]
  const float* weight;     // [T, k] (combine, combine_bwd)
  float* dweight;          // [T, k] (combine_bwd)
  long lda, ldb, ldo;      // row strides in elements
  int T, k, D, S;          // S: rows of the expert order
  int bf;                  // bf16 rows (else fp32)
};

template <typename T, int V>
struct RowVec {               // (aligned to an element only)
  typedef T type __attribute__((ext_vector_type(V), aligned(sizeof(T))));
};
enum { EX_DISPATCH = 0, EX_DISPATCH_BWD = 1, EX_COMBINE = 2, EX_COMBINE_BWD = 3 };

// Columns c + 64 V u .. + V - 1 of token t's rows, for the U turns u of them that lie before `end`; all rows'
// loads of the U turns are under way before any is used or written (combine_bwd may write over ys).
template <typename T, int V, int U, int K, int MODE>
__device__ __forceinline__ void exchange_cols(const ExchArgs& a, size_t t, int c, int end, const int (&p)[K], const float (&w)[K],
                                              float (&dot)[K]) {
  const T* A = reinterpret_cast<const T*>(a.a) + c;
  const T* B = reinterpret_cast<const T*>(a.b) + c;
  T* O = reinterpret_cast<T*>(a.out) + c;
  typedef typename RowVec<T, V>::type vec;
  auto at = [&](const T* x, size_t row, long ld, int u) -> vec { return *reinterpret_cast<const vec*>(x + row * ld + u * 64 * V); };
  auto on = [&](int u) { return u == 0 || c + u * 64 * V < end; };
  vec g[U], y[U][K];
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!on(u)) continue;
    if (MODE == EX_DISPATCH || MODE == EX_COMBINE_BWD) g[u] = at(A, t, a.lda, u);
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (MODE == EX_COMBINE_BWD && p[j] >= 0) y[u][j] = at(B, p[j], a.ldb, u);
      if ((MODE == EX_COMBINE || MODE == EX_DISPATCH_BWD) && p[j] >= 0) y[u][j] = at(A, p[j], a.lda, u);
    }
  }
#pragma unroll
  for (int u = 0; u < U; ++u) {
    if (!on(u)) continue;
    float s[V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j) {
      if (p[j] < 0) continue;
      if (MODE == EX_DISPATCH) {
        *reinterpret_cast<vec*>(O + (size_t)p[j] * a.ldo + u * 64 * V) = g[u];
      } else if (MODE == EX_COMBINE_BWD) {
        vec d;
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = (T)(w[j] * (float)g[u][i]);
          dot[j] = fmaf((float)g[u][i], (float)y[u][j][i], dot[j]);
        }
        *reinterpret_cast<vec*>(O + (size_t)p[j] * a.ldo + u * 64 * V) = d;
      } else {
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = MODE == EX_COMBINE ? fmaf(w[j], (float)y[u][j][i], s[i]) : s[i] + (float)y[u][j][i];
      }
    }
    if (MODE == EX_COMBINE || MODE == EX_DISPATCH_BWD) {
      vec d;
#pragma unroll
      for (int i = 0; i < V; ++i) d[i] = (T)s[i];
      *reinterpret_cast<vec*>(O + (size_t)t * a.ldo + u * 64 * V) = d;
    }
  }
}

template <typename T, int K, int MODE>
__global__ void __launch_bounds__(256) exchange_kernel(ExchArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const long t = ((long)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (t >= a.T) return;
  int p[K];
  float w[K], dot[K];
#pragma unroll
  for (int j = 0; j < K; ++j) {
    p[j] = j < a.k ? a.pos[(size_t)t * a.k + j] : -1;
    if (p[j] >= a.S) p[j] = -1;            // (never out of the rows)
    w[j] = MODE == EX_COMBINE || MODE == EX_COMBINE_BWD ? (j < a.k ? a.weight[(size_t)t * a.k + j] : 0.f) : 1.f;
    dot[j] = 0.f;
  }
  const int D16 = a.D / V * V;
  constexpr int U = K <= 4 && MODE != EX_DISPATCH ? 2 : 1;           // (dispatch has one load a turn)
  for (int c = lane * V; c < D16; c += U * 64 * V) exchange_cols<T, V, U, K, MODE>(a, t, c, D16, p, w, dot);
  if (D16 + lane < a.D) exchange_cols<T, 1, 1, K, MODE>(a, t, D16 + lane, a.D, p, w, dot);
  if (MODE == EX_COMBINE_BWD) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      dot[j] = group_all<64>(dot[j], [](float x, float y) { return x + y; });
      if (lane == 0 && j < a.k) a.dweight[(size_t)t * a.k + j] = p[j] >= 0 ? dot[j] : 0.f;
    }
  }
}

template <typename T, int MODE>
static void exchange_k(const ExchArgs& a, hipStream_t st) {
  const dim3 grid = wide_grid((a.T + 3l) / 4), blk(256);
  if (a.k <= 1) hipLaunchKernelGGL((exchange_kernel<T, 1, MODE>), grid, blk, 0, st, a);
  else if (a.k <= 2) hipLaunchKernelGGL((exchange_kernel<T, 2, MODE>), grid, blk, 0, st, a);
  else if (a.k <= 4) hipLaunchKernelGGL((exchange_kernel<T, 4, MODE>), grid, blk, 0, st, a);
  else if (a.k <= 8) hipLaunchKernelGGL((exchange_kernel<T, 8, MODE>), grid, blk, 0, st, a);
  else hipLaunchKernelGGL((exchange_kernel<T, 16, MODE>), grid, blk, 0, st, a);
}

template <int MODE>
static void exchange_mode(const ExchArgs& a, hipStream_t st) {
  if (a.bf) exchange_k<bf16, MODE>(a, st);
  else exchange_k<float, MODE>(a, st);
}

HFM_API int hfm_exchange(int mode, const ExchArgs* ap, hipStream_t st) {
  const ExchArgs& a = *ap;
  if (a.T < 0 || a.k < 1 || a.k > RT_MAXK || a.D < 0) return (int)hipErrorInvalidValue;
  if (a.T == 0) return 0;
  switch (mode) {
    case EX_DISPATCH: exchange_mode<EX_DISPATCH>(a, st); break;
    case EX_DISPATCH_BWD: exchange_mode<EX_DISPATCH_BWD>(a, st); break;
    case EX_COMBINE: exchange_mode<EX_COMBINE>(a, st); break;
    case EX_COMBINE_BWD: exchange_mode<EX_COMBINE_BWD>(a, st); break;
    default: return (int)hipErrorInvalidValue;
  }
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_exch_args_bytes() { return (int)sizeof(ExchArgs); }
