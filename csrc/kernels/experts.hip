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

#define RT_MAXE 1024     // experts (LDS histograms: 8 waves x 1024 x 4 B)
#define RT_MAXK 16
#define RT_THREADS 512
#define RT_WAVES (RT_THREADS / 64)
#define RT_CHUNK 512     // slots a wave keeps between its two phases
#define RT_MAXBLK 256

struct RouteArgs {
  const void* logits;      // [T, E] fp32 or bf16, row stride ld
  const uint8_t* valid;    // [T] or null
  int* expert;             // [T, k]
  float* weight;           // [T, k]
  int* pos;                // [T, k]
  int* src;                // [T k]
  int* offs;               // [E + 1]
  int* bh;                 // workspace [nblk, E]: a block's slots per expert
  int* wpre;               // workspace [nblk, waves, E]: slots of the block's waves before this one
  long ld;
  int T, E, k, renorm, bf, nblk, tpb;   // tpb: tokens per block
};

struct RouteBwdArgs {
  const void* logits;
  const int* expert;
  const float* weight;
  const float* dweight;    // [T, k]
  void* dlogits;           // [T, E], row stride ldo
  long ld, ldo;
  int T, E, k, renorm, bf;
};

__device__ __forceinline__ float gate_value(const void* l, size_t i, int bf) {
  float v = bf ? bf2f(reinterpret_cast<const bf16*>(l)[i]) : reinterpret_cast<const float*>(l)[i];
  if (!(v == v)) v = -INFINITY;
  return fminf(v, 3.402823466e38f);
}

// Maximum and sum over each group of G lanes (G a power of two), in all of its lanes, by lane swaps
// in the vector unit: a shuffle through LDS takes over 100 cycles, and a choice needs one for each of
// log2 G steps (16384 x 64, top 2: 26 us with shuffles, 11 with these).
template <int G, typename F>
__device__ __forceinline__ float group_all(float v, F op) {
#define HFM_DPP(ctrl) __uint_as_float((uint32_t)__builtin_amdgcn_mov_dpp((int)__float_as_uint(v), ctrl, 0xF, 0xF, true))
  if (G >= 2) v = op(v, HFM_DPP(0xB1));        // quad: 1 0 3 2
  if (G >= 4) v = op(v, HFM_DPP(0x4E));        // quad: 2 3 0 1
  if (G >= 8) v = op(v, HFM_DPP(0x141));       // half row mirrored (quads are uniform by now)
  if (G >= 16) v = op(v, HFM_DPP(0x140));      // row mirrored
#undef HFM_DPP
  if (G >= 32) {
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  if (G >= 64) {
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(v), __float_as_uint(v), false, false);
    v = op(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  return v;
}

// The top_k experts of one token by a group of G lanes (lane gl of the group holds experts gl + G q).
// Lane j of the group ends with choice j (expert, weight; -1, 0 if none).
template <int G, int V>
__device__ __forceinline__ void route_token(float (&v)[V], int k, int renorm, int lane, int& my_e, float& my_w) {
  const int gl = lane & (G - 1);
  const unsigned long long mine = (G == 64 ? ~0ull : ((1ull << G) - 1) << (lane & ~(G - 1)));
  float top = -INFINITY, my_v = -INFINITY, o[V];
  my_e = -1;
#pragma unroll
  for (int q = 0; q < V; ++q) o[q] = v[q];
  for (int j = 0; j < k; ++j) {
    float m = v[0];
#pragma unroll
    for (int q = 1; q < V; ++q) m = fmaxf(m, v[q]);
    m = group_all<G>(m, [](float a, float b) { return fmaxf(a, b); });
    if (j == 0) top = m;
    // the lowest index among equals: the first q that has one, its first lane
    int at = -1;
#pragma unroll
    for (int q = V - 1; q >= 0; --q) {
      const unsigned long long has = __ballot(v[q] == m) & mine;
      if (has) at = G * q + ((__ffsll(has) - 1) & (G - 1));
    }
    if (m == -INFINITY) at = -1;              // (all closed)
    if (gl == j) {
      my_e = at;
      my_v = m;
    }
#pragma unroll
    for (int q = 0; q < V; ++q)
      if (at == gl + G * q) v[q] = -INFINITY;
  }
  const float ex = my_e >= 0 ? expf(my_v - top) : 0.f;
  float den = ex;
  if (!renorm) {
    den = 0.f;
#pragma unroll
    for (int q = 0; q < V; ++q) den += o[q] == -INFINITY ? 0.f : expf(o[q] - top);
  }
  den = group_all<G>(den, [](float a, float b) { return a + b; });
  my_w = den > 0.f ? ex / den : 0.f;
}

// Places of a block's slots, once every block's histogram is known (sums over blocks in LDS).
__device__ __forceinline__ void route_place(const RouteArgs& a, int b, int* base, int* scan, const int* wpre) {
  const int tid = threadIdx.x;
  // base[e] = slots of expert e in earlier blocks, tot[e] in all: rows split over thread groups
  int* tot = base + RT_MAXE;
  for (int e = tid; e < a.E; e += RT_THREADS) base[e] = tot[e] = 0;
  __syncthreads();
  int ep = 1;
  while (ep < a.E) ep <<= 1;
  if (ep > RT_THREADS) ep = RT_THREADS;
  const int ng = RT_THREADS / ep, gr = tid / ep;
  for (int e = tid % ep; e < a.E; e += ep) {
    int before = 0, all = 0;
#pragma unroll 8
    for (int r = gr; r < a.nblk; r += ng) {
      const int c = a.bh[(size_t)r * a.E + e];
      all += c;
      before += r < b ? c : 0;
    }
    atomicAdd(&base[e], before);           // (integers: the order does not matter)
    atomicAdd(&tot[e], all);
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
  const int per = (a.tpb + RT_WAVES - 1) / RT_WAVES;
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
  for (int p = live + b * RT_THREADS + tid; p < n; p += a.nblk * RT_THREADS) a.src[p] = -1;
}

// grid nblk.  A wave takes a contiguous run of its block's tokens: choices first (a group of G lanes
// per token), then the rank of each slot among the wave's earlier slots of its expert (64 slots at a
// time: the lanes with the same expert by one ballot per index bit).  One block (few tokens) places
// its slots at once, several leave it to route_place_kernel.
template <int G, int V>
__global__ void __launch_bounds__(RT_THREADS) route_kernel(RouteArgs a) {
  extern __shared__ int lds[];
  int* wh = lds;                                                // [waves, E]
  short* se = reinterpret_cast<short*>(lds + RT_WAVES * a.E);   // [waves, RT_CHUNK]
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  for (int i = tid; i < RT_WAVES * a.E; i += RT_THREADS) wh[i] = 0;
  __syncthreads();
  int* hist = wh + wave * a.E;
  short* es = se + wave * RT_CHUNK;
  const int b = blockIdx.x;
  const int t0 = b * a.tpb, t1 = min(a.T, t0 + a.tpb);
  const int per = (a.tpb + RT_WAVES - 1) / RT_WAVES;
  const int w0 = min(t1, t0 + wave * per), w1 = min(t1, t0 + (wave + 1) * per);
  const int gl = lane & (G - 1), gi = lane / G;
  constexpr int NG = 64 / G;                                     // tokens at a time
  const int ct = RT_CHUNK / a.k / NG * NG;                       // tokens per chunk
  int bits = 0;
  while ((1 << bits) < a.E) ++bits;
  float nv[V];                                                   // the next tokens' logits, under way
  auto fetch = [&](int t) {
    const bool on = t < w1 && (!a.valid || a.valid[t]);
#pragma unroll
    for (int q = 0; q < V; ++q) {
      const int e = gl + G * q;
      nv[q] = on && e < a.E ? gate_value(a.logits, (size_t)t * a.ld + e, a.bf) : -INFINITY;
    }
  };
  fetch(w0 + gi);
  for (int c0 = w0; c0 < w1; c0 += ct) {
    const int c1 = min(w1, c0 + ct);
    for (int t = c0 + gi; t - gi < c1; t += NG) {
      float v[V];
#pragma unroll
      for (int q = 0; q < V; ++q) v[q] = nv[q];
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
  int* base = reinterpret_cast<int*>(se + RT_WAVES * RT_CHUNK);
  int* pre = gridDim.x == 1 ? wh : a.wpre + (size_t)b * RT_WAVES * a.E;
  if (gridDim.x == 1) a.bh = base + 2 * RT_MAXE + 1;
  for (int e = tid; e < a.E; e += RT_THREADS) {
    int run = 0;
    for (int w = 0; w < RT_WAVES; ++w) {
      const int c = wh[w * a.E + e];
      pre[w * a.E + e] = run;
      run += c;
    }
    a.bh[(size_t)b * a.E + e] = run;
  }
  if (gridDim.x != 1) return;
  __threadfence_block();
  __syncthreads();
  route_place(a, 0, base, base + 2 * RT_MAXE, wh);
}

__global__ void __launch_bounds__(RT_THREADS) route_place_kernel(RouteArgs a) {
  __shared__ int base[2 * RT_MAXE + 1];
  route_place(a, blockIdx.x, base, base + 2 * RT_MAXE, a.wpre + (size_t)blockIdx.x * RT_WAVES * a.E);
}

static int route_group(int E) {
  int G = 1;
  while (G < E && G < 64) G <<= 1;
  return G;
}

// Blocks of a call: one while a block's 8 waves take at most 8 rounds of tokens, else at most 256
// (a placing block reads every block's histogram), each with 4 rounds or more.
HFM_API int hfm_route_blocks(int T, int E) {
  const int round = RT_WAVES * (64 / route_group(E));
  if (T <= 8 * round) return 1;
  const int n = (T + 4 * round - 1) / (4 * round);
  return n < RT_MAXBLK ? n : RT_MAXBLK;
}
HFM_API int hfm_route_ws_ints(int T, int E) {
  const int n = hfm_route_blocks(T, E);
  return n == 1 ? 0 : n * E * (1 + RT_WAVES);      // (one block keeps its counts in LDS)
}

HFM_API int hfm_route(const RouteArgs* ap, hipStream_t st) {
  RouteArgs a = *ap;
  if (a.T < 0 || a.E < 1 || a.E > RT_MAXE || a.k < 1 || a.k > RT_MAXK || a.k > a.E ||
      (long)a.T * a.k > (1l << 30))
    return (int)hipErrorInvalidValue;
  const int G = route_group(a.E);
  a.nblk = hfm_route_blocks(a.T, a.E);
  a.tpb = a.T > 0 ? (a.T + a.nblk - 1) / a.nblk : 1;
  a.wpre = a.bh + (size_t)a.nblk * a.E;
  size_t lds = (size_t)RT_WAVES * a.E * 4 + RT_WAVES * RT_CHUNK * 2;
  if (a.nblk == 1) lds += (3 * RT_MAXE + 1) * 4;
  const dim3 grid(a.nblk), blk(RT_THREADS);
#define HFM_ROUTE(G, V) hipLaunchKernelGGL((route_kernel<G, V>), grid, blk, lds, st, a)
  switch (G) {
    case 1: HFM_ROUTE(1, 1); break;
    case 2: HFM_ROUTE(2, 1); break;
    case 4: HFM_ROUTE(4, 1); break;
    case 8: HFM_ROUTE(8, 1); break;
    case 16: HFM_ROUTE(16, 1); break;
    case 32: HFM_ROUTE(32, 1); break;
    default:
      if (a.E <= 64) HFM_ROUTE(64, 1);
      else if (a.E <= 128) HFM_ROUTE(64, 2);
      else if (a.E <= 256) HFM_ROUTE(64, 4);
      else if (a.E <= 512) HFM_ROUTE(64, 8);
      else HFM_ROUTE(64, 16);
  }
#undef HFM_ROUTE
  if (a.nblk > 1) hipLaunchKernelGGL(route_place_kernel, grid, blk, 0, st, a);
  HFM_LAUNCH_CHECK();
}

// A group of G lanes per token again.  p_i needs no second softmax: the first choice has the largest
// logit m and the weight exp(0) / den, so p_i = exp(l_i - m) w_0.
template <int K>
__global__ void __launch_bounds__(256) route_bwd_kernel(RouteBwdArgs a, int G) {
  const int lane = threadIdx.x & 63;
  const int gl = lane & (G - 1);
  const int t = (int)(((long)blockIdx.x * 256 + threadIdx.x) / G);
  if (t >= a.T) return;
  int ex[K];
  float w[K], g[K], dot = 0.f;
#pragma unroll
  for (int j = 0; j < K; ++j) {
    const size_t o = (size_t)t * a.k + j;
    ex[j] = j < a.k ? a.expert[o] : -1;
    w[j] = j < a.k ? a.weight[o] : 0.f;
    g[j] = j < a.k ? a.dweight[o] : 0.f;
  }
#pragma unroll
  for (int j = 0; j < K; ++j)
    if (ex[j] >= 0) dot = fmaf(w[j], g[j], dot);
  const bool any = ex[0] >= 0 && ex[0] < a.E;
  const float m = any && !a.renorm ? gate_value(a.logits, (size_t)t * a.ld + ex[0], a.bf) : 0.f;
#pragma unroll 4
  for (int i = gl; i < a.E; i += G) {
    float d = 0.f;
    if (any) {
      if (!a.renorm) {
        const float l = gate_value(a.logits, (size_t)t * a.ld + i, a.bf);
        if (l != -INFINITY) d = -expf(l - m) * w[0] * dot;
      }
#pragma unroll
      for (int j = 0; j < K; ++j)
        if (ex[j] == i) d = a.renorm ? w[j] * (g[j] - dot) : fmaf(w[j], g[j], d);
    }
    const size_t o = (size_t)t * a.ldo + i;
    if (a.bf) reinterpret_cast<bf16*>(a.dlogits)[o] = f2bf(d);
    else reinterpret_cast<float*>(a.dlogits)[o] = d;
  }
}

HFM_API int hfm_route_bwd(const RouteBwdArgs* ap, hipStream_t st) {
  const RouteBwdArgs a = *ap;
  if (a.T < 0 || a.E < 1 || a.E > RT_MAXE || a.k < 1 || a.k > RT_MAXK) return (int)hipErrorInvalidValue;
  if (a.T == 0) return 0;
  const int G = route_group(a.E), per = 256 / G;
  const dim3 grid((a.T + per - 1) / per), blk(256);
  if (a.k <= 1) hipLaunchKernelGGL(route_bwd_kernel<1>, grid, blk, 0, st, a, G);
  else if (a.k <= 2) hipLaunchKernelGGL(route_bwd_kernel<2>, grid, blk, 0, st, a, G);
  else if (a.k <= 4) hipLaunchKernelGGL(route_bwd_kernel<4>, grid, blk, 0, st, a, G);
  else if (a.k <= 8) hipLaunchKernelGGL(route_bwd_kernel<8>, grid, blk, 0, st, a, G);
  else hipLaunchKernelGGL(route_bwd_kernel<16>, grid, blk, 0, st, a, G);
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_route_args_bytes() { return (int)sizeof(RouteArgs); }
HFM_API int hfm_route_bwd_args_bytes() { return (int)sizeof(RouteBwdArgs); }

// ------------------------------------------------------------------ exchange
// One wave per token, 16 bytes per lane and turn, a row's last elements (fewer than 16 bytes) one by one;
// a token's row is read once for all its slots (dispatch, combine_bwd), or its slots' rows summed in
// order (combine, dispatch_bwd).  Bound by the rows' bytes.  A 16-byte access of global memory may start at
// any element: rows of an odd width take the same accesses as aligned ones (10007 rows of 313 floats with
// 4 slots, the four exchanges: 88 us, 95 with single elements, 3 TB/s; 16384 rows of 1248 bf16 with 2 slots: 118
// us, 4.2 TB/s).
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
template <typename T, int V>
__device__ __forceinline__ void row_load(const T* p, float (&f)[V]) {
  typename RowVec<T, V>::type v = *reinterpret_cast<const typename RowVec<T, V>::type*>(p);
#pragma unroll
  for (int i = 0; i < V; ++i) f[i] = (float)v[i];
}
template <typename T, int V>
__device__ __forceinline__ void row_store(T* p, const float (&f)[V]) {
  typename RowVec<T, V>::type v;
#pragma unroll
  for (int i = 0; i < V; ++i) v[i] = (T)f[i];
  *reinterpret_cast<typename RowVec<T, V>::type*>(p) = v;
}

enum { EX_DISPATCH = 0, EX_DISPATCH_BWD = 1, EX_COMBINE = 2, EX_COMBINE_BWD = 3 };

// Columns c .. c + V - 1 of token t's rows.
template <typename T, int V, int K, int MODE>
__device__ __forceinline__ void exchange_cols(const ExchArgs& a, int t, int c, const int (&p)[K], const float (&w)[K],
                                              float (&dot)[K]) {
  const T* A = reinterpret_cast<const T*>(a.a);
  const T* B = reinterpret_cast<const T*>(a.b);
  T* O = reinterpret_cast<T*>(a.out);
  if (MODE == EX_DISPATCH) {
    typedef typename RowVec<T, V>::type vec;
    const vec v = *reinterpret_cast<const vec*>(A + (size_t)t * a.lda + c);
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (p[j] >= 0) *reinterpret_cast<vec*>(O + (size_t)p[j] * a.ldo + c) = v;
  } else if (MODE == EX_COMBINE_BWD) {
    float g[V], y[K][V];
    row_load<T, V>(A + (size_t)t * a.lda + c, g);
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (p[j] >= 0) row_load<T, V>(B + (size_t)p[j] * a.ldb + c, y[j]);
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (p[j] >= 0) {
        float d[V];
#pragma unroll
        for (int i = 0; i < V; ++i) {
          d[i] = w[j] * g[i];
          dot[j] = fmaf(g[i], y[j][i], dot[j]);
        }
        row_store<T, V>(O + (size_t)p[j] * a.ldo + c, d);
      }
  } else {
    float s[V], y[K][V];
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] = 0.f;
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (p[j] >= 0) row_load<T, V>(A + (size_t)p[j] * a.lda + c, y[j]);
#pragma unroll
    for (int j = 0; j < K; ++j)
      if (p[j] >= 0) {
#pragma unroll
        for (int i = 0; i < V; ++i) s[i] = MODE == EX_COMBINE ? fmaf(w[j], y[j][i], s[i]) : s[i] + y[j][i];
      }
    row_store<T, V>(O + (size_t)t * a.ldo + c, s);
  }
}

template <typename T, int K, int MODE>
__global__ void __launch_bounds__(256) exchange_kernel(ExchArgs a) {
  constexpr int V = 16 / sizeof(T);
  const int lane = threadIdx.x & 63;
  const int t = blockIdx.x * 4 + (threadIdx.x >> 6);
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
  for (int c = lane * V; c < D16; c += 64 * V) exchange_cols<T, V, K, MODE>(a, t, c, p, w, dot);
  if (D16 + lane < a.D) exchange_cols<T, 1, K, MODE>(a, t, D16 + lane, p, w, dot);
  if (MODE == EX_COMBINE_BWD) {
#pragma unroll
    for (int j = 0; j < K; ++j) {
      for (int d = 32; d; d >>= 1) dot[j] += __shfl_xor(dot[j], d);
      if (lane == 0 && j < a.k) a.dweight[(size_t)t * a.k + j] = p[j] >= 0 ? dot[j] : 0.f;
    }
  }
}

template <typename T, int MODE>
static void exchange_k(const ExchArgs& a, hipStream_t st) {
  const dim3 grid((a.T + 3) / 4), blk(256);
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
