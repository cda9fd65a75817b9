// Grouped products: one layer of every expert over its own rows.  Rows are sorted by expert, expert
// e has rows offs[e] .. offs[e + 1) (device memory: no host synchronization, ragged and empty groups
// allowed); rows behind offs[E] are not touched.
//
//   group_nt     out[p, n] = epi(sum_k A[row(p), k] B[e, n, k])      A, B bf16, K-contiguous
//                forward:  A = x (row(p) = p, or src[p] / top_k: the sorted slot's token), B = w,
//                          epi = + bias[e, n], relu
//                gradient: A = dz, B = w^T, epi = * scale, masked where the layer input is not > 0
//                          (the input in bf16 or as 8-bit codes)
//   group_wgrad  dw[e, n, k] = sum_p dz[p, n] x[row(p), k],  db[e, n] = sum_p dz[p, n]    (fp32)
//                x in bf16, or 8-bit codes with one scale per 32 columns (act8.h)
//
// A workgroup finds its expert by a scan over the group sizes in its own registers.  Accumulation is
// fp32 on MFMA; nothing is summed by atomics.
#include "act8.h"

struct GroupNtArgs {
  const bf16* a;           // [rows, K], row stride lda
  const bf16* b;           // [E, N, K], row stride ldb, expert stride es
  const float* bias;       // [E, N] or null
  const void* mask;        // null, bf16 [S, N] or codes [S, N], row stride ldm
  void* out;               // [S, N], row stride ldo, bf16 or fp32
  const int* offs;         // [E + 1]
  const int* src;          // [S] or null
  long lda, ldb, es, ldm, ldo;
  int S, rows, K, N, E, top_k, relu, mask8, out_f32;
  float scale;
};

struct GroupWgArgs {
  const bf16* dz;          // [S, N], row stride ldz
  const void* x;           // bf16 or codes [rows, K], row stride ldx
  const uint8_t* xs;       // scales [rows, ceil(K / 32)] (codes), else null
  const int* offs;
  const int* src;
  float* dw;               // [E, N, K]
  float* db;               // [E, N] or null
  float* ws;               // [ns, E, N, K] + [ns, E, N] (ns > 1)
  long ldz, ldx;
  int S, rows, K, N, E, top_k, ns;
};

// The offsets are the caller's device data: whatever they hold, no row outside [0, S) is touched.
__device__ __forceinline__ void group_rows(const int* offs, int e, int S, int& lo, int& hi) {
  lo = min(max(offs[e], 0), S);
  hi = min(max(offs[e + 1], lo), S);
}

// Row tile `tm` (of BM rows) over all groups in order: its expert, first row and the group's end.
template <int BM>
__device__ __forceinline__ bool group_find(const int* offs, int E, int S, int tm, int& e, int& r0, int& r1) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    int lo = 0, hi = 0;
    if (e0 + lane < E) group_rows(offs, e0 + lane, S, lo, hi);
    const int n = (hi - lo + BM - 1) / BM;
    int inc = n;
    for (int d = 1; d < 64; d <<= 1) {
      const int u = __shfl_up(inc, d);
      if (lane >= d) inc += u;
    }
    const unsigned long long past = __ballot(run + inc > tm);
    if (past) {
      const int l = __ffsll(past) - 1;
      e = e0 + l;
      r0 = __shfl(lo, l) + (tm - run - __shfl(inc - n, l)) * BM;
      r1 = __shfl(hi, l);
      e = __builtin_amdgcn_readfirstlane(e);
      r0 = __builtin_amdgcn_readfirstlane(r0);
      r1 = __builtin_amdgcn_readfirstlane(r1);
      return true;
    }
    run += __shfl(inc, 63);
  }
  return false;
}

// the row of x behind sorted place p, or -1 (a slot that is none of the rows reads as zeros)
__device__ __forceinline__ int group_row(const int* src, int p, int rows, int top_k) {
  if (!src) return p;
  const int s = src[p];
  const int r = s / top_k;
  return s >= 0 && r < rows ? r : -1;
}

// 8 elements of a row from column c, zeros past n (VEC: 16-byte aligned, n a multiple of 8)
template <bool VEC>
__device__ __forceinline__ bf16x8 load8_bf(const bf16* row, int c, int n) {
  bf16x8 v = {};
  if (!row || c >= n) return v;
  if (VEC) return *reinterpret_cast<const bf16x8*>(row + c);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c + j < n) v[j] = row[c + j];
  return v;
}
template <bool VEC>
__device__ __forceinline__ uint2 load8_code(const uint8_t* row, int c, int n) {
  uint2 v = make_uint2(0, 0);
  if (!row || c >= n) return v;
  if (VEC) return *reinterpret_cast<const uint2*>(row + c);
#pragma unroll
  for (int j = 0; j < 8; ++j)
    if (c + j < n) {
      const uint32_t b = row[c + j];
      if (j < 4) v.x |= b << (8 * j);
      else v.y |= b << (8 * (j - 4));
    }
  return v;
}

// ------------------------------------------------------------------ NT product, 128 x 128 tile
// 256 threads = 4 waves of 64 x 64 outputs (4 x 4 MFMA 16x16x32), 64-deep steps through two LDS
// buffers of 32 KB: the next step's 16-byte row chunks are in registers while this one multiplies.
// LDS image: rows of 64 elements (128 B), 16-byte chunk c of row r at c ^ ((r >> 1) & 7).
constexpr int GN_B = 128, GN_K = 64, GN_PANEL = GN_B * GN_K * 2;

template <bool VEC>
__global__ void __launch_bounds__(256) group_nt_kernel(GroupNtArgs g, int tiles_n) {
  __shared__ __attribute__((aligned(16))) char smem[4 * GN_PANEL];
  int e, r0, r1;
  if (!group_find<GN_B>(g.offs, g.E, g.S, blockIdx.x / tiles_n, e, r0, r1)) return;
  const int n0 = (blockIdx.x % tiles_n) * GN_B;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  const int fr = lane & 15, fq = lane >> 4;
  // staging: chunk tid & 7 of rows (tid >> 3) + 32 i
  const int ch = tid & 7, sr = tid >> 3;
  const bf16* pa[4];
  const bf16* pb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    const int p = r0 + sr + 32 * i, n = n0 + sr + 32 * i;
    const int row = p < r1 ? group_row(g.src, p, g.rows, g.top_k) : -1;
    pa[i] = row >= 0 ? g.a + (size_t)row * g.lda : nullptr;
    pb[i] = n < g.N ? g.b + (size_t)e * g.es + (size_t)n * g.ldb : nullptr;
  }
  f32x4 acc[4][4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  bf16x8 ra[4], rb[4];
  auto fetch = [&](int k0) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      ra[i] = load8_bf<VEC>(pa[i], k0 + ch * 8, g.K);
      rb[i] = load8_bf<VEC>(pb[i], k0 + ch * 8, g.K);
    }
  };
  auto stage = [&](int buf) {
    char* s = smem + buf * 2 * GN_PANEL;
#pragma unroll
    for (int i = 0; i < 4; ++i) {
      const int r = sr + 32 * i, o = r * 128 + ((ch ^ ((r >> 1) & 7)) << 4);
      *reinterpret_cast<bf16x8*>(s + o) = ra[i];
      *reinterpret_cast<bf16x8*>(s + GN_PANEL + o) = rb[i];
    }
  };
  const int nt = (g.K + GN_K - 1) / GN_K;
  const int sw = (fr >> 1) & 7;
  if (nt > 0) {
    fetch(0);
    stage(0);
  }
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) fetch((t + 1) * GN_K);
    const char* s = smem + (t & 1) * 2 * GN_PANEL;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8 fa[4], fb[4];
      const int c = ((ks * 4 + fq) ^ sw) << 4;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        fa[i] = *reinterpret_cast<const bf16x8*>(s + (wr + i * 16 + fr) * 128 + c);
        fb[i] = *reinterpret_cast<const bf16x8*>(s + GN_PANEL + (wc + i * 16 + fr) * 128 + c);
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
    }
    if (t + 1 < nt) stage((t + 1) & 1);
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + wc + j * 16 + fr;
    if (n >= g.N) continue;
    const float bias = g.bias ? g.bias[(size_t)e * g.N + n] : 0.f;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int p = r0 + wr + i * 16 + fq * 4 + q;
        if (p >= r1) continue;
        float v = acc[i][j][q] * g.scale + bias;
        if (g.relu && v < 0.f) v = 0.f;        // (NaN stays)
        if (g.mask) {
          const size_t m = (size_t)p * g.ldm + n;
          const bool on = g.mask8 ? a8_positive(reinterpret_cast<const uint8_t*>(g.mask)[m])
                                  : bf2f(reinterpret_cast<const bf16*>(g.mask)[m]) > 0.f;
          if (!on) v = 0.f;
        }
        const size_t o = (size_t)p * g.ldo + n;
        if (g.out_f32) reinterpret_cast<float*>(g.out)[o] = v;
        else reinterpret_cast<bf16*>(g.out)[o] = f2bf(v);
      }
  }
}

// 8 neighbouring outputs of row p from column n: mask, rounding, store (vec: 16-byte aligned rows of
// the output and the mask, N a multiple of 8)
__device__ __forceinline__ void group_store8(const GroupNtArgs& g, int p, int n, const float (&v)[8], int vec) {
  const size_t o = (size_t)p * g.ldo + n, m = (size_t)p * g.ldm + n;
  if (vec) {
    float w[8];
    if (g.mask && g.mask8) {
      const uint2 c = *reinterpret_cast<const uint2*>(reinterpret_cast<const uint8_t*>(g.mask) + m);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = a8_positive(((j < 4 ? c.x : c.y) >> (8 * (j & 3))) & 0xFFu) ? v[j] : 0.f;
    } else if (g.mask) {
      const bf16x8 h = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const bf16*>(g.mask) + m);
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = bf2f(h[j]) > 0.f ? v[j] : 0.f;
    } else {
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = v[j];
    }
    if (g.out_f32) {
      float* d = reinterpret_cast<float*>(g.out) + o;
      *reinterpret_cast<f32x4*>(d) = f32x4{w[0], w[1], w[2], w[3]};
      *reinterpret_cast<f32x4*>(d + 4) = f32x4{w[4], w[5], w[6], w[7]};
    } else {
      bf16x8 d;
#pragma unroll
      for (int j = 0; j < 8; ++j) d[j] = f2bf(w[j]);
      *reinterpret_cast<bf16x8*>(reinterpret_cast<bf16*>(g.out) + o) = d;
    }
    return;
  }
#pragma unroll
  for (int j = 0; j < 8; ++j) {
    if (n + j >= g.N) break;
    float w = v[j];
    if (g.mask) {
      const bool on = g.mask8 ? a8_positive(reinterpret_cast<const uint8_t*>(g.mask)[m + j])
                              : bf2f(reinterpret_cast<const bf16*>(g.mask)[m + j]) > 0.f;
      if (!on) w = 0.f;
    }
    if (g.out_f32) reinterpret_cast<float*>(g.out)[o + j] = w;
    else reinterpret_cast<bf16*>(g.out)[o + j] = f2bf(w);
  }
}

// ------------------------------------------------------------------ 256 x 256 ping-pong products
// 512 threads = 8 waves in two groups of 4 (group g owns rows g * 128 .., wave c of a group columns
// c * 64 ..: 8 x 4 MFMA 16x16x32 tiles, 128 accumulators).  Every SIMD hosts one wave of each group and
// the groups run one barrier apart: between two barriers one group reads the fragments of its next
// phase from LDS and stages the next step by LDS-DMA while the other group's 16 MFMAs run.  A 64-deep
// step is 4 phases of one 64 x 32 output quadrant, in the order (A0,B0) (A0,B1) (A1,B1) (A1,B0), so a
// phase reads only the half that changes.  Staging of step t + 1 goes into the other buffer: group 1 in
// its load slots 0-2, group 0 in 1-3 (the buffer's last reads retire in group 1's last compute slot of
// step t - 1, which is group 0's load slot 0); each wave waits for its own DMA once per step, before
// the barrier that publishes the step.
// LDS: 2 buffers x (A 32 KB + B 32 KB).
constexpr int GP_B = 256, GP_K = 64, GP_THREADS = 512;
constexpr int GP_PANEL = GP_B * GP_K * 2, GP_BUF = 2 * GP_PANEL;

constexpr int GP_MIN_TILES = 128;
__device__ __attribute__((aligned(16))) uint32_t g_zero16[4];      // the source of padding chunks

__device__ __forceinline__ void dma16(const void* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// One step's 4 phases on buffers `pa` / `pb`.  load_a(half), load_b(half) read fragments, stage(slot)
// is called in this group's three staging slots (0 .. 2) of the step, wait() once before it ends.
template <typename LA, typename LB, typename ST, typename MM>
__device__ __forceinline__ void pp_step(int grp, LA load_a, LB load_b, ST stage, MM mma) {
#pragma unroll
  for (int q = 0; q < 4; ++q) {
    const int qa = (q == 0 || q == 1) ? 0 : 1, qb = (q == 0 || q == 3) ? 0 : 1;
    if (q == 3 && grp == 1) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    if (q == 0 || q == 2) load_a(qa);
    load_b(qb);
    stage(q - (grp == 0 ? 1 : 0));
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("" ::: "memory");          // (no access moves over a barrier)
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_setprio(1);
    mma(q, qa, qb);
    __builtin_amdgcn_s_setprio(0);
    if (q == 3 && grp == 0) asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
    __builtin_amdgcn_s_barrier();
    asm volatile("" ::: "memory");
    __builtin_amdgcn_sched_barrier(0);
  }
}

// block b of n -> position in an order where each XCD (blocks go round the 8 of them) has a run of
// neighbouring tiles, which share operand panels in its L2
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int xcd = b & 7, q8 = n >> 3, rr = n & 7;
  return (xcd < rr ? xcd * (q8 + 1) : rr * (q8 + 1) + (xcd - rr) * q8) + (b >> 3);
}

// A wave's 128 x 64 outputs leave through its 16 KB of LDS, 64 rows a pass, so that a lane holds 8
// neighbouring columns of a row: emit(row in the block, first column in the block, 8 values).
template <typename F>
__device__ __forceinline__ void pp_emit(const f32x4 (&acc)[8][4], char* img, int lane, F emit) {
  // (the lane hidden from the optimizer: in a loop over tiles it would otherwise keep the image's
  // addresses in registers through the product, which has none left)
  asm volatile("" : "+v"(lane));
  const int fr = lane & 15, fq = lane >> 4;
  auto wsync = [] {
    __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
    __builtin_amdgcn_wave_barrier();
    __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
  };
  // rows of 64 floats; 16-byte chunk c of row r at chunk c ^ (r & 15)
  auto off = [](int r, int c) { return r * 256 + ((((c >> 2) ^ (r & 15))) << 4) + (c & 3) * 4; };
#pragma unroll
  for (int p = 0; p < 2; ++p) {
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j)
#pragma unroll
        for (int k = 0; k < 4; ++k)
          *reinterpret_cast<float*>(img + off(i * 16 + fq * 4 + k, j * 16 + fr)) = acc[p * 4 + i][j][k];
    wsync();
#pragma unroll 2
    for (int it = 0; it < 8; ++it) {
      const int r = it * 8 + (lane >> 3), c = (lane & 7) * 8;
      const f32x4 a = *reinterpret_cast<const f32x4*>(img + off(r, c));
      const f32x4 b = *reinterpret_cast<const f32x4*>(img + off(r, c + 4));
      const float v[8] = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
      emit(p * 64 + r, c, v);
    }
    wsync();
  }
}

// ---- NT: rows of A and B are K-contiguous, LDS image as in the 128 x 128 kernel.  K a multiple of 8;
// the last step's chunks past K come from the zero source.
__global__ void __launch_bounds__(GP_THREADS, 1) group_nt_pp_kernel(GroupNtArgs g, int tiles_n, int ovec) {
  __shared__ __attribute__((aligned(16))) char smem[2 * GP_BUF];
  const int tile = xcd_order(blockIdx.x, gridDim.x);
  int e, r0, r1;
  if (!group_find<GP_B>(g.offs, g.E, g.S, tile / tiles_n, e, r0, r1)) return;
  const int n0 = (tile % tiles_n) * GP_B;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int grp = wave >> 2, wc = wave & 3;
  const int fr = lane & 15, fq = lane >> 4, swz = (fr >> 1) & 7;
  const int la[2] = {(grp * 128 + fr) * 128 + ((fq ^ swz) << 4), (grp * 128 + fr) * 128 + (((4 + fq) ^ swz) << 4)};
  const int lb[2] = {(wc * 64 + fr) * 128 + ((fq ^ swz) << 4), (wc * 64 + fr) * 128 + (((4 + fq) ^ swz) << 4)};
  // staging pieces of 8 rows x 128 B: 4 of A and 4 of B per wave.  Rows past the group's end and
  // columns past N read the last one (their outputs are not stored).
  const bf16* src[8];
  int ck[8];
#pragma unroll
  for (int p = 0; p < 8; ++p) {
    const int r = (wave * 4 + (p & 3)) * 8 + (lane >> 3);
    ck[p] = ((lane & 7) ^ ((r >> 1) & 7)) * 8;
    if (p < 4) {
      const int row = max(group_row(g.src, min(r0 + r, r1 - 1), g.rows, g.top_k), 0);
      src[p] = g.a + (size_t)row * g.lda + ck[p];
    } else {
      src[p] = g.b + (size_t)e * g.es + (size_t)min(n0 + r, g.N - 1) * g.ldb + ck[p];
    }
  }
  const int nt = (g.K + GP_K - 1) / GP_K;
  const bool ragged = (g.K & (GP_K - 1)) != 0;
  auto piece = [&](int p, char* buf, int t) {
    const void* s = src[p] + t * GP_K;
    if (ragged && t == nt - 1 && t * GP_K + ck[p] >= g.K) s = g_zero16;
    dma16(s, buf + (p >= 4 ? GP_PANEL : 0) + (wave * 4 + (p & 3)) * 1024);
  };
  f32x4 acc[8][4];
#pragma unroll
  for (int i = 0; i < 8; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
  for (int p = 0; p < 8; ++p) piece(p, smem, 0);
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
  __builtin_amdgcn_s_barrier();
  __builtin_amdgcn_sched_barrier(0);
  if (grp == 1) {                         // the stagger: group 1 runs one slot behind
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
  }
  bf16x8 fa[4][2], fb[2][2];
  for (int t = 0; t < nt; ++t) {
    const char* pa = smem + (t & 1) * GP_BUF;
    const char* pb = pa + GP_PANEL;
    char* nxt = smem + ((t + 1) & 1) * GP_BUF;
    pp_step(
        grp,
        [&](int h) {
#pragma unroll
          for (int i = 0; i < 4; ++i)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
              fa[i][ks] = *reinterpret_cast<const bf16x8*>(pa + la[ks] + (h * 64 + i * 16) * 128);
        },
        [&](int h) {
#pragma unroll
          for (int j = 0; j < 2; ++j)
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
              fb[j][ks] = *reinterpret_cast<const bf16x8*>(pb + lb[ks] + (h * 32 + j * 16) * 128);
        },
        [&](int s) {
          if (t + 1 >= nt) return;
          if (s == 0)
            for (int p = 0; p < 3; ++p) piece(p, nxt, t + 1);
          if (s == 1)
            for (int p = 3; p < 6; ++p) piece(p, nxt, t + 1);
          if (s == 2)
            for (int p = 6; p < 8; ++p) piece(p, nxt, t + 1);
        },
        [&](int, int qa, int qb) {
#pragma unroll
          for (int ks = 0; ks < 2; ++ks)
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int j = 0; j < 2; ++j)
                acc[qa * 4 + i][qb * 2 + j] =
                    __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i][ks], fb[j][ks], acc[qa * 4 + i][qb * 2 + j], 0, 0, 0);
        });
  }
  if (grp == 0) __builtin_amdgcn_s_barrier();   // (every wave passes the same number of barriers)
  __syncthreads();
  // a source that is no slot: a row of zeros
  if (g.src) {
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        const int p = r0 + grp * 128 + i * 16 + fq * 4 + q;
        if (p < r1 && group_row(g.src, p, g.rows, g.top_k) < 0) {
#pragma unroll
          for (int j = 0; j < 4; ++j) acc[i][j][q] = 0.f;
        }
      }
  }
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int n = n0 + wc * 64 + j * 16 + fr;
    const float bias = g.bias && n < g.N ? g.bias[(size_t)e * g.N + n] : 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int q = 0; q < 4; ++q) {
        float v = acc[i][j][q] * g.scale + bias;
        if (g.relu && v < 0.f) v = 0.f;
        acc[i][j][q] = v;
      }
  }
  pp_emit(acc, smem + wave * 16384, lane, [&](int r, int c, const float (&v)[8]) {
    const int p = r0 + grp * 128 + r, n = n0 + wc * 64 + c;
    if (p < r1 && n < g.N) group_store8(g, p, n, v, ovec);
  });
}

HFM_API int hfm_group_nt(const GroupNtArgs* gp, hipStream_t st) {
  const GroupNtArgs g = *gp;
  if (g.S < 0 || g.K < 0 || g.N < 0 || g.E < 1 || g.top_k < 1) return (int)hipErrorInvalidValue;
  if (g.S == 0 || g.N == 0) return 0;
  const bool vec = ((uintptr_t)g.a | (uintptr_t)g.b) % 16 == 0 && g.K % 8 == 0 && g.lda % 8 == 0 && g.ldb % 8 == 0 &&
                   g.es % 8 == 0;
  const bool ovec = g.N % 8 == 0 && g.ldo % 8 == 0 && (uintptr_t)g.out % 16 == 0 &&
                    (!g.mask || (g.ldm % 8 == 0 && (uintptr_t)g.mask % (g.mask8 ? 8 : 16) == 0));
  if (vec && g.K >= GP_K) {
    const int tn = (g.N + GP_B - 1) / GP_B;
    const long blocks = (long)(g.S / GP_B + g.E) * tn;
    if (blocks >= GP_MIN_TILES && blocks <= 0x7FFFFFFFl) {
      hipLaunchKernelGGL(group_nt_pp_kernel, dim3((unsigned)blocks), dim3(GP_THREADS), 0, st, g, tn, ovec ? 1 : 0);
      HFM_LAUNCH_CHECK();
    }
  }
  const int tn = (g.N + GN_B - 1) / GN_B;
  const long blocks = (long)(g.S / GN_B + g.E) * tn;      // (each group adds less than one tile)
  if (blocks > 0x7FFFFFFFl) return (int)hipErrorInvalidValue;
  if (vec) hipLaunchKernelGGL(group_nt_kernel<true>, dim3((unsigned)blocks), dim3(256), 0, st, g, tn);
  else hipLaunchKernelGGL(group_nt_kernel<false>, dim3((unsigned)blocks), dim3(256), 0, st, g, tn);
  HFM_LAUNCH_CHECK();
}

// ------------------------------------------------------------------ weight gradient, 128 x 128 tile
// The reduction runs over rows, both operands are row-major: a thread takes an 8 x 8 block (8 rows
// p, 8 columns) into registers, transposes it (bf16 pairs, one byte permute per output word) and
// writes 8 chunks of 8 p-contiguous elements into the LDS image [column][64 p], which the MFMA
// fragments read like the NT kernel's.  256 threads = 128 blocks of dz + 128 of x per 64-row step.
// Image swizzle: 16-byte chunk m of row n at m ^ s(n), s(n) = ((n >> 1) ^ (n >> 3)) & 7: the 8 rows a
// thread writes and the 16 rows a fragment reads both spread over the banks.
__device__ __forceinline__ int wg_swz(int n) { return ((n >> 1) ^ (n >> 3)) & 7; }

// in[m] = 8 columns of row m  ->  out[c] = 8 rows of column c
__device__ __forceinline__ void transpose8(const uint4 (&in)[8], uint4 (&out)[8]) {
#pragma unroll
  for (int c2 = 0; c2 < 4; ++c2) {
    uint32_t lo[4], hi[4];
#pragma unroll
    for (int m2 = 0; m2 < 4; ++m2) {
      const uint32_t a = reinterpret_cast<const uint32_t*>(&in[2 * m2])[c2];
      const uint32_t b = reinterpret_cast<const uint32_t*>(&in[2 * m2 + 1])[c2];
      lo[m2] = __builtin_amdgcn_perm(b, a, 0x05040100u);
      hi[m2] = __builtin_amdgcn_perm(b, a, 0x07060302u);
    }
    out[2 * c2] = make_uint4(lo[0], lo[1], lo[2], lo[3]);
    out[2 * c2 + 1] = make_uint4(hi[0], hi[1], hi[2], hi[3]);
  }
}

template <bool VEC, bool X8>
__global__ void __launch_bounds__(256) group_wgrad_kernel(GroupWgArgs g, int tiles_n, int tiles_k) {
  __shared__ __attribute__((aligned(16))) char smem[4 * GN_PANEL];
  int bid = blockIdx.x;
  const int kt = bid % tiles_k;
  bid /= tiles_k;
  const int ntile = bid % tiles_n;
  bid /= tiles_n;
  const int e = bid % g.E, sp = bid / g.E;
  int lo, hi;
  group_rows(g.offs, e, g.S, lo, hi);
  // this split's rows: whole 64-row steps
  const int steps = (hi - lo + 63) / 64, per = (steps + g.ns - 1) / g.ns;
  const int p0 = lo + min(steps, sp * per) * 64, p1 = min(hi, lo + min(steps, (sp + 1) * per) * 64);
  const int n0 = ntile * GN_B, k0 = kt * GN_B;
  const int tid = threadIdx.x, wave = tid >> 6, lane = tid & 63;
  const int wr = (wave >> 1) * 64, wc = (wave & 1) * 64;
  const int fr = lane & 15, fq = lane >> 4;
  // staging block: waves 0, 1 take dz, waves 2, 3 take x; 16 column blocks x 8 row blocks
  const bool isx = wave >= 2;
  const int cb = lane & 15, mb = (wave & 1) * 4 + (lane >> 4);
  const int col = (isx ? k0 : n0) + cb * 8;
  const int sblk = (g.K + A8_BLOCK - 1) / A8_BLOCK;
  uint4 in[8];
  auto fetch = [&](int pbase) {
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const int p = pbase + mb * 8 + m;
      bf16x8 v = {};
      if (p < p1) {
        if (!isx) {
          v = load8_bf<VEC>(g.dz + (size_t)p * g.ldz, col, g.N);
        } else {
          const int row = group_row(g.src, p, g.rows, g.top_k);
          if (row >= 0) {
            if (X8) {
              const uint2 w = load8_code<VEC>(reinterpret_cast<const uint8_t*>(g.x) + (size_t)row * g.ldx, col, g.K);
              const float s = col < g.K ? a8_scale(g.xs[(size_t)row * sblk + col / A8_BLOCK]) : 0.f;
              float f[8];
              a8_unpack8(w, s, f);
#pragma unroll
              for (int j = 0; j < 8; ++j) v[j] = f2bf(f[j]);
            } else {
              v = load8_bf<VEC>(reinterpret_cast<const bf16*>(g.x) + (size_t)row * g.ldx, col, g.K);
            }
          }
        }
      }
      in[m] = *reinterpret_cast<const uint4*>(&v);
    }
  };
  auto stage = [&](int buf) {
    char* s = smem + buf * 2 * GN_PANEL + (isx ? GN_PANEL : 0);
    uint4 o[8];
    transpose8(in, o);
#pragma unroll
    for (int c = 0; c < 8; ++c) {
      const int n = cb * 8 + c;
      *reinterpret_cast<uint4*>(s + n * 128 + ((mb ^ wg_swz(n)) << 4)) = o[c];
    }
  };
  f32x4 acc[4][4], accb[4];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    accb[i] = f32x4{0.f, 0.f, 0.f, 0.f};
#pragma unroll
    for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
  }
  // db: one more product, with a column of ones (first k tile, waves of its first columns)
  const bool sum = g.db != nullptr && kt == 0 && wc == 0;
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = f2bf(1.f);
  const int nt = p1 > p0 ? (p1 - p0 + 63) / 64 : 0;
  if (nt > 0) {
    fetch(p0);
    stage(0);
  }
  for (int t = 0; t < nt; ++t) {
    __syncthreads();
    if (t + 1 < nt) fetch(p0 + (t + 1) * 64);
    const char* s = smem + (t & 1) * 2 * GN_PANEL;
#pragma unroll
    for (int ks = 0; ks < 2; ++ks) {
      bf16x8 fa[4], fb[4];
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int a = wr + i * 16 + fr, b = wc + i * 16 + fr;
        fa[i] = *reinterpret_cast<const bf16x8*>(s + a * 128 + (((ks * 4 + fq) ^ wg_swz(a)) << 4));
        fb[i] = *reinterpret_cast<const bf16x8*>(s + GN_PANEL + b * 128 + (((ks * 4 + fq) ^ wg_swz(b)) << 4));
      }
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], fb[j], acc[i][j], 0, 0, 0);
      if (sum) {
#pragma unroll
        for (int i = 0; i < 4; ++i) accb[i] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i], ones, accb[i], 0, 0, 0);
      }
    }
    if (t + 1 < nt) stage((t + 1) & 1);
  }
  const size_t en = (size_t)g.E * g.N;
  float* dw = g.ns > 1 ? g.ws + (size_t)sp * en * g.K : g.dw;
  float* db = g.ns > 1 ? g.ws + (size_t)g.ns * en * g.K + sp * en : g.db;
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int q = 0; q < 4; ++q) {
      const int n = n0 + wr + i * 16 + fq * 4 + q;
      if (n >= g.N) continue;
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        const int k = k0 + wc + j * 16 + fr;
        if (k < g.K) dw[((size_t)e * g.N + n) * g.K + k] = acc[i][j][q];
      }
      if (sum && fr == 0) db[(size_t)e * g.N + n] = accb[i][q];
    }
}

// dw = sum of the ns partial products in order (and db)
__global__ void __launch_bounds__(256) group_wgrad_sum_kernel(GroupWgArgs g) {
  const size_t nw = (size_t)g.E * g.N * g.K, nb = g.db ? (size_t)g.E * g.N : 0;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= nw + nb) return;
  const float* s = i < nw ? g.ws + i : g.ws + (size_t)g.ns * nw + (i - nw);
  const size_t step = i < nw ? nw : (size_t)g.E * g.N;
  float v = s[0];
  for (int q = 1; q < g.ns; ++q) v += s[q * step];
  (i < nw ? g.dw[i] : g.db[i - nw]) = v;
}

// ---- TN: the weight gradient on the ping-pong tile.  Both panels keep their global layout, [64 rows][256
// columns]; the fragments (8 rows of one column per lane) come from transposing LDS reads
// (ds_read_b64_tr_b16: a 16-lane group reads 4 rows x 16 columns, lane l gets column l's 4 rows).
// A panel row is 512 B, so a fragment's 16 rows would meet in the same banks: 32-byte granule c of row r
// lies at c ^ f(r), f(r) = (r & 3) | (r >> 1 & 4), which spreads them over all 8 granules of 256 B.
// 8-bit x: 16 codes a thread are loaded one step ahead, turned into bf16 times the block's scale
// (one conversion per pair, exact) and written into the same image.
//
// The work is cut evenly, not by tiles: `units` = 64-row steps of all tiles (a group without rows counts
// one per tile, which writes its zeros), tiles in expert order, and workgroup w takes the units from
// w U / W to (w + 1) U / W.  A tile within one workgroup goes straight to dw; a workgroup's first and last tile
// may be parts, which go to its two workspace tiles and are summed in row order by a second launch.
// Groups of any sizes thus load the CUs evenly (by whole tiles the fullest of 16 groups set the
// time), for at most 512 tiles of 256 KB.
constexpr int GW_SLAB = GP_B * GP_B + GP_B;      // floats of a workspace tile: dw part, db part

struct WgCut {
  long u0, u1;             // the workgroup's units
};
__device__ __forceinline__ WgCut wg_cut(long U, int W, int w) { return {U * w / W, U * (w + 1) / W}; }
__device__ __forceinline__ int wg_owner(long U, int W, long u) {        // the workgroup of unit u
  int w = (int)((u * W) / U);
  while (U * (w + 1) / W <= u) ++w;
  while (w > 0 && U * w / W > u) --w;
  return w;
}
__device__ __forceinline__ int wg_steps(const int* offs, int e, int S) {
  int lo, hi;
  group_rows(offs, e, S, lo, hi);
  return max(1, (hi - lo + GP_K - 1) / GP_K);
}
// a value that is the same in all lanes, into scalar registers
__device__ __forceinline__ long uni64(long v) {
  return (long)(((unsigned long long)(uint32_t)__builtin_amdgcn_readfirstlane((int)(v >> 32)) << 32) |
                (uint32_t)__builtin_amdgcn_readfirstlane((int)v));
}
// units of all groups, by every wave for itself
__device__ __forceinline__ long wg_units(const int* offs, int E, int S, int tiles) {
  const int lane = threadIdx.x & 63;
  long n = 0;
  for (int e = lane; e < E; e += 64) n += wg_steps(offs, e, S);
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  return uni64(n) * tiles;
}
// the expert of unit u, and its first unit
__device__ __forceinline__ void wg_find(const int* offs, int E, int S, int tiles, long u, int& e, long& first) {
  const int lane = threadIdx.x & 63;
  long run = 0;
  e = 0;
  first = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const long n = e0 + lane < E ? (long)wg_steps(offs, e0 + lane, S) * tiles : 0;
    long inc = n;
    for (int d = 1; d < 64; d <<= 1) {
      const long v = __shfl_up(inc, d);
      if (lane >= d) inc += v;
    }
    const unsigned long long past = __ballot(run + inc > u);
    if (past) {
      const int l = __ffsll(past) - 1;
      e = e0 + l;
      first = run + __shfl(inc - n, l);
      break;
    }
    run += __shfl(inc, 63);
  }
  e = __builtin_amdgcn_readfirstlane(e);
  first = uni64(first);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
typedef short s16x8 __attribute__((ext_vector_type(8)));
__device__ __forceinline__ bf16x8 tr_read(const char* p0, const char* p1) {
  typedef __attribute__((address_space(3))) s16x4* lp;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p0);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p1);
  const s16x8 v = {a[0], a[1], a[2], a[3], b[0], b[1], b[2], b[3]};
  return __builtin_bit_cast(bf16x8, v);
}

template <bool X8, bool GATHER>
__global__ void __launch_bounds__(GP_THREADS, 1) group_wgrad_pp_kernel(GroupWgArgs g, int tiles_n, int tiles_k, int ovec) {
  __shared__ __attribute__((aligned(16))) char smem[2 * GP_BUF];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int grp = wave >> 2, wc = wave & 3;
  const int fr = lane & 15, fq = lane >> 4;
  const int tiles = tiles_n * tiles_k;
  const int w = xcd_order(blockIdx.x, gridDim.x);
  const WgCut cut = wg_cut(wg_units(g.offs, g.E, g.S, tiles), gridDim.x, w);
  int e;
  long first;
  wg_find(g.offs, g.E, g.S, tiles, cut.u0, e, first);
  // fragment addresses: granule (base + i) ^ f(row) = f-and-base part ^ i, rows of fq and fr >> 2
  const int fsw = (fr >> 2) | ((fq & 1) << 2);
  const int rowoff = (fq * 8 + (fr >> 2)) * 512 + (fr & 3) * 8;
  int la = rowoff + ((grp * 8 ^ fsw) << 5), lb = rowoff + ((wc * 4 ^ fsw) << 5);
  // staging pieces: 2 rows of 512 B, 4 of each operand per wave.  Row 2 i + hi of the wave's 8 has
  // f = ((2 i + hi) & 3) | 4 (wave & 1), so the lane's 16-byte chunk is one column for even i and
  // that column ^ 32 for odd i.
  const int hi = lane >> 5, c16 = lane & 31;
  const int ce = (((c16 >> 1) ^ (hi | ((wave & 1) << 2))) * 2 + (c16 & 1)) * 8;
  const int sblk = (g.K + A8_BLOCK - 1) / A8_BLOCK;
  // 8-bit x: 16 codes at column xc of rows xr, xr + 32
  const int xr = threadIdx.x >> 4, xc = (threadIdx.x & 15) * 16;
  const int xo = GP_PANEL + xr * 512 + (((xc >> 4) ^ ((xr & 3) | ((xr >> 1) & 4))) << 5);
  bf16x8 ones;
#pragma unroll
  for (int j = 0; j < 8; ++j) ones[j] = f2bf(1.f);

  long u = cut.u0;
  while (u < cut.u1) {
    int steps = wg_steps(g.offs, e, g.S);
    while (u >= first + (long)steps * tiles) {      // the next group
      first += (long)steps * tiles;
      ++e;
      steps = wg_steps(g.offs, e, g.S);
    }
    int lo, hi_row;
    group_rows(g.offs, e, g.S, lo, hi_row);
    const int ti = (int)((u - first) / steps), s0 = (int)((u - first) % steps);
    const int s1 = (int)min((long)steps, s0 + (cut.u1 - u));
    const int n0 = (ti / tiles_k) * GP_B, k0 = (ti % tiles_k) * GP_B;
    const int p0 = lo + s0 * GP_K, p1 = min(hi_row, lo + s1 * GP_K);
    const int nt = p1 > p0 ? (p1 - p0 + GP_K - 1) / GP_K : 0;
    const bool ragged = ((p1 - p0) & (GP_K - 1)) != 0;
    const bool sum = g.db != nullptr && k0 == 0;
    f32x4 acc[8][4], accb[2];
#pragma unroll
    for (int i = 0; i < 8; ++i)
#pragma unroll
      for (int j = 0; j < 4; ++j) acc[i][j] = f32x4{0.f, 0.f, 0.f, 0.f};
    accb[0] = accb[1] = f32x4{0.f, 0.f, 0.f, 0.f};

    // columns past N or K read column 0 (their outputs are not stored), rows past p1 the zero source
    // (the last step only).  Scalar row base + the lane's 32-bit byte offset.
    const uint32_t ao0 = 2u * (uint32_t)(hi * (int)g.ldz + (n0 + ce < g.N ? n0 + ce : 0));
    const uint32_t ao1 = 2u * (uint32_t)(hi * (int)g.ldz + (n0 + (ce ^ 32) < g.N ? n0 + (ce ^ 32) : 0));
    const int bc0 = k0 + ce < g.K ? k0 + ce : 0, bc1 = k0 + (ce ^ 32) < g.K ? k0 + (ce ^ 32) : 0;
    const bool xin = k0 + xc < g.K;
    int xrow[4];                                       // GATHER: x rows of the next step's pieces (-1: zeros)
    uint4 cd[2];
    uint32_t cs[2];
    auto piece_a = [&](int i, char* buf, int t) {
      const int p = p0 + t * GP_K + wave * 8 + 2 * i;
      const void* s = reinterpret_cast<const char*>(g.dz + (size_t)p * g.ldz) + ((i & 1) ? ao1 : ao0);
      if (ragged && t == nt - 1 && p + hi >= p1) s = g_zero16;
      dma16(s, buf + (wave * 4 + i) * 1024);
    };
    auto rows_of = [&](int t) {
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const int p = p0 + t * GP_K + wave * 8 + 2 * i + hi;
        xrow[i] = p < p1 ? group_row(g.src, p, g.rows, g.top_k) : -1;
      }
    };
    auto piece_b = [&](int i, char* buf, int t) {
      const bf16* xb = reinterpret_cast<const bf16*>(g.x);
      const void* s;
      if (GATHER) {
        s = xrow[i] >= 0 ? (const void*)(xb + (size_t)(uint32_t)xrow[i] * g.ldx + ((i & 1) ? bc1 : bc0)) : (const void*)g_zero16;
      } else {
        const int p = p0 + t * GP_K + wave * 8 + 2 * i;
        s = reinterpret_cast<const char*>(xb + (size_t)p * g.ldx) + 2u * (uint32_t)(hi * (int)g.ldx + ((i & 1) ? bc1 : bc0));
        if (ragged && t == nt - 1 && p + hi >= p1) s = g_zero16;
      }
      dma16(s, buf + GP_PANEL + (wave * 4 + i) * 1024);
    };
    auto codes_of = [&](int t) {                       // X8: the codes of step t into registers
#pragma unroll
      for (int h = 0; h < 2; ++h) {
        const int pb = p0 + t * GP_K + 32 * h, p = pb + xr;
        cd[h] = make_uint4(0, 0, 0, 0);
        cs[h] = 127;
        if (p < p1 && xin) {
          const uint8_t* x8 = reinterpret_cast<const uint8_t*>(g.x) + k0;
          if (GATHER) {
            const int row = group_row(g.src, p, g.rows, g.top_k);
            if (row >= 0) {
              cd[h] = *reinterpret_cast<const uint4*>(x8 + (size_t)row * g.ldx + xc);
              cs[h] = g.xs[(size_t)row * sblk + (k0 + xc) / A8_BLOCK];
            }
          } else {
            cd[h] = *reinterpret_cast<const uint4*>(x8 + (size_t)pb * g.ldx + (uint32_t)(xr * (int)g.ldx + xc));
            cs[h] = g.xs[(size_t)pb * sblk + (uint32_t)(xr * sblk + (k0 + xc) / A8_BLOCK)];
          }
        }
      }
    };
    auto codes_to = [&](char* buf) {                   // X8: registers -> bf16 image
#pragma unroll
      for (int h = 0; h < 2; ++h) {                    // (row + 32: the same f)
        const float s = a8_scale(cs[h]);
        char* d = buf + xo + h * 32 * 512;
        *reinterpret_cast<uint4*>(d) = make_uint4(a8_pair_bf16<false>(cd[h].x, s), a8_pair_bf16<true>(cd[h].x, s),
                                                  a8_pair_bf16<false>(cd[h].y, s), a8_pair_bf16<true>(cd[h].y, s));
        *reinterpret_cast<uint4*>(d + 16) = make_uint4(a8_pair_bf16<false>(cd[h].z, s), a8_pair_bf16<true>(cd[h].z, s),
                                                       a8_pair_bf16<false>(cd[h].w, s), a8_pair_bf16<true>(cd[h].w, s));
      }
    };
    if (nt > 0) {
      if (X8) codes_of(0);
      else if (GATHER) rows_of(0);
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        piece_a(i, smem, 0);
        if (!X8) piece_b(i, smem, 0);
      }
      if (X8) {
        codes_to(smem);
        if (nt > 1) codes_of(1);
      } else if (GATHER && nt > 1) {
        rows_of(1);
      }
    }
    asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");
    __builtin_amdgcn_s_barrier();
    __builtin_amdgcn_sched_barrier(0);
    if (grp == 1) {
      __builtin_amdgcn_s_barrier();
      __builtin_amdgcn_sched_barrier(0);
    }
    bf16x8 fa[4][2], fb[2][2];
    for (int t = 0; t < nt; ++t) {
      const char* pa = smem + (t & 1) * GP_BUF;
      const char* pb = pa + GP_PANEL;
      char* nxt = smem + ((t + 1) & 1) * GP_BUF;
      asm volatile("" : "+v"(la), "+v"(lb));           // (12 addresses made by one xor each, not kept)
      pp_step(
          grp,
          [&](int h) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                const char* a = pa + (la ^ ((h * 4 + i) << 5)) + ks * 32 * 512;
                fa[i][ks] = tr_read(a, a + 4 * 512);
              }
          },
          [&](int h) {
#pragma unroll
            for (int j = 0; j < 2; ++j)
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                const char* b = pb + (lb ^ ((h * 2 + j) << 5)) + ks * 32 * 512;
                fb[j][ks] = tr_read(b, b + 4 * 512);
              }
          },
          [&](int s) {
            if (t + 1 >= nt) return;
            if (X8) {
              if (s == 0) codes_to(nxt);
              if (s == 1) {
                piece_a(0, nxt, t + 1);
                piece_a(1, nxt, t + 1);
                if (t + 2 < nt) codes_of(t + 2);
              }
              if (s == 2) {
                piece_a(2, nxt, t + 1);
                piece_a(3, nxt, t + 1);
              }
            } else {
              if (s == 0) {
                piece_a(0, nxt, t + 1);
                piece_a(1, nxt, t + 1);
                piece_a(2, nxt, t + 1);
              }
              if (s == 1) {
                piece_a(3, nxt, t + 1);
                piece_b(0, nxt, t + 1);
                piece_b(1, nxt, t + 1);
              }
              if (s == 2) {
                piece_b(2, nxt, t + 1);
                piece_b(3, nxt, t + 1);
                if (GATHER && t + 2 < nt) rows_of(t + 2);
              }
            }
          },
          [&](int q, int qa, int qb) {
#pragma unroll
            for (int ks = 0; ks < 2; ++ks)
#pragma unroll
              for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int j = 0; j < 2; ++j)
                  acc[qa * 4 + i][qb * 2 + j] =
                      __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[i][ks], fb[j][ks], acc[qa * 4 + i][qb * 2 + j], 0, 0, 0);
            // db: dz against a column of ones; wave c of a group takes row tiles 2 c, 2 c + 1
            if (sum && (q & 1) == 0 && (wc >> 1) == qa) {
#pragma unroll
              for (int ks = 0; ks < 2; ++ks) {
                if (wc & 1) {
                  accb[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[2][ks], ones, accb[0], 0, 0, 0);
                  accb[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[3][ks], ones, accb[1], 0, 0, 0);
                } else {
                  accb[0] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[0][ks], ones, accb[0], 0, 0, 0);
                  accb[1] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(fa[1][ks], ones, accb[1], 0, 0, 0);
                }
              }
            }
          });
    }
    if (grp == 0) __builtin_amdgcn_s_barrier();
    __syncthreads();
    // a whole tile goes to dw, a part to the workspace: slot 2 w if it is the workgroup's first, 2 w + 1
    // if it goes on in the next one
    const bool whole = s0 == 0 && s1 == steps;
    if (whole) {
      float* dw = g.dw + (size_t)e * g.N * g.K;
      pp_emit(acc, smem + wave * 16384, lane, [&](int r, int c, const float (&v)[8]) {
        const int n = n0 + grp * 128 + r, k = k0 + wc * 64 + c;
        if (n >= g.N || k >= g.K) return;
        float* d = dw + (size_t)n * g.K + k;
        if (ovec) {
          *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
          *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
        } else {
#pragma unroll
          for (int j = 0; j < 8; ++j)
            if (k + j < g.K) d[j] = v[j];
        }
      });
    } else {
      float* slab = g.ws + (size_t)(2 * w + (s0 > 0 ? 0 : 1)) * GW_SLAB;
      pp_emit(acc, smem + wave * 16384, lane, [&](int r, int c, const float (&v)[8]) {
        float* d = slab + (grp * 128 + r) * GP_B + wc * 64 + c;
        *reinterpret_cast<f32x4*>(d) = f32x4{v[0], v[1], v[2], v[3]};
        *reinterpret_cast<f32x4*>(d + 4) = f32x4{v[4], v[5], v[6], v[7]};
      });
    }
    if (sum && fr == 0) {
      float* db = whole ? g.db + (size_t)e * g.N : g.ws + (size_t)(2 * w + (s0 > 0 ? 0 : 1)) * GW_SLAB + GP_B * GP_B;
#pragma unroll
      for (int i = 0; i < 2; ++i)
#pragma unroll
        for (int q = 0; q < 4; ++q) {
          const int r = grp * 128 + (wc * 2 + i) * 16 + fq * 4 + q;
          if (!whole) db[r] = accb[i][q];
          else if (n0 + r < g.N) db[n0 + r] = accb[i][q];
        }
    }
    u += s1 - s0;
    __syncthreads();                      // (the next tile's staging reuses the images)
  }
}

// Tiles that two or more workgroups made: their parts in row order.  grid (tiles of an expert, E, 4
// quarters); the same cut as the product's.
__global__ void __launch_bounds__(256) group_wgrad_join_kernel(GroupWgArgs g, int tiles_n, int tiles_k, int W, int ovec) {
  const int tiles = tiles_n * tiles_k, ti = blockIdx.x, e = blockIdx.y;
  const int lane = threadIdx.x & 63;
  long before = 0, n = 0;
  for (int i = lane; i < g.E; i += 64) {
    const int s = wg_steps(g.offs, i, g.S);
    n += s;
    if (i < e) before += s;
  }
  for (int d = 32; d; d >>= 1) {
    n += __shfl_xor(n, d);
    before += __shfl_xor(before, d);
  }
  const long U = n * tiles;
  const int steps = wg_steps(g.offs, e, g.S);
  const long a = before * tiles + (long)ti * steps, b = a + steps - 1;
  const int w0 = wg_owner(U, W, a), w1 = wg_owner(U, W, b);
  if (w0 == w1) return;
  const int n0 = (ti / tiles_k) * GP_B, k0 = (ti % tiles_k) * GP_B;
  // the part that starts the tile is the last of w0 (slot 1), the others are the first of theirs
  auto slab = [&](int w) { return g.ws + (size_t)(2 * w + (w == w0 ? 1 : 0)) * GW_SLAB; };
  const int row0 = blockIdx.z * 64;
  for (int i = threadIdx.x; i < 64 * (GP_B / 4); i += 256) {
    const int r = row0 + i / (GP_B / 4), c = (i % (GP_B / 4)) * 4;
    if (n0 + r >= g.N || k0 + c >= g.K) continue;
    f32x4 v = *reinterpret_cast<const f32x4*>(slab(w0) + r * GP_B + c);
    for (int q = w0 + 1; q <= w1; ++q) v += *reinterpret_cast<const f32x4*>(slab(q) + r * GP_B + c);
    float* d = g.dw + ((size_t)e * g.N + n0 + r) * g.K + k0 + c;
    if (ovec) {
      *reinterpret_cast<f32x4*>(d) = v;
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + c + j < g.K) d[j] = v[j];
    }
  }
  if (g.db && k0 == 0 && threadIdx.x < 64 && n0 + row0 + threadIdx.x < g.N) {
    const int r = row0 + threadIdx.x;
    float v = slab(w0)[GP_B * GP_B + r];
    for (int q = w0 + 1; q <= w1; ++q) v += slab(q)[GP_B * GP_B + r];
    g.db[(size_t)e * g.N + n0 + r] = v;
  }
}

// Where the large tile is taken, and its workgroups (one per CU: 128 KB of LDS each): operands with 16-byte
// rows, and enough work for every CU (GP_MIN_UNITS steps each; below that the 128 x 128 tile's smaller
// pieces fill the chip better).
constexpr int GW_WGS = 256, GP_MIN_UNITS = 2;
static bool wgrad_big(const GroupWgArgs& g) {
  const bool x8 = g.xs != nullptr;
  if ((uintptr_t)g.dz % 16 || (uintptr_t)g.x % 16 || g.N % 8 || g.ldz % 8) return false;
  if (g.K % (x8 ? 16 : 8) || g.ldx % (x8 ? 16 : 8)) return false;
  if (g.ldz >= 1l << 25 || g.ldx >= 1l << 25) return false;      // (32-bit offsets within 64 rows)
  const long tiles = (long)((g.N + GP_B - 1) / GP_B) * ((g.K + GP_B - 1) / GP_B);
  return tiles * (g.S / GP_K) >= (long)GW_WGS * GP_MIN_UNITS;
}

// Splits of the rows: enough workgroups for two rounds of the 256 CUs while a split keeps 8 steps of
// 64 rows on average.
static int wgrad_splits(int S, int N, int K, int E) {
  const long tiles = (long)E * ((N + GN_B - 1) / GN_B) * ((K + GN_B - 1) / GN_B);
  if (tiles <= 0) return 1;
  long ns = 512 / tiles;
  const long most = (long)S / E / 512;
  if (ns > most) ns = most;
  if (ns > 32) ns = 32;
  return ns < 1 ? 1 : (int)ns;
}

HFM_API long hfm_group_wgrad_ws_floats(const GroupWgArgs* gp) {
  if (wgrad_big(*gp)) return 2l * GW_WGS * GW_SLAB;
  const int ns = wgrad_splits(gp->S, gp->N, gp->K, gp->E);
  return ns > 1 ? (long)ns * gp->E * gp->N * (gp->K + 1) : 0;
}

HFM_API int hfm_group_wgrad(const GroupWgArgs* gp, hipStream_t st) {
  GroupWgArgs g = *gp;
  if (g.S < 0 || g.K < 0 || g.N < 0 || g.E < 1 || g.top_k < 1) return (int)hipErrorInvalidValue;
  if (g.N == 0) return 0;
  if (wgrad_big(g)) {
    const int tn = (g.N + GP_B - 1) / GP_B, tk = (g.K + GP_B - 1) / GP_B;
    if (!g.ws || (uintptr_t)g.ws % 16 || g.E > 65535) return (int)hipErrorInvalidValue;
    const int ovec = g.K % 8 == 0 && (uintptr_t)g.dw % 16 == 0;
    const dim3 grid(GW_WGS), blk(GP_THREADS);
    if (g.xs && g.src) hipLaunchKernelGGL((group_wgrad_pp_kernel<true, true>), grid, blk, 0, st, g, tn, tk, ovec);
    else if (g.xs) hipLaunchKernelGGL((group_wgrad_pp_kernel<true, false>), grid, blk, 0, st, g, tn, tk, ovec);
    else if (g.src) hipLaunchKernelGGL((group_wgrad_pp_kernel<false, true>), grid, blk, 0, st, g, tn, tk, ovec);
    else hipLaunchKernelGGL((group_wgrad_pp_kernel<false, false>), grid, blk, 0, st, g, tn, tk, ovec);
    hipLaunchKernelGGL(group_wgrad_join_kernel, dim3(tn * tk, g.E, 4), dim3(256), 0, st, g, tn, tk, GW_WGS, ovec);
    HFM_LAUNCH_CHECK();
  }
  g.ns = wgrad_splits(g.S, g.N, g.K, g.E);
  if (g.ns > 1 && !g.ws) return (int)hipErrorInvalidValue;
  const bool x8 = g.xs != nullptr;
  const bool vec = (uintptr_t)g.dz % 16 == 0 && g.N % 8 == 0 && g.ldz % 8 == 0 && (uintptr_t)g.x % (x8 ? 8 : 16) == 0 &&
                   g.K % 8 == 0 && g.ldx % 8 == 0;
  const int tn = (g.N + GN_B - 1) / GN_B, tk = g.K > 0 ? (g.K + GN_B - 1) / GN_B : 1;
  const long blocks = (long)tn * tk * g.E * g.ns;
  if (blocks > 0x7FFFFFFFl) return (int)hipErrorInvalidValue;
  const dim3 grid((unsigned)blocks), blk(256);
  if (x8) {
    if (vec) hipLaunchKernelGGL((group_wgrad_kernel<true, true>), grid, blk, 0, st, g, tn, tk);
    else hipLaunchKernelGGL((group_wgrad_kernel<false, true>), grid, blk, 0, st, g, tn, tk);
  } else {
    if (vec) hipLaunchKernelGGL((group_wgrad_kernel<true, false>), grid, blk, 0, st, g, tn, tk);
    else hipLaunchKernelGGL((group_wgrad_kernel<false, false>), grid, blk, 0, st, g, tn, tk);
  }
  if (g.ns > 1) {
    const size_t n = (size_t)g.E * g.N * g.K + (g.db ? (size_t)g.E * g.N : 0);
    const size_t nb = (n + 255) / 256;
    if (nb > 0x7FFFFFFFull) return (int)hipErrorInvalidValue;
    hipLaunchKernelGGL(group_wgrad_sum_kernel, dim3((unsigned)nb), dim3(256), 0, st, g);
  }
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_group_nt_args_bytes() { return (int)sizeof(GroupNtArgs); }
HFM_API int hfm_group_wg_args_bytes() { return (int)sizeof(GroupWgArgs); }
