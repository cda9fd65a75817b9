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
#include <math.h>

#include <type_traits>

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
  void* ws;                // hfm_group_nt_ws_bytes
};

struct GroupWgArgs {
  const bf16* dz;          // [S, N], row stride ldz
  const void* x;           // bf16 or codes [rows, K], row stride ldx
  const uint8_t* xs;       // scales [rows, ceil(K / 32)] (codes), else null
  const int* offs;
  const int* src;
  float* dw;               // [E, N, K]
  float* db;               // [E, N] or null
  float* ws;               // hfm_group_wgrad_ws_floats
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

// The kernels that count the rows of all groups in one line do so in 32 bits.  Offsets that are not in order may give every
// second group all rows (a group ends where the next one begins), in units of 64 rows and 7 more a group, at most.
static bool groups_count(int E, int S) { return (E / 2 + 1l) * (S / 64 + 1l) + 7l * E < 1l << 31; }

// row tiles of all groups
template <int BM>
__device__ __forceinline__ int group_tiles(const int* offs, int E, int S) {
  const int lane = threadIdx.x & 63;
  int n = 0, lo, hi;
  for (int e = lane; e < E; e += 64) {
    group_rows(offs, e, S, lo, hi);
    n += (hi - lo + BM - 1) / BM;
  }
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  return __builtin_amdgcn_readfirstlane(n);
}

// the row of x behind sorted place p, or -1 (a slot that is none of the rows reads as zeros)
__device__ __forceinline__ int group_row(const int* src, int p, int rows, int top_k) {
  if (!src) return p;
  const int s = src[p];
  const int r = s / top_k;
  return s >= 0 && r < rows ? r : -1;
}

// 8 elements of a row of n from column c, zeros past n.  The access may start at any element (192 rows of 8 experts,
// 1249 -> 400: 97 us by single elements, 15 so).
typedef bf16 any_bf16x8 __attribute__((ext_vector_type(8), aligned(2)));
__device__ __forceinline__ bf16x8 load8_bf(const bf16* row, int c, int n) {
  bf16x8 v = {};
  if (!row || c >= n) return v;
  if (c + 8 <= n) return __builtin_bit_cast(bf16x8, *reinterpret_cast<const any_bf16x8*>(row + c));
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (c + j < n) v[j] = row[c + j];
  return v;
}
// The same in two halves, for many rows at the same columns: a load that ends with the row, and what moves the row's
// last elements to their place once all loads are under way (the loads of a last piece's elements would wait
// for the others: 3000 rows of 4 groups, 999 x 1001: 133 us, 72 so).  WHOLE: n is a multiple of 8, there is no
// second half (4096 rows of 4 groups, 512 x 512: 31 us, with it 46).
template <bool WHOLE>
__device__ __forceinline__ bf16x8 begin8_bf(const bf16* row, int c, int n) {
  bf16x8 v = {};
  if (!row || c >= n) return v;
  if (WHOLE || n >= 8) {
    return __builtin_bit_cast(bf16x8, *reinterpret_cast<const any_bf16x8*>(row + (WHOLE ? c : min(c, n - 8))));
  }
  return load8_bf(row, c, n);
}
__device__ __forceinline__ void end8_bf(bf16x8& v, int c, int n) {
  const int bits = (c + 8 - n) * 16;
  if (bits <= 0 || n < 8) return;
  typedef uint64_t u64x2 __attribute__((ext_vector_type(2)));
  u64x2 u = __builtin_bit_cast(u64x2, v);
  u[0] = bits < 64 ? u[0] >> bits | u[1] << (64 - bits) : bits < 128 ? u[1] >> (bits - 64) : 0;
  u[1] = bits < 64 ? u[1] >> bits : 0;
  v = __builtin_bit_cast(bf16x8, u);
}
template <bool WHOLE>
__device__ __forceinline__ uint64_t begin8_code(const uint8_t* row, int c, int n) {
  typedef uint64_t any8 __attribute__((aligned(1)));
  uint64_t v = 0;
  if (!row || c >= n) return v;
  if (WHOLE || n >= 8) return *reinterpret_cast<const any8*>(row + (WHOLE ? c : min(c, n - 8)));
#pragma unroll
  for (int j = 0; j < 7; ++j)
    if (c + j < n) v |= (uint64_t)row[c + j] << (8 * j);
  return v;
}
__device__ __forceinline__ void end8_code(uint64_t& v, int c, int n) {
  const int bits = (c + 8 - n) * 8;
  if (bits > 0 && n >= 8) v = bits < 64 ? v >> bits : 0;
}

// Rows of any alignment into rows of whole 16-byte chunks, zeros behind their ends (and in place of rows that are
// none), for the large tiles' LDS-DMA: a wave a row.  The copies cost the operands' bytes twice where the
// 128 x 128 tile takes up to ten times as long as the large one.
struct PadArgs {
  const char* from;        // row r at from + (r / per) * gs + (r % per) * lds, or at `map`'s row
  char* to;                // row r at to + r * ldd
  const int* map;          // sources as in group_row, or null
  long gs, lds, ldd, rows;
  int per, bytes, have, top_k;
};
__global__ void __launch_bounds__(256) group_pad_kernel(PadArgs a) {
  typedef uint32_t any16 __attribute__((ext_vector_type(4), aligned(1)));
  const long r = ((long)blockIdx.y * gridDim.x + blockIdx.x) * 4 + (threadIdx.x >> 6);
  if (r >= a.rows) return;
  const int row = group_row(a.map, a.map ? (int)r : 0, a.have, a.top_k);
  const char* from = a.map ? a.from + (size_t)max(row, 0) * a.lds
                           : a.from + (size_t)(r / a.per) * a.gs + (size_t)(r % a.per) * a.lds;
  char* to = a.to + (size_t)r * a.ldd;
  for (int c = (threadIdx.x & 63) * 16; c < a.ldd; c += 1024) {
    uint4 v = make_uint4(0, 0, 0, 0);
    if (row >= 0) {
      if (c + 16 <= a.bytes) {
        v = __builtin_bit_cast(uint4, *reinterpret_cast<const any16*>(from + c));
      } else {
        uint8_t b[16];
#pragma unroll
        for (int i = 0; i < 16; ++i) b[i] = c + i < a.bytes ? (uint8_t)from[c + i] : 0;
        __builtin_memcpy(&v, b, 16);
      }
    }
    *reinterpret_cast<uint4*>(to + c) = v;
  }
}
static void group_pad(const PadArgs& a, hipStream_t st) {
  const unsigned n = (unsigned)((a.rows + 3) / 4), row = 1u << 23;       // (a launch has less than 2^32 threads in x)
  hipLaunchKernelGGL(group_pad_kernel, dim3(n < row ? n : row, (n + row - 1) / row), dim3(256), 0, st, a);
}
constexpr long GROUP_PAD_MAX = 1l << 33;                   // (grid)
static long up16(long bytes) { return (bytes + 15) / 16 * 16; }

// One output of the NT product: scale, bias, relu (NaN stays), mask, rounding.
__device__ __forceinline__ void group_put(const GroupNtArgs& g, int p, int n, float acc, float bias) {
  float v = acc * g.scale + bias;
  if (g.relu && v < 0.f) v = 0.f;
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

// ------------------------------------------------------------------ NT product, 128 x 128 tile
// 256 threads = 4 waves of 64 x 64 outputs (4 x 4 MFMA 16x16x32), 64-deep steps through two LDS
// buffers of 32 KB: the next step's 16-byte row chunks are in registers while this one multiplies.
// LDS image: rows of 64 elements (128 B), 16-byte chunk c of row r at c ^ ((r >> 1) & 7).
constexpr int GN_B = 128, GN_K = 64, GN_PANEL = GN_B * GN_K * 2;

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
      ra[i] = load8_bf(pa[i], k0 + ch * 8, g.K);
      rb[i] = load8_bf(pb[i], k0 + ch * 8, g.K);
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
        if (p < r1) group_put(g, p, n, acc[i][j][q], bias);
      }
  }
}

// ------------------------------------------------------------------ NT product, few rows
// 32 x 32 outputs of a workgroup whose 8 waves share the reduction: wave w takes the 16-deep steps w, w + 8, ...
// (together they read 256 neighbouring bytes of a row), fragments straight from memory, 8 steps under way at
// once, and the 8 partial tiles are summed through LDS.  A request's rows leave a larger tile with a
// handful of workgroups that go through the whole reduction one after another: 192 rows, 8 experts,
// 1248 -> 400: 25 us by the 128 x 128 tile, 6.2 here.
constexpr int GS_B = 32, GS_WAVES = 8, GS_DEEP = 8;
__global__ void __launch_bounds__(GS_WAVES * 64) group_nt_few_kernel(GroupNtArgs g, int tiles_n) {
  typedef float f32x16 __attribute__((ext_vector_type(16)));
  __shared__ float part[GS_WAVES][GS_B][GS_B + 1];
  int e, r0, r1;
  if (!group_find<GS_B>(g.offs, g.E, g.S, blockIdx.x / tiles_n, e, r0, r1)) return;
  const int n0 = (blockIdx.x % tiles_n) * GS_B;
  const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, fr = lane & 31, fq = lane >> 5;
  const int row = r0 + fr < r1 ? group_row(g.src, r0 + fr, g.rows, g.top_k) : -1;
  const bf16* a = row >= 0 ? g.a + (size_t)row * g.lda : nullptr;
  const bf16* b = n0 + fr < g.N ? g.b + (size_t)e * g.es + (size_t)(n0 + fr) * g.ldb : nullptr;
  f32x16 acc = {};
  for (int k0 = wave * 16 + fq * 8; k0 - fq * 8 < g.K; k0 += GS_DEEP * GS_WAVES * 16) {
    bf16x8 fa[GS_DEEP], fb[GS_DEEP];
#pragma unroll
    for (int i = 0; i < GS_DEEP; ++i) {
      fa[i] = load8_bf(a, k0 + i * GS_WAVES * 16, g.K);
      fb[i] = load8_bf(b, k0 + i * GS_WAVES * 16, g.K);
    }
#pragma unroll
    for (int i = 0; i < GS_DEEP; ++i) acc = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[i], fb[i], acc, 0, 0, 0);
  }
#pragma unroll
  for (int q = 0; q < 16; ++q) part[wave][(q >> 2) * 8 + fq * 4 + (q & 3)][fr] = acc[q];
  __syncthreads();
  const int r = threadIdx.x >> 4, p = r0 + r;
#pragma unroll
  for (int i = 0; i < 2; ++i) {
    const int c = (threadIdx.x & 15) * 2 + i, n = n0 + c;
    float v = 0.f;
#pragma unroll
    for (int w = 0; w < GS_WAVES; ++w) v += part[w][r][c];
    if (p < r1 && n < g.N) group_put(g, p, n, v, g.bias ? g.bias[(size_t)e * g.N + n] : 0.f);
  }
}

// ------------------------------------------------------------------ 256 x 256 products
// 256 threads = 4 waves, one per SIMD, of 128 x 128 outputs (4 x 4 MFMA 32x32x16 tiles: 256 accumulators; 32
// cycles an MFMA leave room for the other instructions of the one wave).  The reduction runs in 32-deep steps
// through a ring of 4 LDS buffers (A 16 KB + B 16 KB each).  In step s a wave multiplies fragments that it read
// during step s - 1, reads those of step s + 1 and starts the LDS-DMA of step s + 3, spread between the MFMAs,
// so that no load is waited for: a fragment has 4 rounds of 128 cycles of MFMA or more to arrive, DMA two
// steps.  Row fragment i is replaced after its round; the 8 column fragments serve all rounds and are held
// twice.
//   Top of step s: the wave's own DMA of step s + 1 has landed; the barrier makes that true for all waves,
//   and buffer (s + 3) % 4 = (s - 1) % 4 free: its fragments were multiplied in step s - 1.
// A 128 x 128 block per wave reads 64 KB of fragments a step and CU and writes 32 KB: 768 cycles of LDS
// against 1024 of MFMA; 128 x 64 blocks (8 waves) need 1024 + 256.
typedef float f32x16 __attribute__((ext_vector_type(16)));
constexpr int GP_B = 256, GP_K = 32, GP_THREADS = 256;
constexpr int GP_PANEL = GP_B * GP_K * 2, GP_BUF = 2 * GP_PANEL, GP_RING = 4;

__device__ __attribute__((aligned(16))) uint32_t g_zero16[4];      // the source of padding chunks

__device__ __forceinline__ void dma16(const void* src, char* lds) {
  __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)src,
                                   (__attribute__((address_space(3))) void*)lds, 16, 0, 0);
}

// 16 bytes a lane from `base` + soff + voff, zeros where that lies at or past `bytes` (the buffer's own check)
__device__ __forceinline__ void dma16_buf(const void* base, uint32_t bytes, uint32_t voff, uint32_t soff, char* lds) {
  const __amdgpu_buffer_rsrc_t r = __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, (int)bytes, 0x00020000);
  __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)lds, 16, (int)voff, (int)soff, 0, 0);
}

// One step of a wave.  D: its DMA pieces per step.  stage(i): piece i of the step three ahead; load_a(i),
// load_b(j): fragments of the next step; PAR: which of the two sets of column fragments is multiplied.
// cs: where `take`, column sums of A (a lane's share: column lane & 31 of tile i).  Two bf16 an instruction: in
// every step they cost 90 us of 400 (16384 x 4096 x 4096), in a launch of their own 31, in one of 2 tiles_k steps
// 13.  The branch is in the assembly, where the compiler does not see it: its accumulators do not survive
// another block in the loop.
__device__ __forceinline__ void col_sums(float (&c)[4], const bf16x8 (&fa)[8], int take) {
  uint4 u[8];
#pragma unroll
  for (int r = 0; r < 8; ++r) u[r] = __builtin_bit_cast(uint4, fa[r]);
  asm volatile(
      "s_cmp_lg_u32 %36, 0\n\ts_cbranch_scc0 .Lskip%=\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %4\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %8\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %12\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %16\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %20\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %24\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %28\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %32\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %5\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %9\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %13\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %17\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %21\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %25\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %29\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %33\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %6\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %10\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %14\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %18\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %22\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %26\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %30\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %34\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %7\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %11\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %15\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %19\n\t"
      "v_dot2c_f32_bf16 %0, 0x3f803f80, %23\n\t" "v_dot2c_f32_bf16 %1, 0x3f803f80, %27\n\t"
      "v_dot2c_f32_bf16 %2, 0x3f803f80, %31\n\t" "v_dot2c_f32_bf16 %3, 0x3f803f80, %35\n\t"
      "s_nop 3\n.Lskip%=:"
      : "+v"(c[0]), "+v"(c[1]), "+v"(c[2]), "+v"(c[3])
      : "v"(u[0].x), "v"(u[0].y), "v"(u[0].z), "v"(u[0].w), "v"(u[1].x), "v"(u[1].y), "v"(u[1].z), "v"(u[1].w),
        "v"(u[2].x), "v"(u[2].y), "v"(u[2].z), "v"(u[2].w), "v"(u[3].x), "v"(u[3].y), "v"(u[3].z), "v"(u[3].w),
        "v"(u[4].x), "v"(u[4].y), "v"(u[4].z), "v"(u[4].w), "v"(u[5].x), "v"(u[5].y), "v"(u[5].z), "v"(u[5].w),
        "v"(u[6].x), "v"(u[6].y), "v"(u[6].z), "v"(u[6].w), "v"(u[7].x), "v"(u[7].y), "v"(u[7].z), "v"(u[7].w), "s"(take)
      : "scc");
}
// extra(k): what else the step does, after MFMA k (-1: before all); WAIT: the loads that may be in flight at its
// top, those issued after the DMA of the step after this one.
template <int NI, int D, int WAIT, int PAR, typename ST, typename LA, typename LB, typename EX>
__device__ __forceinline__ void mm_step(f32x16 (&acc)[NI][4], float (&cs)[NI], int take, bf16x8 (&fa)[2 * NI], bf16x8 (&fb)[2][8],
                                        ST stage, LA load_a, LB load_b, EX extra) {
  constexpr int NA = 2 * NI, c = PAR, n = c ^ 1;      // row fragment r: 16-deep half r / NI, rows 32 (r % NI) ..
  static_assert(NI >= 3 && NI <= 4 && D <= 2 * NA - 4, "a place for every load");
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(WAIT) : "memory");     // (the DMA of the step after next stays in flight)
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");          // (no access moves over the barrier)
  __builtin_amdgcn_sched_barrier(0);
  extra(-1);
#pragma unroll
  for (int k = 0; k < 4 * NA; ++k) {
    const int r = k >> 2, j = k & 3;
    acc[r % NI][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[r], fb[c][(r / NI) * 4 + j], acc[r % NI][j], 0, 0, 0);
    if (k == 3) col_sums(cs, fa, take);          // (row fragments are replaced after their rounds)
    // at most one load between two MFMAs: a wave issues an instruction every 4 cycles, an MFMA runs 32
    if (j == 0 && r > 0) fa[r - 1] = load_a(r - 1);
    if (j == 1 && r < 4) fb[n][2 * r] = load_b(2 * r);
    if (j == 2 && r < 4) fb[n][2 * r + 1] = load_b(2 * r + 1);
    if (j == 3 && r < D) stage(r);
    if (j == 1 && r >= 4 && NA + r - 4 < D) stage(NA + r - 4);
    if (k == 4 * NA - 1) fa[NA - 1] = load_a(NA - 1);
    extra(k);
    __builtin_amdgcn_sched_barrier(0);
  }
}

// The first three steps' DMA under way, the first step's fragments in registers.  (Where a step's top lets other loads
// be in flight too, there are none yet behind these: they have landed here.)
template <int NI, int D, int WAIT, typename ST, typename LA, typename LB>
__device__ __forceinline__ void mm_begin(bf16x8 (&fa)[2 * NI], bf16x8 (&fb)[2][8], ST stage, LA load_a, LB load_b) {
#pragma unroll
  for (int s = 0; s < GP_RING - 1; ++s)
#pragma unroll
    for (int i = 0; i < D; ++i) stage(i, s);
  asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(WAIT == D ? 2 * D : 0) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
#pragma unroll
  for (int i = 0; i < 8; ++i) fb[0][i] = load_b(i);
#pragma unroll
  for (int i = 0; i < 2 * NI; ++i) fa[i] = load_a(i);
}

// A whole reduction of ns steps.  stage(i, step): zeros from the step `ns` on (the loop runs on a pair of steps
// at a time and three steps ahead, without a branch: its registers do not survive one).
template <int NI, int D, int WAIT, typename ST, typename LA, typename LB, typename EX>
__device__ __forceinline__ void mm_loop(char* smem, int ns, f32x16 (&acc)[NI][4], float (&cs)[NI], int turn, int period, ST stage,
                                        LA load_a, LB load_b, EX extra) {
  bf16x8 fa[2 * NI], fb[2][8];
  mm_begin<NI, D, WAIT>(fa, fb, stage, [&](int i) { return load_a(i, smem); }, [&](int j) { return load_b(j, smem); });
  auto step = [&](auto PAR, int s) {
    const char* nb = smem + ((s + 1) & (GP_RING - 1)) * GP_BUF;
    const int take = __builtin_amdgcn_readfirstlane(turn == 0 ? 1 : 0);
    turn = __builtin_amdgcn_readfirstlane(turn == 0 ? period - 1 : turn - 1);
    mm_step<NI, D, WAIT, decltype(PAR)::value>(
        acc, cs, take, fa, fb, [&](int i) { stage(i, s + GP_RING - 1); }, [&](int i) { return load_a(i, nb); },
        [&](int j) { return load_b(j, nb); }, [&](int k) { extra(PAR, s, k); });
  };
  for (int s = 0; s < ns; s += 2) {
    step(std::integral_constant<int, 0>{}, s);
    step(std::integral_constant<int, 1>{}, s + 1);
  }
  asm volatile("s_waitcnt vmcnt(0) lgkmcnt(0)" ::: "memory");     // (nothing in flight into LDS)
}

// block b of n -> position in an order where each XCD (blocks go round the 8 of them) has a run of
// neighbouring tiles, which share operand panels in its L2
__device__ __forceinline__ int xcd_order(int b, int n) {
  const int xcd = b & 7, q8 = n >> 3, rr = n & 7;
  return (xcd < rr ? xcd * (q8 + 1) : rr * (q8 + 1) + (xcd - rr) * q8) + (b >> 3);
}

// Tile t of a rows x cols grid, in bands of GP_BAND rows walked column by column: the 32 CUs of an XCD then
// work on about 8 x 4 tiles, which share 12 panels (row by row, at 16 columns: 18, and the panels' way
// from the other side of the L2 sets the time).
constexpr int GP_BAND = 8;
__device__ __forceinline__ void band_tile(int t, int rows, int cols, int& r, int& c) {
  const int band = t / (GP_BAND * cols), r0 = band * GP_BAND, h = min(GP_BAND, rows - r0);
  const int i = t - r0 * cols;
  r = r0 + i % h;
  c = i / h;
}

// A wave's 128 x 128 fp32 outputs, straight from the accumulators (a lane holds rows 8 (q >> 2) + 4 (lane >> 5)
// + (q & 3) of column lane & 31 of a 32 x 32 tile: a store is two rows' 128 B): rows past `rows` and columns
// past `cols` are dropped by the buffer's end.  One wave per SIMD issues an instruction every 4 cycles,
// so the way through LDS to 16-byte stores cost more (9 us a tile of 256 x 256) than it saved.
constexpr uint32_t GP_FAR = 0x80000000u;                 // an offset past every buffer here
constexpr long GP_MAXLD = 1l << 21;                      // (128 rows of fp32 within 2^30 bytes)
__device__ __forceinline__ __amdgpu_buffer_rsrc_t out_rows(const void* base, uint32_t bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(const_cast<void*>(base), 0, __builtin_amdgcn_readfirstlane((int)bytes), 0x00020000);
}
__device__ __forceinline__ void mm_out_f32(const f32x16 (&acc)[4][4], float* base, int rows, int cols, int ld, int lane) {
  if (rows <= 0) return;
  const __amdgpu_buffer_rsrc_t o = out_rows(base, (uint32_t)min(rows, 128) * ld * 4u);
  const int fr = lane & 31, h = lane >> 5;
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = j * 32 + fr;
    const uint32_t at = c < cols ? (uint32_t)(h * 4 * ld + c) * 4u : GP_FAR;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
      for (int q = 0; q < 16; ++q)
        __builtin_amdgcn_raw_buffer_store_b32(__float_as_uint(acc[i][j][q]), o, (int)at,
                                              (i * 32 + (q >> 2) * 8 + (q & 3)) * ld * 4, 0);
  }
}

// The NT kernel's outputs: max(acc * scale + bias, floor) (floor 0: relu, -inf: none; NaN stays), masked,
// in fp32 as above, or in bf16 two columns a lane: the lanes of a column pair trade a row each
// (pack two rows, one lane swap, one byte permute), so that a store is four rows' 64 B.
// MASK 1: bf16 layer input, 2: its 8-bit codes; where that is not above zero the output is.
// OUT: 0 bf16 in column pairs, 1 fp32, 2 bf16 one by one (rows or masks of odd widths).
template <int NI, int MASK, int OUT>
__device__ __forceinline__ void mm_out_nt(const GroupNtArgs& g, const f32x16 (&acc)[NI][4], int e, int row0, int rows, int n0,
                                          int lane) {
  if (rows <= 0) return;
  constexpr bool ONE = OUT != 0;
  constexpr int ES = OUT == 1 ? 4 : 2, MS = MASK == 1 ? 2 : 1;
  const int fr = lane & 31, h = lane >> 5, odd = lane & 1;
  const int ldo = (int)g.ldo, ldm = (int)g.ldm, left = min(rows, 32 * NI);
  const __amdgpu_buffer_rsrc_t o = out_rows(reinterpret_cast<char*>(g.out) + (size_t)row0 * g.ldo * ES, (uint32_t)left * ldo * ES);
  const __amdgpu_buffer_rsrc_t mr =
      out_rows(reinterpret_cast<const char*>(g.mask) + (size_t)row0 * g.ldm * MS, (uint32_t)left * ldm * MS);
  const float lo = g.relu ? 0.f : -INFINITY;
  const uint32_t sel = odd ? 0x07060302u : 0x01000504u;
  constexpr int NQ = ONE ? 16 : 8;
  auto row_of = [](int i, int q) {
    const int k = ONE ? q : 2 * q;
    return i * 32 + (k >> 2) * 8 + (k & 3);
  };
  // a column block's mask, read while the one before it is written
  uint32_t m[2][NI][NQ];
  const int rr = ONE ? h * 4 : h * 4 + odd;
  auto mask_of = [&](int j) {
    if (MASK == 0) return;
    const int c = n0 + j * 32 + fr, cc = ONE ? c : c & ~1;
    const int mt = (int)(cc < g.N ? (uint32_t)(rr * ldm + cc) * MS : GP_FAR);
#pragma unroll
    for (int i = 0; i < NI; ++i)
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int at = row_of(i, q) * ldm * MS;
        if (MASK == 1) m[j & 1][i][q] = ONE ? (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(mr, mt, at, 0)
                                            : (uint32_t)__builtin_amdgcn_raw_buffer_load_b32(mr, mt, at, 0);
        if (MASK == 2) m[j & 1][i][q] = ONE ? (uint32_t)__builtin_amdgcn_raw_buffer_load_b8(mr, mt, at, 0)
                                            : (uint32_t)__builtin_amdgcn_raw_buffer_load_b16(mr, mt, at, 0);
      }
  };
  float bias[4];
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = n0 + j * 32 + fr;
    bias[j] = g.bias && c < g.N ? g.bias[(size_t)e * g.N + c] : 0.f;
  }
  mask_of(0);
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    const int c = n0 + j * 32 + fr;
    const int cc = ONE ? c : c & ~1;
    const uint32_t at = cc < g.N ? (uint32_t)(rr * ldo + cc) * ES : GP_FAR;
    if (j < 3) mask_of(j + 1);
#pragma unroll
    for (int i = 0; i < NI; ++i) {
#pragma unroll
      for (int q = 0; q < NQ; ++q) {
        const int k = ONE ? q : 2 * q;
        float v = __builtin_elementwise_maximum(fmaf(acc[i][j][k], g.scale, bias[j]), lo);
        uint32_t w;
        if (ONE) {
          if (MASK == 1 && !(__uint_as_float(m[j & 1][i][q] << 16) > 0.f)) v = 0.f;
          if (MASK == 2 && !a8_positive(m[j & 1][i][q])) v = 0.f;
          w = OUT == 1 ? __float_as_uint(v) : (uint32_t)__builtin_bit_cast(uint16_t, f2bf(v));
        } else {
          typedef __bf16 bf16x2 __attribute__((ext_vector_type(2)));
          const float u = __builtin_elementwise_maximum(fmaf(acc[i][j][k + 1], g.scale, bias[j]), lo);
          const uint32_t p = __builtin_bit_cast(uint32_t, bf16x2{f2bf(v), f2bf(u)});
          const uint32_t t = (uint32_t)__builtin_amdgcn_mov_dpp((int)p, 0xB1, 0xF, 0xF, true);     // lane ^ 1
          w = __builtin_amdgcn_perm(p, t, sel);
          const uint32_t mv = m[j & 1][i][q];
          if (MASK == 1) w = (__uint_as_float(mv << 16) > 0.f ? w & 0xFFFFu : 0u) |
                             (__uint_as_float(mv & 0xFFFF0000u) > 0.f ? w & 0xFFFF0000u : 0u);
          if (MASK == 2) w = (a8_positive(mv & 0xFFu) ? w & 0xFFFFu : 0u) | (a8_positive(mv >> 8) ? w & 0xFFFF0000u : 0u);
        }
        if (OUT == 2) __builtin_amdgcn_raw_buffer_store_b16((uint16_t)w, o, (int)at, row_of(i, q) * ldo * ES, 0);
        else __builtin_amdgcn_raw_buffer_store_b32(w, o, (int)at, row_of(i, q) * ldo * ES, 0);
      }
    }
  }
}

// ---- NT: rows of A and B are K-contiguous, and 32-deep steps would ask the L2 for half lines (with whole ones 24 to 41 %
// of its channels' cycles are requests already): so steps of 64 (rows of 128 B, 16-byte chunk c of row r at
// c ^ ((r >> 1) & 7)), A's in a ring of three panels and w's in two, which is all of the LDS.  A step is two halves
// of 32: in half 0 the fragments of half 1 are read, and in half 1, after its second round, comes the step's one
// barrier: the wave has read all of its panels, and its DMA of the next step has landed.  Then the next step's
// first fragments are read, and the DMA of w's step after it goes into this step's panel; A's is a step further
// ahead, and at the barrier its last panel may still be on its way (two panels each: 32768 x 1248 -> 1024 of 16 experts 107
// to 112 us, now 101 to 106; 8192 x 1024 -> 2048 of 8 masked 57.2, now 56.1; the others 0 to 2 %).
// A piece is three instructions: the buffers do the bounds (with addresses of 64 bits and a selected source of
// zeros it was eight, and the loop 8 % slower).  K a multiple of 8.
constexpr uint32_t GP_NONE = 0xFFFF0000u;                // an offset past every buffer here, with a step's added too
constexpr int GN2_K = 64, GN2_PANEL = GP_B * GN2_K * 2;

template <int NI>
__global__ void __launch_bounds__(GP_THREADS) __attribute__((amdgpu_waves_per_eu(1, 1)))
group_nt_mm_kernel(GroupNtArgs g, int tiles_n, int out) {
  constexpr int PANEL_A = 64 * NI * GN2_K * 2, RING_B = 3 * PANEL_A;
  __shared__ __attribute__((aligned(16))) char smem[RING_B + 2 * GN2_PANEL];
  // (the grid has room for one more row tile per group: the tiles that there are go round the XCDs)
  const int tiles_m = group_tiles<64 * NI>(g.offs, g.E, g.S);
  if ((int)blockIdx.x >= tiles_m * tiles_n) return;
  int tm, tn;
  band_tile(xcd_order(blockIdx.x, tiles_m * tiles_n), tiles_m, tiles_n, tm, tn);
  int e, r0, r1;
  if (!group_find<64 * NI>(g.offs, g.E, g.S, tm, e, r0, r1)) return;
  const int n0 = tn * GP_B;
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wr = wave >> 1, wc = wave & 1;
  const int fr = lane & 31, fq = lane >> 5;
  // fragment (16-deep quarter q, rows 32 i ..): row fr, chunk 2 q + fq
  const int sw = (fr >> 1) & 7;
  int fo[4];
#pragma unroll
  for (int q = 0; q < 4; ++q) fo[q] = fr * 128 + (((2 * q + fq) ^ sw) << 4);
  const int la = wr * 32 * NI * 128, lb = wc * 128 * 128;
  // staging pieces of 8 rows x 128 B: 2 NI of A and 8 of B per wave, from buffers that end with the group's
  // rows (with x, where rows are taken through src) and with w's: what lies past them reads as zeros.
  constexpr int PA = 2 * NI, PN = PA + 8;
  const int pr = lane >> 3;                                  // row of a piece
  const int ck0 = ((lane & 7) ^ ((pr >> 1) & 7)) * 8;        // its chunk's column (even pieces of 8 rows; odd: ^ 32)
  const int odd0 = (wave * PA) & 1;
  auto odd_piece = [&](int p) { return p < PA ? ((p + odd0) & 1) != 0 : ((p - PA) & 1) != 0; };
  uint32_t off[PN];
#pragma unroll
  for (int p = 0; p < PN; ++p) {
    const int r = (p < PA ? wave * PA + p : wave * 8 + p - PA) * 8 + pr;
    const uint32_t ck = odd_piece(p) ? ck0 ^ 32 : ck0;
    if (p >= PA) off[p] = 2u * ((uint32_t)r * (uint32_t)g.ldb + ck);
    else if (!g.src) off[p] = 2u * ((uint32_t)r * (uint32_t)g.lda + ck);
    else {
      const int row = r0 + r < r1 ? group_row(g.src, r0 + r, g.rows, g.top_k) : -1;
      off[p] = row < 0 ? GP_NONE : 2u * ((uint32_t)row * (uint32_t)g.lda + ck);
    }
  }
  const __amdgpu_buffer_rsrc_t ab = out_rows(g.src ? g.a : g.a + (size_t)r0 * g.lda,
                                             2u * (uint32_t)((g.src ? g.rows : min(r1 - r0, 64 * NI)) * (uint32_t)g.lda));
  // (w's rows may share memory, by a stride from 0 on: the last one ends K elements after its start)
  const __amdgpu_buffer_rsrc_t bb = out_rows(g.b + (size_t)e * g.es + (size_t)n0 * g.ldb,
                                             2u * ((uint32_t)(min(g.N - n0, GP_B) - 1) * (uint32_t)g.ldb + (uint32_t)g.K));
  // piece i of step t, w's and A's, the latter into the panel at `to` (a chunk past K: zeros too)
  auto stage_b = [&](int i, int t) {
    const uint32_t v = t * GN2_K + (odd_piece(PA + i) ? ck0 ^ 32 : ck0) < g.K ? off[PA + i] : GP_NONE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(
        bb, (__attribute__((address_space(3))) void*)(smem + RING_B + (t & 1) * GN2_PANEL + (wave * 8 + i) * 1024), 16, (int)v,
        t * GN2_K * 2, 0, 0);
  };
  auto stage_a = [&](int i, int t, int to) {
    const uint32_t v = t * GN2_K + (odd_piece(i) ? ck0 ^ 32 : ck0) < g.K ? off[i] : GP_NONE;
    __builtin_amdgcn_raw_ptr_buffer_load_lds(ab, (__attribute__((address_space(3))) void*)(smem + to + (wave * PA + i) * 1024), 16,
                                             (int)v, t * GN2_K * 2, 0, 0);
  };
  // fragments r = 0 .. 2 NI - 1 of a half: quarter 2 h + r / NI, rows 32 (r % NI) ..
  auto load_a = [&](int r, int h, const char* b) {
    return *reinterpret_cast<const bf16x8*>(b + la + fo[2 * h + r / NI] + (r % NI) * 32 * 128);
  };
  auto load_b = [&](int j, int h, const char* b) {
    return *reinterpret_cast<const bf16x8*>(b + lb + fo[2 * h + (j >> 2)] + (j & 3) * 32 * 128);
  };
  constexpr int NA = 2 * NI, EARLY = 2 * (NA - 2);           // pieces that follow the barrier (two a round): w's, then A's
  const int nt = (g.K + GN2_K - 1) / GN2_K;
  static_assert(EARLY >= 8 && EARLY - 8 <= PA, "w's pieces all follow the barrier");
  // (as the steps issue them: all but those of step 0 may be on their way)
#pragma unroll
  for (int s = 0; s < 3; ++s) {
#pragma unroll
    for (int i = 0; i < (s < 2 ? PA : EARLY - 8); ++i) stage_a(i, s, s * PANEL_A);
#pragma unroll
    for (int i = 0; i < (s < 2 ? 8 : 0); ++i) stage_b(i, s);
  }
  asm volatile("s_waitcnt vmcnt(%0)" ::"n"(PA + EARLY) : "memory");
  __builtin_amdgcn_s_barrier();
  asm volatile("" ::: "memory");
  bf16x8 fa[NA], fb[2][8];
#pragma unroll
  for (int j = 0; j < 8; ++j) fb[0][j] = load_b(j, 0, smem + RING_B);
#pragma unroll
  for (int r = 0; r < NA - 1; ++r) fa[r] = load_a(r, 0, smem);
  f32x16 acc[NI][4] = {};
  int pa = 0, qa = PANEL_A, ra = 2 * PANEL_A;                // A's panels of the steps t, t + 1, t + 2
  for (int t = 0; t < nt; ++t) {
    const char *cur = smem + pa, *nxt = smem + qa;
    const char *bcur = smem + RING_B + (t & 1) * GN2_PANEL, *bnxt = smem + RING_B + ((t + 1) & 1) * GN2_PANEL;
    // (a row fragment is read after its round, the last one after the next half's first MFMA: nothing is
    // read just before a half begins, where the compiler waits for all reads)
    constexpr int FB0 = 2, FB1 = NI == 4 ? 2 : 3;            // column fragments a round, in halves 0 and 1
    // half 0
#pragma unroll
    for (int k = 0; k < 4 * NA; ++k) {
      const int r = k >> 2, j = k & 3;
      acc[r % NI][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[r], fb[0][(r / NI) * 4 + j], acc[r % NI][j], 0, 0, 0);
      if (k == 0) fa[NA - 1] = load_a(NA - 1, 0, cur);
      if (j == 0 && r > 0) fa[r - 1] = load_a(r - 1, 1, cur);
      if (j == 2) {
#pragma unroll
        for (int i = FB0 * r; i < FB0 * r + FB0 && i < 8; ++i) fb[1][i] = load_b(i, 1, bcur);
      }
      if ((j & 1) && EARLY + 2 * r + (j >> 1) < PN) stage_a(EARLY - 8 + 2 * r + (j >> 1), t + 2, ra);
      __builtin_amdgcn_sched_barrier(0);
    }
    // half 1
#pragma unroll
    for (int k = 0; k < 4 * NA; ++k) {
      const int r = k >> 2, j = k & 3;
      acc[r % NI][j] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(fa[r], fb[1][(r / NI) * 4 + j], acc[r % NI][j], 0, 0, 0);
      if (k == 0) fa[NA - 1] = load_a(NA - 1, 1, cur);
      if (k == 7) {
        asm volatile("s_waitcnt vmcnt(%0) lgkmcnt(0)" ::"n"(PA) : "memory");
        __builtin_amdgcn_s_barrier();
        asm volatile("" ::: "memory");      // (no access moves over the barrier)
      }
      if (r >= 2) {
        if (j == 0) {
          fa[r - 1] = load_a(r - 1, 0, nxt);
          if (r == 2) fa[0] = load_a(0, 0, nxt);
        }
        if (j == 2) {
#pragma unroll
          for (int i = FB1 * (r - 2); i < FB1 * (r - 2) + FB1 && i < 8; ++i) fb[0][i] = load_b(i, 0, bnxt);
        }
        if (j & 1) {
          const int i = 2 * (r - 2) + (j >> 1);
          if (i < 8) stage_b(i, t + 2);
          else stage_a(i - 8, t + 3, pa);
        }
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    const int x = pa;
    pa = qa;
    qa = ra;
    ra = x;
  }
  asm volatile("s_waitcnt vmcnt(0)" ::: "memory");           // (nothing in flight into LDS at the end)
  const int row0 = r0 + wr * 32 * NI, n1 = n0 + wc * 128;
#define HFM_OUT(MASK)                                                                   \
  if (out == 0) mm_out_nt<NI, MASK, 0>(g, acc, e, row0, r1 - row0, n1, lane);           \
  else if (out == 1) mm_out_nt<NI, MASK, 1>(g, acc, e, row0, r1 - row0, n1, lane);      \
  else mm_out_nt<NI, MASK, 2>(g, acc, e, row0, r1 - row0, n1, lane);
  if (!g.mask) {
    HFM_OUT(0)
  } else if (!g.mask8) {
    HFM_OUT(1)
  } else {
    HFM_OUT(2)
  }
#undef HFM_OUT
}

// How a call runs: rows a large tile (0: one of the small ones, 32 x 32 where `few`), and the bytes of the operands'
// copies for it.
struct NtPlan {
  int rows;
  long pa, pb;
  bool few;
};
// The least of three times in us, each as measured:
//   32 x 32: 3.5, 3 for 1024 tiles, and the operands from the L2s (twice the time for rows that end within 16 bytes);
//   128 x 128: rounds of 512 tiles, 1.2 a step of 64 with one tile a CU or 1.4 with two, and 10 more (rows at odd
//   places: 1.5 and 2.7 a step; a mask: 1.4 times);
//   the large tile, 256 or 192 rows: rounds of 256 tiles, 0.5 a step of 32 and 8 more (12 with a mask) while there
//   is one round, 0.85 and 12 with more (32768 x 1248 -> 1024, 16 experts: 114 us at 256 rows = 3 rounds, the last one
//   seventh full; 102 to 105 at 192).  It takes 16-byte chunks by LDS-DMA, and rows through 32-bit offsets (all of
//   x where src says which, else 256 rows): operands that are otherwise are copied first (x with its rows in order).
// 32 x 32, 128 x 128, large in us: 192 rows of 8 experts, 1248 -> 400: 7, 25, 22; 256 rows, 4096 -> 4096: 66, 66, 56; 4096
// rows of 4 experts, 512 -> 512: 25, 24, 14; 2048 of 8, 1024 -> 1024 masked: 42, 44, 25; 8192 of 8, 128 -> 64: 7, 17, 9.
// Copies and large against 128 x 128: 25092 rows of 2 experts, 2937 -> 3216 masked: 530, 1264; 32000 of 16, 255 -> 257
// masked: 49, 95; short reductions: 31639 of 33, 32 -> 3368 masked: 174 to 183 against 633 to 676.
static NtPlan nt_plan(const GroupNtArgs& g) {
  const bool whole = g.K % 8 == 0, mask = g.mask != nullptr;
  const long groups = g.E < g.S ? g.E : g.S;                // (those with rows)
  const bool odd_a = !whole || (uintptr_t)g.a % 16 || g.lda % 8, odd_b = !whole || (uintptr_t)g.b % 16 || g.ldb % 8 || g.es % 8;
  const double ft = ((double)g.S / GS_B + 0.5 * groups) * ((g.N + GS_B - 1) / GS_B);
  const double few = (3.5 + ft * (3.0 / 1024) + ft * g.K * 1.2e-5) * (whole ? 1.0 : 2.0);
  const double st = ((double)g.S / GN_B + 0.5 * groups) * ((g.N + GN_B - 1) / GN_B), steps = (g.K + GN_K - 1) / GN_K;
  const double step = odd_a || odd_b ? (st <= 256 ? 1.5 : 2.7) : (st <= 256 ? 1.2 : 1.4);
  const double small = ceil(st / 512) * (step * steps + 10.0) * (mask ? 1.4 : 1.0);
  NtPlan p{0, 0, 0, few < small && (long)(g.S / GS_B + groups) * ((g.N + GS_B - 1) / GS_B) <= 1l << 20};
  if (g.K < 8 || g.K >= 0x7F00 || g.ldo >= GP_MAXLD || g.ldm >= GP_MAXLD || !groups_count(g.E, g.S)) return p;
  const int tn = (g.N + GP_B - 1) / GP_B;
  auto time = [&](int rows) {
    const double tiles = (groups == 1 ? (double)((g.S + rows - 1) / rows) : (double)g.S / rows + 0.5 * groups) * tn;
    const double deep = (g.K + GP_K - 1) / GP_K * (rows / 256.0);
    const double t = tiles <= 256 ? 0.5 * deep + 8.0 + (mask ? 4.0 : 0.0) : ceil(tiles / 256) * (0.85 * deep + 12.0);
    return t + groups * tn / 256.0;                          // (workgroups without a tile: the grid is made for the most)
  };
  const int rows = time(192) < time(256) ? 192 : 256;
  const bool a = odd_a || (g.src ? (long)g.rows * g.lda : 256l * g.lda) >= 0x7F000000l;
  const bool b = odd_b || 256l * g.ldb >= 0x7F000000l;
  const long row = up16(2l * g.K), pa = a ? (long)g.S * row : 0, pb = b ? (long)g.E * g.N * row : 0;
  const double big = time(rows) + (a + b) * 5.0 + (pa + pb) * (2.0 / 4e6);
  if (big >= (p.few ? few : small) || (g.S / rows + groups) * tn > 0xFFFFFFl || (a && g.S >= GROUP_PAD_MAX) ||
      (b && (long)g.E * g.N >= GROUP_PAD_MAX))
    return p;
  return NtPlan{rows, pa, pb, false};
}

HFM_API long hfm_group_nt_ws_bytes(const GroupNtArgs* gp) {
  if (gp->S <= 0 || gp->K <= 0 || gp->N <= 0 || gp->E < 1) return 0;
  const NtPlan p = nt_plan(*gp);
  return p.pa + p.pb;
}

HFM_API int hfm_group_nt(const GroupNtArgs* gp, hipStream_t st) {
  GroupNtArgs g = *gp;
  if (g.S < 0 || g.K < 0 || g.N < 0 || g.E < 1 || g.top_k < 1) return (int)hipErrorInvalidValue;
  if (g.S == 0 || g.N == 0) return 0;
  const NtPlan p = nt_plan(g);
  if (p.rows) {
    if (p.pa + p.pb > 0 && !g.ws) return -1;                 // (nothing launched: the caller brings hfm_group_nt_ws_bytes)
    if ((uintptr_t)g.ws % 16) return (int)hipErrorInvalidValue;
    const long row = up16(2l * g.K);
    char* ws = reinterpret_cast<char*>(g.ws);
    if (p.pa) {
      group_pad(PadArgs{(const char*)g.a, ws, g.src, 0, 2 * g.lda, row, g.S, g.S, 2 * g.K, g.rows, g.top_k}, st);
      g.a = (const bf16*)ws;
      g.lda = row / 2;
      g.src = nullptr;
      g.rows = g.S;
    }
    if (p.pb) {
      group_pad(PadArgs{(const char*)g.b, ws + p.pa, nullptr, 2 * g.es, 2 * g.ldb, row, (long)g.E * g.N, g.N, 2 * g.K, 0, 1}, st);
      g.b = (const bf16*)(ws + p.pa);
      g.ldb = row / 2;
      g.es = (long)g.N * g.ldb;
    }
    g.K = (int)(up16(2l * g.K) / 2);
    const int tn = (g.N + GP_B - 1) / GP_B;
    const long groups = g.E < g.S ? g.E : g.S;
    const dim3 grid((unsigned)((g.S / p.rows + groups) * tn)), blk(GP_THREADS);
    // bf16 outputs in column pairs, with their masks, where the rows are pairs
    const bool pairs = g.N % 2 == 0 && g.ldo % 2 == 0 && g.ldm % 2 == 0 && (uintptr_t)g.out % 4 == 0 &&
                       (uintptr_t)g.mask % (g.mask8 ? 2 : 4) == 0;
    const int out = g.out_f32 ? 1 : pairs ? 0 : 2;
    if (p.rows == 256) hipLaunchKernelGGL(group_nt_mm_kernel<4>, grid, blk, 0, st, g, tn, out);
    else hipLaunchKernelGGL(group_nt_mm_kernel<3>, grid, blk, 0, st, g, tn, out);
    HFM_LAUNCH_CHECK();
  }
  const long groups = g.E < g.S ? g.E : g.S;               // (each adds less than one tile)
  if (p.few) {
    const int fn = (g.N + GS_B - 1) / GS_B;
    hipLaunchKernelGGL(group_nt_few_kernel, dim3((unsigned)((g.S / GS_B + groups) * fn)), dim3(GS_WAVES * 64), 0, st, g, fn);
    HFM_LAUNCH_CHECK();
  }
  const int tn = (g.N + GN_B - 1) / GN_B;
  const long blocks = (g.S / GN_B + groups) * tn;
  if (blocks > 0xFFFFFFl) return (int)hipErrorInvalidValue;       // (a launch has less than 2^32 threads in x)
  hipLaunchKernelGGL(group_nt_kernel, dim3((unsigned)blocks), dim3(256), 0, st, g, tn);
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

template <bool WHOLE, bool X8>
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
    uint64_t w[8];
    uint32_t sc[8];
#pragma unroll
    for (int m = 0; m < 8; ++m) {
      const int p = pbase + mb * 8 + m;
      bf16x8 v = {};
      if (p < p1) {
        if (!isx) {
          v = begin8_bf<WHOLE>(g.dz + (size_t)p * g.ldz, col, g.N);
        } else {
          const int row = group_row(g.src, p, g.rows, g.top_k);
          if (X8) {
            w[m] = row >= 0 ? begin8_code<WHOLE>(reinterpret_cast<const uint8_t*>(g.x) + (size_t)row * g.ldx, col, g.K) : 0;
            sc[m] = row >= 0 && col < g.K ? g.xs[(size_t)row * sblk + col / A8_BLOCK] : 0;
          } else if (row >= 0) {
            v = begin8_bf<WHOLE>(reinterpret_cast<const bf16*>(g.x) + (size_t)row * g.ldx, col, g.K);
          }
        }
      } else if (X8) {
        w[m] = sc[m] = 0;
      }
      in[m] = __builtin_bit_cast(uint4, v);
    }
    if (X8 && isx) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        if (!WHOLE) end8_code(w[m], col, g.K);
        float f[8];
        a8_unpack8(make_uint2((uint32_t)w[m], (uint32_t)(w[m] >> 32)), sc[m], f);
        bf16x8 v;
#pragma unroll
        for (int j = 0; j < 8; ++j) v[j] = f2bf(f[j]);
        in[m] = __builtin_bit_cast(uint4, v);
      }
    } else if (!WHOLE && col + 8 > (isx ? g.K : g.N)) {
#pragma unroll
      for (int m = 0; m < 8; ++m) {
        bf16x8 v = __builtin_bit_cast(bf16x8, in[m]);
        end8_bf(v, col, isx ? g.K : g.N);
        in[m] = __builtin_bit_cast(uint4, v);
      }
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
#pragma unroll 8
  for (int q = 1; q < g.ns; ++q) v += s[q * step];
  (i < nw ? g.dw[i] : g.db[i - nw]) = v;
}

// ---- TN: the weight gradient on the large tile.  Both panels keep their global layout, [32 rows][256
// columns]; the fragments (8 rows of one column per lane) come from transposing LDS reads
// (ds_read_b64_tr_b16: a 16-lane group reads 4 rows x 16 columns, lane l gets column l's 4 rows).
// A panel row is 512 B, so a fragment's 16 rows would meet in the same banks: 32-byte granule c of row r
// lies at c ^ f(r), f(r) = (r & 3) << 1 | (r >> 3 & 1): a half-wave's 4 rows x 2 granules take all 8 of 256 B.
// 8-bit x: 32 codes a thread (one scale) are loaded two steps ahead, turned into bf16 times the
// scale (one conversion per pair, exact) and written into the same image.
//
// The rows are cut evenly, not by groups: all groups' rows in a line (in units of 64, and GW_SEG more for
// each group, which is what its prologue and outputs cost) are cut into `lanes` equal parts, and
// workgroup (lane, tile) sums its tile over its lane, group after group.  The tiles of a lane are
// neighbours: they run side by side on an XCD and read the same rows at the same time (cut tile by
// tile, every workgroup at its own rows, the panels came from beyond the L2: 150 us for 16 groups of
// 2048 rows x 1024 x 1024 against 71 us for one of as many steps).  A group within one lane goes straight
// to dw; what a lane boundary cuts goes to the workspace, two tiles per workgroup at most, and is
// summed in row order by a second launch.
constexpr int GW_UNIT = 64;                      // rows of a unit
constexpr int GW_SLAB = GP_B * GP_B;             // floats of a workspace tile

constexpr int GW_SEG = 6;                        // a group's own units (10 us against 1.7 us a unit)

// Unit u of the line belongs to lane l with U l / L <= u < U (l + 1) / L.
__device__ __forceinline__ int wg_cut(int U, int L, int l) { return (int)((long)U * l / L); }
__device__ __forceinline__ int wg_owner(int U, int L, int u) {
  int l = (int)((long)u * L / U);
  while (wg_cut(U, L, l + 1) <= u) ++l;
  while (l > 0 && wg_cut(U, L, l) > u) --l;
  return l;
}
// 64-row steps of a group (one for an empty group: the lane that has it writes the zeros)
__device__ __forceinline__ int wg_steps(const int* offs, int e, int S) {
  int lo, hi;
  group_rows(offs, e, S, lo, hi);
  return max(1, (hi - lo + GW_UNIT - 1) / GW_UNIT);
}
// units of the groups below `upto`, by every wave for itself
__device__ __forceinline__ int wg_units(const int* offs, int upto, int S) {
  const int lane = threadIdx.x & 63;
  int n = 0;
  for (int e = lane; e < upto; e += 64) n += wg_steps(offs, e, S) + GW_SEG;
  for (int d = 32; d; d >>= 1) n += __shfl_xor(n, d);
  return __builtin_amdgcn_readfirstlane(n);
}
// the group of unit u, and its first unit
__device__ __forceinline__ void wg_find(const int* offs, int E, int S, int u, int& e, int& first) {
  const int lane = threadIdx.x & 63;
  int run = 0;
  e = 0;
  first = 0;
  for (int e0 = 0; e0 < E; e0 += 64) {
    const int n = e0 + lane < E ? wg_steps(offs, e0 + lane, S) + GW_SEG : 0;
    int inc = n;
    for (int d = 1; d < 64; d <<= 1) {
      const int v = __shfl_up(inc, d);
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
  first = __builtin_amdgcn_readfirstlane(first);
}

typedef short s16x4 __attribute__((ext_vector_type(4)));
// (restrict: a transposing read carries no type that would tell it from the LDS-DMA in flight, and without
// an aliasing fact the compiler waits for all DMA before each; mm_loop has the waits that are needed)
__device__ __forceinline__ bf16x8 tr_read(const char* __restrict__ p0, const char* __restrict__ p1) {
  typedef __attribute__((address_space(3))) s16x4* lp;
  const s16x4 a = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p0);
  const s16x4 b = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lp)p1);
  return __builtin_bit_cast(bf16x8, __builtin_shufflevector(a, b, 0, 1, 2, 3, 4, 5, 6, 7));
}

// 16 bytes into LDS (restrict: as for tr_read)
__device__ __forceinline__ void lds_put(char* __restrict__ p, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  *reinterpret_cast<uint4*>(p) = make_uint4(a, b, c, d);
}

// db: the waves that hold the same rows of dz take turns with its steps (wave wc of tile column tk those with s %
// (2 tiles_k) == 2 tk + wc), and leave 256 sums for each group and lane, behind the tiles of the workspace:
// [group + lane][row of tiles][tile column, wave][256].  (group + lane tells the parts of the line
// apart: from one to the next, one of the two grows.)
__host__ __device__ __forceinline__ size_t wg_slabs(int tiles, int lanes) {
  return lanes > 1 ? (size_t)2 * lanes * tiles * GW_SLAB : 0;
}
__device__ __forceinline__ float* wg_sums(const GroupWgArgs& g, int tiles_n, int tiles_k, int lanes, int part, int tn) {
  return g.ws + wg_slabs(tiles_n * tiles_k, lanes) + ((size_t)part * tiles_n + tn) * 2 * tiles_k * GP_B;
}

template <bool X8, bool GATHER>
__global__ void __launch_bounds__(GP_THREADS) __attribute__((amdgpu_waves_per_eu(1, 1)))
group_wgrad_mm_kernel(GroupWgArgs g, int tiles_n, int tiles_k, int lanes) {
  __shared__ __attribute__((aligned(16))) char smem[GP_RING * GP_BUF];
  const int wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6), lane = threadIdx.x & 63;
  const int wr = wave >> 1, wc = wave & 1;
  const int tiles = tiles_n * tiles_k;
  const int w = xcd_order(blockIdx.x, gridDim.x);
  const int U = wg_units(g.offs, g.E, g.S), L = min(lanes, U);       // (fewer rows than S: no lane without a unit)
  if (w / tiles >= L) return;
  const int u0 = wg_cut(U, L, w / tiles), u1 = wg_cut(U, L, w / tiles + 1);
  int tn, tk;
  band_tile(w % tiles, tiles_n, tiles_k, tn, tk);
  const int n0 = tn * GP_B, k0 = tk * GP_B;
  int e, first;
  wg_find(g.offs, g.E, g.S, u0, e, first);
  // fragment (half h, columns 32 i ..): the lane's 16-lane group takes rows 16 h + 8 (lane >> 5) .. and
  // columns 32 i + (lane & 16) ..: granule (2 i + (lane >> 4 & 1)) ^ f(row), which is an xor with 2 i
  const int l4 = (lane >> 2) & 3, h5 = lane >> 5;
  const int rowoff = (h5 * 8 + l4) * 512 + (lane & 3) * 8 + ((((lane >> 4) & 1) ^ (l4 << 1) ^ h5) << 5);
  int la = rowoff + wr * 256, lb = GP_PANEL + rowoff + wc * 256;
  // staging pieces: 2 rows of 512 B, 4 of each operand per wave.  Row 2 i + hi of the wave's 8 has
  // f = 2 ((2 i + hi) & 3) + (wave & 1), so the lane's 16-byte chunk is one column for even i and
  // that column ^ 64 for odd i.
  const int hi = lane >> 5, c16 = lane & 31;
  const int ce = (((c16 >> 1) ^ ((hi << 1) | (wave & 1))) * 2 + (c16 & 1)) * 8;
  const int sblk = (g.K + A8_BLOCK - 1) / A8_BLOCK;
  // 8-bit x: 32 codes (granules 2 xq, 2 xq + 1) of row xr, in four pieces of 8 (16 bytes as bf16).  A lane's piece in
  // turn q is q ^ xp: eight neighbouring lanes then write to eight different 16-byte places of 128 bytes (all in
  // the same order: four in one place, half of the LDS cycles were conflicts, a product of 466 us took 434 so).
  const int xr = threadIdx.x >> 3, xq = threadIdx.x & 7, xc = xq * 32, xp = xq >> 1;
  const int xf = ((xr & 3) << 1) | ((xr >> 3) & 1);
  const int xo = GP_PANEL + xr * 512 + ((((2 * xq) ^ xf) << 5) ^ (xp << 4));           // (piece of turn q: ^ q << 4)
  for (; e < g.E && first < u1; ++e) {
    const int steps = wg_steps(g.offs, e, g.S), rows0 = first + GW_SEG;      // (the group's rows begin here)
    first = rows0 + steps;
    const int s0 = max(0, u0 - rows0), s1 = min(steps, u1 - rows0);
    if (s0 >= s1) continue;
    int lo, hi_row;
    group_rows(g.offs, e, g.S, lo, hi_row);
    // (scalar for certain: the buffers below are made of them)
    const int p0 = __builtin_amdgcn_readfirstlane(lo + s0 * GW_UNIT);
    const int p1 = __builtin_amdgcn_readfirstlane(min(hi_row, lo + s1 * GW_UNIT));
    const int ns = p1 > p0 ? (p1 - p0 + GP_K - 1) / GP_K : 0;
    f32x16 acc[4][4] = {};
    float sum[4] = {0.f, 0.f, 0.f, 0.f};
    // columns past N or K read column 0 (their outputs are not stored)
    const uint32_t ao0 = 2u * (uint32_t)(hi * (int)g.ldz + (n0 + ce < g.N ? n0 + ce : 0));
    const uint32_t ao1 = 2u * (uint32_t)(hi * (int)g.ldz + (n0 + (ce ^ 64) < g.N ? n0 + (ce ^ 64) : 0));
    const int bc0 = k0 + ce < g.K ? k0 + ce : 0, bc1 = k0 + (ce ^ 64) < g.K ? k0 + (ce ^ 64) : 0;
    const uint32_t bo0 = GATHER ? 0u : 2u * (uint32_t)(hi * (int)g.ldx + bc0);
    const uint32_t bo1 = GATHER ? 0u : 2u * (uint32_t)(hi * (int)g.ldx + bc1);
    // GATHER: rows of x of a step's pieces (or of its codes), read two steps before they are used;
    // -1: a row of zeros (past p1, or a source that is no slot)
    int xrow[2][4];
    auto row_at = [&](int p) {
      const int s = g.src[min(p, g.S - 1)], r = s / g.top_k;
      return p < p1 && s >= 0 && r < g.rows ? r : -1;
    };
    auto rows_of = [&](int set, int s) {
      if (!GATHER) return;
      if (X8) {
        xrow[set][0] = row_at(p0 + s * GP_K + xr);
      } else {
#pragma unroll
        for (int i = 0; i < 4; ++i) xrow[set][i] = row_at(p0 + s * GP_K + wave * 8 + 2 * i + hi);
      }
    };
    // A step's rows of the wave as a buffer that ends with the last row of the part: past it read zeros
    auto bytes_left = [&](int s, uint32_t row) {
      const int n = p1 - (p0 + s * GP_K + wave * 8);
      return (uint32_t)__builtin_amdgcn_readfirstlane((n < 0 ? 0 : n > 8 ? 8 : n) * (int)row);
    };
    auto piece_a = [&](int i, int s) {
      const bf16* base = g.dz + (size_t)(p0 + s * GP_K + wave * 8) * g.ldz;
      const uint32_t row = 2u * (uint32_t)g.ldz;
      dma16_buf(base, bytes_left(s, row), (i & 1) ? ao1 : ao0, 2u * i * row,
                smem + (s & (GP_RING - 1)) * GP_BUF + (wave * 4 + i) * 1024);
    };
    auto piece_b = [&](int i, int s, int row) {
      char* to = smem + (s & (GP_RING - 1)) * GP_BUF + GP_PANEL + (wave * 4 + i) * 1024;
      const bf16* xb = reinterpret_cast<const bf16*>(g.x);
      if (GATHER) {
        const void* q = row >= 0 ? (const void*)(xb + (size_t)(uint32_t)row * g.ldx + ((i & 1) ? bc1 : bc0)) : (const void*)g_zero16;
        dma16(q, to);
      } else {
        const uint32_t rb = 2u * (uint32_t)g.ldx;
        dma16_buf(xb + (size_t)(p0 + s * GP_K + wave * 8) * g.ldx, bytes_left(s, rb), (i & 1) ? bo1 : bo0,
                  2u * i * rb, to);
      }
    };
    // X8: a step's codes and scale into registers (set), and from there into the image.  Rows past p1 are zeros: by
    // the buffer's end; where src says the rows, cleared on the way to the image, where the loads have arrived (the
    // scale too: what row 0 has there may be no scale at all, and zero times it no zero).
    typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
    u32x2 cd[2][4];
    uint32_t cs[2], con[2];
    // (columns past K: any values of the next row, zeros behind the last)
    const int behind = (int)g.ldx - (g.K + 7) / 8 * 8;
    const int xv = xr * (int)g.ldx + k0 + xc, xsv = xr * sblk + (k0 + xc) / A8_BLOCK;
    auto codes_of = [&](int set, int s) {
      const int r0 = p0 + s * GP_K;
      if constexpr (GATHER) {
        const int row = xrow[set][0];
        con[set] = row >= 0 ? 0xFFFFFFFFu : 0u;
        const size_t at = row >= 0 ? (size_t)row : 0;     // (row 0 is there: x has rows)
        const bool in = k0 + xc < g.K;                    // (columns past K: any values)
        const uint8_t* c = reinterpret_cast<const uint8_t*>(g.x) + at * g.ldx + (in ? k0 + xc : 0);
        const int last = in ? (min(32, g.K - k0 - xc) - 1) >> 3 : 0;
#pragma unroll
        for (int q = 0; q < 4; ++q) cd[set][q] = *reinterpret_cast<const u32x2*>(c + min(q ^ xp, last) * 8);
        cs[set] = g.xs[at * sblk + (in ? (k0 + xc) / A8_BLOCK : 0)];
      } else {
        const int n = __builtin_amdgcn_readfirstlane(min(max(p1 - r0, 0), GP_K));
        // (the codes end with the last row's K: what lies behind it may be nobody's, where they are columns of wider rows.
        // A K that is no multiple of 8 has its copies' rows, which go on in zeros)
        const __amdgpu_buffer_rsrc_t c = __builtin_amdgcn_make_buffer_rsrc(
            const_cast<uint8_t*>(reinterpret_cast<const uint8_t*>(g.x)) + (size_t)r0 * g.ldx, 0,
            max(n * (int)g.ldx - behind, 0), 0x00020000);
        const __amdgpu_buffer_rsrc_t sc =
            __builtin_amdgcn_make_buffer_rsrc(const_cast<uint8_t*>(g.xs) + (size_t)r0 * sblk, 0, n * sblk, 0x00020000);
#pragma unroll
        for (int q = 0; q < 4; ++q)
          cd[set][q] = __builtin_bit_cast(u32x2, __builtin_amdgcn_raw_buffer_load_b64(c, xv + ((q ^ xp) << 3), 0, 0));
        cs[set] = __builtin_amdgcn_raw_buffer_load_b8(sc, xsv, 0, 0);
        con[set] = 0xFFFFFFFFu;
      }
    };
    auto codes_put = [&](int set, int s, int q) {
      const float f = a8_scale(GATHER ? cs[set] & con[set] : cs[set]);
      if (q == 0) {
        uint32_t u[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) u[i] = cd[set][i >> 1][i & 1];
        a8_finite_rare(u, f);
#pragma unroll
        for (int i = 0; i < 8; ++i) cd[set][i >> 1][i & 1] = u[i];
      }
      const uint32_t a = GATHER ? cd[set][q][0] & con[set] : cd[set][q][0], b = GATHER ? cd[set][q][1] & con[set] : cd[set][q][1];
      lds_put(smem + (s & (GP_RING - 1)) * GP_BUF + (xo ^ (q << 4)), a8_pair_bf16<false>(a, f), a8_pair_bf16<true>(a, f),
              a8_pair_bf16<false>(b, f), a8_pair_bf16<true>(b, f));
    };
    auto codes_to = [&](int set, int s) {
#pragma unroll
      for (int q = 0; q < 4; ++q) codes_put(set, s, q);
    };
    // (la and lb are hidden from the optimizer in every step: 16 addresses made by one xor each, not kept)
    auto hide = [&]() {
      int a = la, b = lb;
      asm volatile("" : "+v"(a), "+v"(b));
      la = a;
      lb = b;
    };
    auto frag = [](const char* p) { return tr_read(p, p + 4 * 512); };
    auto load_a = [&](int i, const char* b) { return frag(b + (la ^ ((i & 3) << 6)) + (i >> 2) * 16 * 512); };
    auto load_b = [&](int j, const char* b) { return frag(b + (lb ^ ((j & 3) << 6)) + (j >> 2) * 16 * 512); };
    if (ns > 0) {
      rows_of(0, 0);
      rows_of(1, 1);
      if constexpr (X8) {
        // the codes of step s + 3 (read in step s - 2) go to the image in step s, in pieces between the MFMAs,
        // and then those of s + 5 are read; they are in LDS before the last fragment of step s is read, so
        // before step s + 2 reads them.  At a step's top 5 + 4 + 5 loads (or more) follow the DMA that it waits
        // for: two steps' codes and one's DMA.
        codes_of(0, 0);
        codes_of(1, 1);
        codes_to(0, 0);
        codes_to(1, 1);
        rows_of(0, 2);
        rows_of(1, 3);
        codes_of(0, 2);
        codes_to(0, 2);
        rows_of(0, 4);
        codes_of(1, 3);
        codes_of(0, 4);
        rows_of(1, 5);
        rows_of(0, 6);
        mm_loop<4, 4, 14>(smem, ns, acc, sum, 2 * tk + wc, 2 * tiles_k, piece_a, load_a, load_b, [&](auto PAR, int s, int k) {
          constexpr int set = decltype(PAR)::value ^ 1;
          if (k == -1) hide();
          if (k >= 0 && k % 6 == 5 && k / 6 < 4) codes_put(set, s + 3, k / 6);
          if (k == 29) {
            codes_of(set, s + 5);
            rows_of(set, s + 7);
          }
        });
      } else {
        // GATHER: a step's rows are read two steps before its DMA starts
        mm_loop<4, 8, 8>(
            smem, ns, acc, sum, 2 * tk + wc, 2 * tiles_k,
            [&](int i, int s) {
              if (i < 4) piece_a(i, s);
              else piece_b(i - 4, s, xrow[s & 1][i - 4]);
              if (i == 7) rows_of(s & 1, s + 2);
            },
            load_a, load_b, [&](auto, int, int k) { if (k == -1) hide(); });
      }
    }
    __syncthreads();                      // (the next part's staging overwrites what was read here)
    // a whole tile goes to dw, a part to the workspace: slot 2 w if it is the workgroup's first, 2 w + 1
    // if it goes on in the next one
    const bool whole = s0 == 0 && s1 == steps;
    if (g.db) {
      float* d = wg_sums(g, tiles_n, tiles_k, lanes, e + w / tiles, tn) + (2 * tk + wc) * GP_B + wr * 128;
#pragma unroll
      for (int i = 0; i < 4; ++i) {
        const float v = sum[i] + __shfl_xor(sum[i], 32);
        if (lane < 32) d[i * 32 + lane] = v;
      }
    }
    if (whole)
      mm_out_f32(acc, g.dw + ((size_t)e * g.N + n0 + wr * 128) * g.K + k0 + wc * 128, g.N - n0 - wr * 128,
                 g.K - k0 - wc * 128, g.K, lane);
    else
      mm_out_f32(acc, g.ws + (size_t)(2 * w + (s0 > 0 ? 0 : 1)) * GW_SLAB + wr * 128 * GP_B + wc * 128, 128, 128, GP_B, lane);
  }
}

// Groups that two or more lanes made: their parts in row order; db of all.  grid (tiles, E, strips of 4 R rows, or
// 1 for db alone).
template <int R>
__global__ void __launch_bounds__(256) group_wgrad_join_kernel(GroupWgArgs g, int tiles_n, int tiles_k, int lanes, int ovec) {
  const int tiles = tiles_n * tiles_k, ti = blockIdx.x, e = blockIdx.y;
  int tn, tk;
  band_tile(ti, tiles_n, tiles_k, tn, tk);
  const bool sums = g.db && tk == 0 && blockIdx.z == 0;
  if (lanes == 1 && !sums) return;
  const int U = wg_units(g.offs, g.E, g.S), rows0 = wg_units(g.offs, e, g.S) + GW_SEG, steps = wg_steps(g.offs, e, g.S);
  const int L = min(lanes, U), l0 = wg_owner(U, L, rows0), l1 = wg_owner(U, L, rows0 + steps - 1);
  const int n0 = tn * GP_B, k0 = tk * GP_B;
  if (sums && n0 + (int)threadIdx.x < g.N) {
    float v = 0.f;
    for (int l = l0; l <= l1; ++l) {
      const float* s = wg_sums(g, tiles_n, tiles_k, lanes, e + l, tn) + threadIdx.x;
#pragma unroll 8
      for (int i = 0; i < 2 * tiles_k; ++i) v += s[i * GP_B];
    }
    g.db[(size_t)e * g.N + n0 + threadIdx.x] = v;
  }
  if (l0 == l1) return;
  // the lane that starts the group left it in its second tile, the others in their first
  const float* s0 = g.ws + (size_t)(2 * (l0 * tiles + ti) + 1) * GW_SLAB;
  const float* s1 = g.ws + (size_t)(2 * ((l0 + 1) * tiles + ti)) * GW_SLAB;
  const size_t next = (size_t)2 * tiles * GW_SLAB;
  const int r0 = blockIdx.z * (4 * R) + (threadIdx.x >> 6), c = (threadIdx.x & 63) * 4;
  f32x4 v[R];
#pragma unroll
  for (int i = 0; i < R; ++i) v[i] = *reinterpret_cast<const f32x4*>(s0 + (r0 + 4 * i) * GP_B + c);
  int l = l0 + 1;
  for (; l + 3 <= l1; l += 4, s1 += 4 * next) {             // (four parts' loads at a time, summed in order)
    f32x4 a[4][R];
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < R; ++i) a[m][i] = *reinterpret_cast<const f32x4*>(s1 + m * next + (r0 + 4 * i) * GP_B + c);
#pragma unroll
    for (int m = 0; m < 4; ++m)
#pragma unroll
      for (int i = 0; i < R; ++i) v[i] += a[m][i];
  }
  for (; l <= l1; ++l, s1 += next) {
#pragma unroll
    for (int i = 0; i < R; ++i) v[i] += *reinterpret_cast<const f32x4*>(s1 + (r0 + 4 * i) * GP_B + c);
  }
#pragma unroll
  for (int i = 0; i < R; ++i) {
    const int r = r0 + 4 * i;
    if (n0 + r >= g.N || k0 + c >= g.K) continue;
    float* d = g.dw + ((size_t)e * g.N + n0 + r) * g.K + k0 + c;
    if (ovec) {
      *reinterpret_cast<f32x4*>(d) = v[i];
    } else {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        if (k0 + c + j < g.K) d[j] = v[i][j];
    }
  }
}

// Where the large tile is taken: enough work for every CU (GP_MIN_UNITS steps of 64 rows each, from 8 bits half as
// many; below that the 128 x 128 tile's smaller pieces fill the chip better).  128 x 128 against 256 x 256 in us, one
// group: 16384 rows, 256 x 256: 32, 44 (8 bits: 52, 46); 32768: 48, 56; 1024 rows, 1024 x 1024: 28, 26; 4096: 52, 35;
// 16384: 145, 58; 4 groups, 4096 rows, 512 x 512: 27, 35 (8 bits: 44, 34); 16 groups, 32768 rows, 1024 x
// 1024: 290, 115.
constexpr int GW_CUS = 256, GP_MIN_UNITS = 2;
static bool wgrad_big(const GroupWgArgs& g) {
  if (g.ldz >= 1l << 25 || g.ldx >= 1l << 25 || g.K >= GP_MAXLD || g.E > 65535 || !groups_count(g.E, g.S))
    return false;                                          // (32-bit offsets; grid; the line's units)
  const long tiles = (long)((g.N + GP_B - 1) / GP_B) * ((g.K + GP_B - 1) / GP_B);
  return g.rows > 0 && tiles <= 1l << 20 && tiles * (g.S / GW_UNIT) >= (long)GW_CUS * GP_MIN_UNITS / (g.xs ? 2 : 1);
}
// Time in us by l lanes: the rounds of the CUs times a lane's length (its rows, and a group's own cost); then
// the parts' way through the workspace (0.065 us each, as many as there are cuts through rows) and the
// longest sum of them.
static double wgrad_time(const GroupWgArgs& g, long tiles, int l) {
  const double rows = (double)(g.S / GW_UNIT) + g.E, units = rows + (double)g.E * GW_SEG;
  const double t = (double)((l * tiles + GW_CUS - 1) / GW_CUS) * (units / l + GW_SEG) * 1.7;
  return l == 1 ? t : t + 6 + 2 * (l - 1) * (rows / units) * tiles * 0.065 + ((double)l / g.E + 1) * 0.3;
}
// Lanes: the least time within 512 workgroups (a workspace of 256 MB) unless the tiles alone are more.
static int wgrad_lanes(const GroupWgArgs& g) {
  const long tiles = (long)((g.N + GP_B - 1) / GP_B) * ((g.K + GP_B - 1) / GP_B);
  int best = 1;
  double least = wgrad_time(g, tiles, 1);
  for (int l = 2; l * tiles <= 512; ++l) {
    const double t = wgrad_time(g, tiles, l);
    if (t < least) {
      least = t;
      best = l;
    }
  }
  return best;
}
// The operands' copies that the large tile needs (rows of whole 16-byte chunks), as for the NT product: where they
// and the large tile take less than the 128 x 128 tile (20 us and 60 TFLOP/s of whole tiles for such operands,
// 25 from 8 bits).  Copies against 128 x 128 in us: 25092 rows of 2 groups, 2937 x 3216: 524, 4125, from 8-bit x
// 560, 6340; 1500 of 16, 1501 x 1001: 62, 73; 20000 of 8, 201 x 401: 54, 76; 26966 of 10, 42 x 2191: 114, 223.
struct WgPlan {
  bool big;
  long pz, px;
};
static WgPlan wg_plan(const GroupWgArgs& g) {
  WgPlan p{wgrad_big(g), 0, 0};
  if (!p.big) return p;
  const int per = g.xs ? 16 : 8, xb = g.xs ? 1 : 2;
  const bool z = (uintptr_t)g.dz % 16 || g.N % 8 || g.ldz % 8, x = (uintptr_t)g.x % 16 || g.K % per || g.ldx % per;
  if (z) p.pz = (long)g.S * up16(2l * g.N);
  if (x) p.px = (long)g.rows * up16((long)xb * g.K);
  if (z || x) {
    const long tiles = (long)((g.N + GP_B - 1) / GP_B) * ((g.K + GP_B - 1) / GP_B);
    const double t = (z + x) * 5.0 + (p.pz + p.px) * (2.0 / 4.5e6) + wgrad_time(g, tiles, wgrad_lanes(g));
    const double wide = 2.0 * g.S * ((g.N + GN_B - 1) / GN_B * GN_B) * ((g.K + GN_B - 1) / GN_B * GN_B);
    if (t > 20.0 + wide / (g.xs ? 25e6 : 60e6) || g.S >= GROUP_PAD_MAX || g.rows >= GROUP_PAD_MAX) p = WgPlan{false, 0, 0};
  }
  return p;
}

// Two parts a workgroup (a single lane cuts no group), and the sums for db.
static long wgrad_ws_floats(const GroupWgArgs& g) {
  const long l = wgrad_lanes(g), tn = (g.N + GP_B - 1) / GP_B, tk = (g.K + GP_B - 1) / GP_B;
  return (long)wg_slabs((int)(tn * tk), (int)l) + (g.db ? (g.E + l) * tn * 2 * tk * GP_B : 0);
}

// Splits of the rows, within a workgroup for every CU: the least of the steps of 64 rows that follow one another
// (2.2 us each) and the partial products' way (6 us and their bytes at 4.5 TB/s).  762 rows of 2 groups, 64 x 59: 14
// us, with 2 steps a split 19, with 4 25; 4096 rows of 4 groups, 512 x 512: 27, with two workgroups for every
// CU 34; 512 rows of them: 12 unsplit, 17 in two.
static int wgrad_splits(int S, int N, int K, int E) {
  const long tiles = (long)E * ((N + GN_B - 1) / GN_B) * ((K + GN_B - 1) / GN_B);
  if (tiles <= 0) return 1;
  const int steps = (int)((long)S / E / 64) + 1;
  const double bytes = 4.0 * E * N * K;
  int best = 1;
  double least = 2.2 * steps;
  for (int ns = 2; ns <= 32 && ns <= steps && ns * tiles <= GW_CUS; ++ns) {
    const double t = 2.2 * ((steps + ns - 1) / ns) + 6.0 + (2 * ns + 1) * bytes / 4.5e6;
    if (t < least) {
      least = t;
      best = ns;
    }
  }
  return best;
}

HFM_API long hfm_group_wgrad_ws_floats(const GroupWgArgs* gp) {
  const WgPlan p = wg_plan(*gp);
  if (p.big) return (p.pz + p.px) / 4 + wgrad_ws_floats(*gp);
  const int ns = wgrad_splits(gp->S, gp->N, gp->K, gp->E);
  return ns > 1 ? (long)ns * gp->E * gp->N * (gp->K + 1) : 0;
}

HFM_API int hfm_group_wgrad(const GroupWgArgs* gp, hipStream_t st) {
  GroupWgArgs g = *gp;
  if (g.S < 0 || g.K < 0 || g.N < 0 || g.E < 1 || g.top_k < 1) return (int)hipErrorInvalidValue;
  if (g.N == 0) return 0;
  const WgPlan p = wg_plan(g);
  if (p.big) {
    const int tn = (g.N + GP_B - 1) / GP_B, tk = (g.K + GP_B - 1) / GP_B;
    const int lanes = wgrad_lanes(g);
    if ((lanes > 1 || g.db || p.pz || p.px) && (!g.ws || (uintptr_t)g.ws % 16)) return (int)hipErrorInvalidValue;
    char* ws = reinterpret_cast<char*>(g.ws);
    if (p.pz) {
      const long row = up16(2l * g.N);
      group_pad(PadArgs{(const char*)g.dz, ws, nullptr, 0, 2 * g.ldz, row, g.S, g.S, 2 * g.N, 0, 1}, st);
      g.dz = (const bf16*)ws;
      g.ldz = row / 2;
    }
    if (p.px) {
      const int xb = g.xs ? 1 : 2;
      const long row = up16((long)xb * g.K);
      group_pad(PadArgs{(const char*)g.x, ws + p.pz, nullptr, 0, xb * g.ldx, row, g.rows, g.rows, xb * g.K, 0, 1}, st);
      g.x = ws + p.pz;
      g.ldx = row / xb;
    }
    g.ws = reinterpret_cast<float*>(ws + p.pz + p.px);
    const int ovec = g.K % 8 == 0 && (uintptr_t)g.dw % 16 == 0;
    const dim3 grid((unsigned)(tn * tk * lanes)), blk(GP_THREADS);
    if (g.xs && g.src) hipLaunchKernelGGL((group_wgrad_mm_kernel<true, true>), grid, blk, 0, st, g, tn, tk, lanes);
    else if (g.xs) hipLaunchKernelGGL((group_wgrad_mm_kernel<true, false>), grid, blk, 0, st, g, tn, tk, lanes);
    else if (g.src) hipLaunchKernelGGL((group_wgrad_mm_kernel<false, true>), grid, blk, 0, st, g, tn, tk, lanes);
    else hipLaunchKernelGGL((group_wgrad_mm_kernel<false, false>), grid, blk, 0, st, g, tn, tk, lanes);
    if (lanes > 1 || g.db) {
      // (16 rows a workgroup, or 4 where that leaves CUs without one: 32768 rows, 256 x 256: 67 us in all, 56 so)
      if ((long)tn * tk * g.E * 16 >= GW_CUS)
        hipLaunchKernelGGL(group_wgrad_join_kernel<4>, dim3(tn * tk, g.E, lanes > 1 ? 16 : 1), dim3(256), 0, st, g, tn, tk, lanes, ovec);
      else
        hipLaunchKernelGGL(group_wgrad_join_kernel<1>, dim3(tn * tk, g.E, lanes > 1 ? 64 : 1), dim3(256), 0, st, g, tn, tk, lanes, ovec);
    }
    HFM_LAUNCH_CHECK();
  }
  g.ns = wgrad_splits(g.S, g.N, g.K, g.E);
  if (g.ns > 1 && !g.ws) return (int)hipErrorInvalidValue;
  const int tn = (g.N + GN_B - 1) / GN_B, tk = g.K > 0 ? (g.K + GN_B - 1) / GN_B : 1;
  const long blocks = (long)tn * tk * g.E * g.ns;
  if (blocks > 0xFFFFFFl) return (int)hipErrorInvalidValue;       // (a launch has less than 2^32 threads in x)
  const dim3 grid((unsigned)blocks), blk(256);
  if (g.N % 8 == 0 && g.K % 8 == 0) {
    if (g.xs) hipLaunchKernelGGL((group_wgrad_kernel<true, true>), grid, blk, 0, st, g, tn, tk);
    else hipLaunchKernelGGL((group_wgrad_kernel<true, false>), grid, blk, 0, st, g, tn, tk);
  } else {
    if (g.xs) hipLaunchKernelGGL((group_wgrad_kernel<false, true>), grid, blk, 0, st, g, tn, tk);
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
