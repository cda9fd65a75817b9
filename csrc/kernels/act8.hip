// Activations to 8 bits and back (act8.h has the format).  Bound by the bytes: 2 (bf16) or 4 read
// and 1 + 1/32 written per value, and the reverse (16384 x 4096 bf16: 48 us there, 4.2 TB/s, 31 us back).
// Accesses of 8 or 16 bytes may start at any element; a row's last values, fewer than 8, go one by one
// (16384 x 4095 bf16: 61 us there, 64 back; with a value a lane 204, 146).
#include "act8.h"

struct Act8Args {
  const void* x;           // pack: values [M, N], row stride ld;  unpack: null
  uint8_t* codes;          // [M, N], row stride ldc
  uint8_t* scales;         // [M, ceil(N / 32)]
  void* out;               // unpack: values, row stride ld
  long ld, ldc;
  int M, N, bf;
};

typedef bf16 any_bf16x8 __attribute__((ext_vector_type(8), aligned(2)));
typedef float any_f32x4 __attribute__((ext_vector_type(4), aligned(4)));
typedef uint32_t any_u32x2 __attribute__((ext_vector_type(2), aligned(1)));

// n (at most 8) values of a row; zeros behind them
template <int BF>
__device__ __forceinline__ void load8(const void* p, size_t i, int n, float (&f)[8]) {
  const bf16* h = reinterpret_cast<const bf16*>(p) + i;
  const float* q = reinterpret_cast<const float*>(p) + i;
  if (n < 8) {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = j < n ? (BF ? bf2f(h[j]) : q[j]) : 0.f;
  } else if (BF) {
    const any_bf16x8 v = *reinterpret_cast<const any_bf16x8*>(h);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = bf2f(v[j]);
  } else {
    const any_f32x4 a = *reinterpret_cast<const any_f32x4*>(q), b = *reinterpret_cast<const any_f32x4*>(q + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = a[j];
      f[4 + j] = b[j];
    }
  }
}
__device__ __forceinline__ size_t act8_thread() { return ((size_t)blockIdx.y * gridDim.x + blockIdx.x) * 256 + threadIdx.x; }
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}

// 4 lanes per 32-column block, 8 values each
template <int BF>
__global__ void __launch_bounds__(256) act8_pack_kernel(Act8Args a) {
  const int nb = (a.N + A8_BLOCK - 1) / A8_BLOCK, q4 = nb * 4;
  const size_t i = act8_thread();
  if (i >= (size_t)a.M * q4) return;        // (whole blocks: a multiple of 4)
  const size_t row = i / q4;
  const int c = (int)(i % q4) * 8, n = a.N - c;
  float f[8];
  load8<BF>(a.x, row * a.ld + c, n, f);
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(f[j]));
  m = fmaxf(m, __shfl_xor(m, 1));
  m = fmaxf(m, __shfl_xor(m, 2));
  const int e = a8_exponent(m);
  const float inv = a8_scale((uint32_t)(127 - e));
  const uint32_t lo = a8_pack4(f[0], f[1], f[2], f[3], inv), hi = a8_pack4(f[4], f[5], f[6], f[7], inv);
  uint8_t* d = a.codes + row * a.ldc + c;
  if (n >= 8) {
    *reinterpret_cast<any_u32x2*>(d) = any_u32x2{lo, hi};
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) d[j] = (uint8_t)((j < 4 ? lo : hi) >> (8 * (j & 3)));
  }
  if ((i & 3) == 0) a.scales[row * nb + c / A8_BLOCK] = (uint8_t)(e + 127);
}

template <int BF>
__global__ void __launch_bounds__(256) act8_unpack_kernel(Act8Args a) {
  const int n8 = (a.N - 1) / 8 + 1, nb = (a.N - 1) / A8_BLOCK + 1;
  const size_t i = act8_thread();
  if (i >= (size_t)a.M * n8) return;
  const size_t row = i / n8;
  const int c = (int)(i % n8) * 8, n = a.N - c;
  const uint8_t* s = a.codes + row * a.ldc + c;
  bf16* h = reinterpret_cast<bf16*>(a.out) + row * a.ld + c;
  float* o = reinterpret_cast<float*>(a.out) + row * a.ld + c;
  uint2 w = make_uint2(0, 0);
  if (n >= 8) {
    w = __builtin_bit_cast(uint2, *reinterpret_cast<const any_u32x2*>(s));
  } else {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) (j < 4 ? w.x : w.y) |= (uint32_t)s[j] << (8 * (j & 3));
  }
  float f[8];
  a8_unpack8(w, a.scales[row * nb + c / A8_BLOCK], f);
  if (n < 8) {
#pragma unroll
    for (int j = 0; j < 7; ++j)
      if (j < n) {
        if (BF) h[j] = f2bf(f[j]);
        else o[j] = f[j];
      }
  } else if (BF) {
    any_bf16x8 v;
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = f2bf(f[j]);
    *reinterpret_cast<any_bf16x8*>(h) = v;
  } else {
    *reinterpret_cast<any_f32x4*>(o) = any_f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<any_f32x4*>(o + 4) = any_f32x4{f[4], f[5], f[6], f[7]};
  }
}

// (a launch has less than 2^32 threads in x)
static dim3 act8_grid(size_t threads) {
  const size_t n = (threads + 255) / 256, row = 1u << 23;
  return dim3((unsigned)(n < row ? n : row), (unsigned)((n + row - 1) / row));
}

HFM_API int hfm_act8_pack(const Act8Args* ap, hipStream_t st) {
  const Act8Args a = *ap;
  if (a.M < 0 || a.N < 0 || a.N > 0x7FFFFFE0) return (int)hipErrorInvalidValue;
  if (a.M == 0 || a.N == 0) return 0;
  const dim3 grid = act8_grid((size_t)a.M * ((a.N + A8_BLOCK - 1) / A8_BLOCK) * 4);
  if (a.bf) hipLaunchKernelGGL(act8_pack_kernel<1>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(act8_pack_kernel<0>, grid, dim3(256), 0, st, a);
  HFM_LAUNCH_CHECK();
}

HFM_API int hfm_act8_unpack(const Act8Args* ap, hipStream_t st) {
  const Act8Args a = *ap;
  if (a.M < 0 || a.N < 0 || a.N > 0x7FFFFFE0) return (int)hipErrorInvalidValue;
  if (a.M == 0 || a.N == 0) return 0;
  const dim3 grid = act8_grid((size_t)a.M * ((a.N - 1) / 8 + 1));
  if (a.bf) hipLaunchKernelGGL(act8_unpack_kernel<1>, grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL(act8_unpack_kernel<0>, grid, dim3(256), 0, st, a);
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_act8_args_bytes() { return (int)sizeof(Act8Args); }
