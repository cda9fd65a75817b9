// Activations to 8 bits and back (act8.h has the format).  Bound by the bytes: 2 (bf16) or 4 read
// and 1 + 1/32 written per value, and the reverse.
#include "act8.h"

struct Act8Args {
  const void* x;           // pack: values [M, N], row stride ld;  unpack: null
  uint8_t* codes;          // [M, N], row stride ldc
  uint8_t* scales;         // [M, ceil(N / 32)]
  void* out;               // unpack: values, row stride ld
  long ld, ldc;
  int M, N, bf;
};

template <int BF>
__device__ __forceinline__ void load8(const void* p, size_t i, float (&f)[8]) {
  if (BF) {
    const bf16x8 v = *reinterpret_cast<const bf16x8*>(reinterpret_cast<const bf16*>(p) + i);
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = bf2f(v[j]);
  } else {
    const float* q = reinterpret_cast<const float*>(p) + i;
    const f32x4 a = *reinterpret_cast<const f32x4*>(q), b = *reinterpret_cast<const f32x4*>(q + 4);
#pragma unroll
    for (int j = 0; j < 4; ++j) {
      f[j] = a[j];
      f[4 + j] = b[j];
    }
  }
}
__device__ __forceinline__ float finite_abs(float v) {
  const float a = fabsf(v);
  return a < INFINITY ? a : 0.f;
}

// 4 lanes per 32-column block, 8 values each (rows of 16-byte multiples)
template <int BF>
__global__ void __launch_bounds__(256) act8_pack_kernel(Act8Args a) {
  const int nb = (a.N + A8_BLOCK - 1) / A8_BLOCK, q4 = nb * 4;
  const size_t n = (size_t)a.M * q4;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= n) return;                       // (whole blocks: n is a multiple of 4)
  const size_t row = i / q4;
  const int c = (int)(i % q4) * 8;
  float f[8];
  if (c < a.N) {
    load8<BF>(a.x, row * a.ld + c, f);
  } else {
#pragma unroll
    for (int j = 0; j < 8; ++j) f[j] = 0.f;
  }
  float m = 0.f;
#pragma unroll
  for (int j = 0; j < 8; ++j) m = fmaxf(m, finite_abs(f[j]));
  m = fmaxf(m, __shfl_xor(m, 1));
  m = fmaxf(m, __shfl_xor(m, 2));
  const int e = a8_exponent(m);
  const float inv = a8_scale((uint32_t)(127 - e));
  if (c < a.N) {
    uint2 w;
    w.x = a8_pack4(f[0], f[1], f[2], f[3], inv);
    w.y = a8_pack4(f[4], f[5], f[6], f[7], inv);
    *reinterpret_cast<uint2*>(a.codes + row * a.ldc + c) = w;
  }
  if ((i & 3) == 0) a.scales[row * nb + c / A8_BLOCK] = (uint8_t)(e + 127);
}

// any width and alignment: one value per lane, 32 lanes per block
template <int BF>
__global__ void __launch_bounds__(256) act8_pack1_kernel(Act8Args a) {
  const int nb = (a.N + A8_BLOCK - 1) / A8_BLOCK;
  const size_t blk = (size_t)blockIdx.x * 8 + (threadIdx.x >> 5);
  if (blk >= (size_t)a.M * nb) return;      // (whole 32-lane halves)
  const size_t row = blk / nb;
  const int b = (int)(blk % nb), c = b * A8_BLOCK + (threadIdx.x & 31);
  float v = 0.f;
  if (c < a.N) v = BF ? bf2f(reinterpret_cast<const bf16*>(a.x)[row * a.ld + c])
                      : reinterpret_cast<const float*>(a.x)[row * a.ld + c];
  float m = finite_abs(v);
  for (int d = 16; d; d >>= 1) m = fmaxf(m, __shfl_xor(m, d));
  const int e = a8_exponent(m);
  if (c < a.N) a.codes[row * a.ldc + c] = (uint8_t)a8_pack4(v, 0.f, 0.f, 0.f, a8_scale((uint32_t)(127 - e)));
  if ((threadIdx.x & 31) == 0) a.scales[row * nb + b] = (uint8_t)(e + 127);
}

template <int BF>
__global__ void __launch_bounds__(256) act8_unpack_kernel(Act8Args a) {
  const int n8 = a.N / 8, nb = (a.N + A8_BLOCK - 1) / A8_BLOCK;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)a.M * n8) return;
  const size_t row = i / n8;
  const int c = (int)(i % n8) * 8;
  float f[8];
  a8_unpack8(*reinterpret_cast<const uint2*>(a.codes + row * a.ldc + c), a8_scale(a.scales[row * nb + c / A8_BLOCK]), f);
  if (BF) {
    bf16x8 o;
#pragma unroll
    for (int j = 0; j < 8; ++j) o[j] = f2bf(f[j]);
    *reinterpret_cast<bf16x8*>(reinterpret_cast<bf16*>(a.out) + row * a.ld + c) = o;
  } else {
    float* o = reinterpret_cast<float*>(a.out) + row * a.ld + c;
    *reinterpret_cast<f32x4*>(o) = f32x4{f[0], f[1], f[2], f[3]};
    *reinterpret_cast<f32x4*>(o + 4) = f32x4{f[4], f[5], f[6], f[7]};
  }
}

template <int BF>
__global__ void __launch_bounds__(256) act8_unpack1_kernel(Act8Args a) {
  const int nb = (a.N + A8_BLOCK - 1) / A8_BLOCK;
  const size_t i = (size_t)blockIdx.x * 256 + threadIdx.x;
  if (i >= (size_t)a.M * a.N) return;
  const size_t row = i / a.N;
  const int c = (int)(i % a.N);
  float f[8];
  a8_unpack8(make_uint2(a.codes[row * a.ldc + c], 0), a8_scale(a.scales[row * nb + c / A8_BLOCK]), f);
  if (BF) reinterpret_cast<bf16*>(a.out)[row * a.ld + c] = f2bf(f[0]);
  else reinterpret_cast<float*>(a.out)[row * a.ld + c] = f[0];
}

static bool act8_vec(const Act8Args& a, const void* values) {
  return ((uintptr_t)values % 16 == 0) && ((uintptr_t)a.codes % 8 == 0) && a.N % 8 == 0 && a.ldc % 8 == 0 &&
         a.ld % (a.bf ? 8 : 4) == 0;
}

static int act8_grid(size_t threads, dim3& grid) {
  const size_t n = (threads + 255) / 256;
  if (n == 0 || n > 0x7FFFFFFFull) return (int)hipErrorInvalidValue;
  grid = dim3((unsigned)n);
  return 0;
}

HFM_API int hfm_act8_pack(const Act8Args* ap, hipStream_t st) {
  const Act8Args a = *ap;
  if (a.M < 0 || a.N < 0) return (int)hipErrorInvalidValue;
  if (a.M == 0 || a.N == 0) return 0;
  const size_t nb = (a.N + A8_BLOCK - 1) / A8_BLOCK;
  dim3 grid;
  if (act8_vec(a, a.x)) {
    if (int rc = act8_grid((size_t)a.M * nb * 4, grid)) return rc;
    if (a.bf) hipLaunchKernelGGL(act8_pack_kernel<1>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(act8_pack_kernel<0>, grid, dim3(256), 0, st, a);
  } else {
    if (int rc = act8_grid((size_t)a.M * nb * 32, grid)) return rc;
    if (a.bf) hipLaunchKernelGGL(act8_pack1_kernel<1>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(act8_pack1_kernel<0>, grid, dim3(256), 0, st, a);
  }
  HFM_LAUNCH_CHECK();
}

HFM_API int hfm_act8_unpack(const Act8Args* ap, hipStream_t st) {
  const Act8Args a = *ap;
  if (a.M < 0 || a.N < 0) return (int)hipErrorInvalidValue;
  if (a.M == 0 || a.N == 0) return 0;
  dim3 grid;
  if (act8_vec(a, a.out)) {
    if (int rc = act8_grid((size_t)a.M * (a.N / 8), grid)) return rc;
    if (a.bf) hipLaunchKernelGGL(act8_unpack_kernel<1>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(act8_unpack_kernel<0>, grid, dim3(256), 0, st, a);
  } else {
    if (int rc = act8_grid((size_t)a.M * a.N, grid)) return rc;
    if (a.bf) hipLaunchKernelGGL(act8_unpack1_kernel<1>, grid, dim3(256), 0, st, a);
    else hipLaunchKernelGGL(act8_unpack1_kernel<0>, grid, dim3(256), 0, st, a);
  }
  HFM_LAUNCH_CHECK();
}
HFM_API int hfm_act8_args_bytes() { return (int)sizeof(Act8Args); }
