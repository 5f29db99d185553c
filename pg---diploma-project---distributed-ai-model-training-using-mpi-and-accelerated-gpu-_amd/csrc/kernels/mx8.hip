// 8-bit activation checkpoints (mx8.h): pack, unpack, and the weight gradient of a linear layer
// or 1x1 convolution whose input was kept as one.
#include "../mx8.h"

#include <stdexcept>

namespace {
constexpr int kHalfMax = 65504;

// one thread per block of 32 channels
template <class T>
__global__ __launch_bounds__(256) void mx8_pack_kernel(const T *__restrict__ x, uint8_t *__restrict__ q,
                                                       uint8_t *__restrict__ qs, long long M, int C, int nb) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < M * nb; i += (long long)gridDim.x * 256) {
    const long long m = i / nb;
    const int c0 = (int)(i % nb) * kMxBlock, c1 = min(C, c0 + kMxBlock);
    float a = 0.f;
    for (int c = c0; c < c1; ++c) a = fmaxf(a, mx8_mag(tof(x[m * C + c])));
    const int e = mx8_exp(a);
    const float inv = mx8_inv_scale(e);
    for (int c = c0; c < c1; ++c) q[m * C + c] = mx8_enc1(tof(x[m * C + c]) * inv);
    qs[i] = (uint8_t)e;
  }
}

template <class T> PG_DEVICE T mx8_out(float v) { return fromf<T>(v); }
// half precision ends at 65504: a value that its block's step rounds up past that stays finite
template <> PG_DEVICE _Float16 mx8_out<_Float16>(float v) {
  return (_Float16)(v > (float)kHalfMax ? (float)kHalfMax : v < -(float)kHalfMax ? -(float)kHalfMax : v);
}

template <class T>
__global__ __launch_bounds__(256) void mx8_unpack_kernel(const uint8_t *__restrict__ q,
                                                         const uint8_t *__restrict__ qs, T *__restrict__ x,
                                                         long long M, int C, int nb) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < M * C; i += (long long)gridDim.x * 256) {
    const long long m = i / C;
    const int c = (int)(i % C);
    x[i] = mx8_out<T>(mx8_dec1(q[i]) * mx8_scale(qs[m * nb + c / kMxBlock]));
  }
}

// dW[n][k] = sum_m dY[m][n] X[m][k]; 64 x 64 outputs a workgroup, 4 x 4 a thread
template <class T>
__global__ __launch_bounds__(256) void mx8_wgrad_kernel(const T *__restrict__ dy, const uint8_t *__restrict__ q,
                                                        const uint8_t *__restrict__ qs, float *__restrict__ dw,
                                                        float *__restrict__ db, int M, int N, int K, int nb) {
  __shared__ float As[16][64], Bs[16][64];
  const int tid = threadIdx.x, tx = tid % 16, ty = tid / 16;
  const int n0 = blockIdx.y * 64, k0 = blockIdx.x * 64;
  float acc[4][4] = {};
  float sum = 0.f;
  for (int m0 = 0; m0 < M; m0 += 16) {
    for (int i = tid; i < 16 * 64; i += 256) {
      const int mm = i / 64, c = i % 64, m = m0 + mm;
      As[mm][c] = m < M && n0 + c < N ? tof(dy[(long long)m * N + n0 + c]) : 0.f;
      Bs[mm][c] = m < M && k0 + c < K ? tof(mx8_out<T>(mx8_dec1(q[(long long)m * K + k0 + c]) *
                                                        mx8_scale(qs[(long long)m * nb + (k0 + c) / kMxBlock])))
                                    : 0.f;
    }
    __syncthreads();
    for (int mm = 0; mm < 16; ++mm) {
      if (tid < 64) sum += As[mm][tid];
#pragma unroll
      for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = fmaf(As[mm][ty * 4 + i], Bs[mm][tx * 4 + j], acc[i][j]);
    }
    __syncthreads();
  }
#pragma unroll
  for (int i = 0; i < 4; ++i)
#pragma unroll
    for (int j = 0; j < 4; ++j)
      if (n0 + ty * 4 + i < N && k0 + tx * 4 + j < K)
        dw[(long long)(n0 + ty * 4 + i) * K + k0 + tx * 4 + j] = acc[i][j];
  if (db && blockIdx.x == 0 && tid < 64 && n0 + tid < N) db[n0 + tid] = sum;
}
}  // namespace

// dt: 0 bf16, 1 fp16, 2 fp32
void launch_mx8_pack(int dt, const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st) {
  const int nb = (C + kMxBlock - 1) / kMxBlock;
  const long long n = M * nb;
  if (n <= 0) return;
  const dim3 grid((unsigned)(n + 255 < 256ll * 65536 ? (n + 255) / 256 : 65536));
#define PACK(T) hipLaunchKernelGGL(mx8_pack_kernel<T>, grid, dim3(256), 0, st, (const T *)x, q, qs, M, C, nb)
  if (dt == 0) PACK(bf16_t);
  else if (dt == 1) PACK(_Float16);
  else PACK(float);
#undef PACK
}

void launch_mx8_unpack(int dt, const uint8_t *q, const uint8_t *qs, void *x, long long M, int C, hipStream_t st) {
  const int nb = (C + kMxBlock - 1) / kMxBlock;
  const long long n = M * C;
  if (n <= 0) return;
  const dim3 grid((unsigned)(n + 255 < 256ll * 65536 ? (n + 255) / 256 : 65536));
#define UNPACK(T) hipLaunchKernelGGL(mx8_unpack_kernel<T>, grid, dim3(256), 0, st, q, qs, (T *)x, M, C, nb)
  if (dt == 0) UNPACK(bf16_t);
  else if (dt == 1) UNPACK(_Float16);
  else UNPACK(float);
#undef UNPACK
}

long long mx8_wgrad_workspace_floats(int, int, int) { return 0; }

void launch_mx8_wgrad(int dt, const void *dy, const uint8_t *q, const uint8_t *qs, float *dw, float *db, float *ws,
                      int M, int N, int K, hipStream_t st) {
  (void)ws;
  const int nb = (K + kMxBlock - 1) / kMxBlock;
  const dim3 grid((K + 63) / 64, (N + 63) / 64);
  if (dt == 0)
    hipLaunchKernelGGL(mx8_wgrad_kernel<bf16_t>, grid, dim3(256), 0, st, (const bf16_t *)dy, q, qs, dw, db, M, N, K, nb);
  else
    hipLaunchKernelGGL(mx8_wgrad_kernel<_Float16>, grid, dim3(256), 0, st, (const _Float16 *)dy, q, qs, dw, db, M, N, K,
                       nb);
}
