// Group norm with an activation over channels-last [B][S][C] tensors, forward and backward, with
// the 8-bit checkpoint of the input (mx8.h) written by the forward and read by the backward.
//
//   y = act(z), z = (x - mean) * rstd * gamma + beta, statistics over the S * C/G values of (b, g)
//   dz = dy act'(z), xh = (x - mean) rstd:  dgamma = sum dz xh, dbeta = sum dz,
//   dx = rstd (dz gamma - (s1 + xh s2) / m), s1 = sum_g dz gamma, s2 = sum_g dz gamma xh
#include "../mx8.h"

namespace {
enum GnAct : int { GN_NONE = 0, GN_RELU = 1, GN_RELU6 = 2, GN_SILU = 3 };

// NaN passes through every activation
PG_DEVICE float gn_act(float z, int act) {
  if (act == GN_RELU) return z < 0.f ? 0.f : z;
  if (act == GN_RELU6) return z < 0.f ? 0.f : z > 6.f ? 6.f : z;
  if (act == GN_SILU) return z / (1.f + __expf(-z));
  return z;
}

// act'(z) dy.  Which side of a border z lies on is decided from the operands as they are: within the
// fp32 rounding of the border (|z - border| below a bound on it) z is formed again in 64 bits.
PG_DEVICE float gn_dz(float dy, float x, float mean, float rstd, float g, float b, int act) {
  const float z = (x - mean) * rstd * g + b;
  if (act == GN_NONE) return dy;
  if (act == GN_SILU) {
    const float s = 1.f / (1.f + __expf(-z));
    return dy * (s * (1.f + z * (1.f - s)));
  }
  const float tol = 1e-6f * (fabsf(z) + 2.f * fabsf(b));
  bool in = z > 0.f && !(act == GN_RELU6 && z >= 6.f);
  if (fabsf(z) <= tol || (act == GN_RELU6 && fabsf(z - 6.f) <= tol)) {
    const double w = ((double)x - (double)mean) * (double)rstd * (double)g + (double)b;
    in = w > 0.0 && !(act == GN_RELU6 && w >= 6.0);
  }
  return in ? dy : 0.f;
}

template <class F> PG_DEVICE float block_sum(float v, F *sh) {
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  float s = 0.f;
  for (int i = 0; i < (int)(blockDim.x >> 6); ++i) s += sh[i];
  return s;
}

// one workgroup per (b, g): mean, then the squares about it
template <class T>
__global__ __launch_bounds__(256) void gn_stats_kernel(const T *__restrict__ x, float *__restrict__ mean,
                                                       float *__restrict__ rstd, long long S, int C, int G, float eps) {
  __shared__ float sh[4];
  const int cg = C / G;
  const long long b = blockIdx.x / G, n = S * cg;
  const T *src = x + b * S * C + (long long)(blockIdx.x % G) * cg;
  float a = 0.f;
  for (long long i = threadIdx.x; i < n; i += 256) a += tof(src[i / cg * C + i % cg]);
  const float mu = block_sum(a, sh) / (float)n;
  float v = 0.f;
  for (long long i = threadIdx.x; i < n; i += 256) {
    const float d = tof(src[i / cg * C + i % cg]) - mu;
    v += d * d;
  }
  v = block_sum(v, sh);
  if (threadIdx.x == 0) {
    mean[blockIdx.x] = mu;
    rstd[blockIdx.x] = 1.f / sqrtf(v / (float)n + eps);
  }
}

template <class T>
__global__ __launch_bounds__(256) void gn_apply_kernel(const T *__restrict__ x, const float *__restrict__ gamma,
                                                       const float *__restrict__ beta, const float *__restrict__ mean,
                                                       const float *__restrict__ rstd, T *__restrict__ y, long long n,
                                                       long long SC, int C, int G, int act) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int c = (int)(i % C);
    const long long k = i / SC * G + c / (C / G);
    const float z = (tof(x[i]) - mean[k]) * rstd[k] * (gamma ? gamma[c] : 1.f) + (beta ? beta[c] : 0.f);
    y[i] = fromf<T>(gn_act(z, act));
  }
}

// one workgroup per (b, c): sum dz, sum dz xh over S
template <class T>
__global__ __launch_bounds__(256) void gn_bwd_sums_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                          const uint8_t *__restrict__ q,
                                                          const uint8_t *__restrict__ qs,
                                                          const float *__restrict__ gamma,
                                                          const float *__restrict__ beta,
                                                          const float *__restrict__ mean,
                                                          const float *__restrict__ rstd, float *__restrict__ part,
                                                          long long S, int C, int G, int act) {
  __shared__ float sh[4];
  const long long b = blockIdx.x / C;
  const int c = blockIdx.x % C, nb = (C + kMxBlock - 1) / kMxBlock;
  const float mu = mean[b * G + c / (C / G)], rs = rstd[b * G + c / (C / G)];
  const float g = gamma ? gamma[c] : 1.f, be = beta ? beta[c] : 0.f;
  float a0 = 0.f, a1 = 0.f;
  for (long long s = threadIdx.x; s < S; s += 256) {
    const long long r = b * S + s, i = r * C + c;
    const float v = x ? tof(x[i]) : mx8_dec1(q[i]) * mx8_scale(qs[r * nb + c / kMxBlock]);
    const float dz = gn_dz(tof(dy[i]), v, mu, rs, g, be, act);
    a0 += dz;
    a1 += dz * ((v - mu) * rs);
  }
  a0 = block_sum(a0, sh);
  a1 = block_sum(a1, sh);
  if (threadIdx.x == 0) {
    part[(b * 2) * C + c] = a1;
    part[(b * 2 + 1) * C + c] = a0;
  }
}

template <class T>
__global__ __launch_bounds__(256) void gn_bwd_apply_kernel(const T *__restrict__ dy, const T *__restrict__ x,
                                                           const uint8_t *__restrict__ q,
                                                           const uint8_t *__restrict__ qs,
                                                           const float *__restrict__ gamma,
                                                           const float *__restrict__ beta,
                                                           const float *__restrict__ mean,
                                                           const float *__restrict__ rstd,
                                                           const float *__restrict__ part, T *__restrict__ dx,
                                                           long long n, long long S, int C, int G, int act) {
  const int cg = C / G, nb = (C + kMxBlock - 1) / kMxBlock;
  const float rm = 1.f / ((float)S * (float)cg);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int c = (int)(i % C), g0 = c / cg * cg;
    const long long r = i / C, b = r / S, k = b * G + c / cg;
    float s1 = 0.f, s2 = 0.f;
    for (int j = g0; j < g0 + cg; ++j) {
      const float g = gamma ? gamma[j] : 1.f;
      s2 += g * part[(b * 2) * C + j];
      s1 += g * part[(b * 2 + 1) * C + j];
    }
    const float v = x ? tof(x[i]) : mx8_dec1(q[i]) * mx8_scale(qs[r * nb + c / kMxBlock]);
    const float g = gamma ? gamma[c] : 1.f;
    const float dz = gn_dz(tof(dy[i]), v, mean[k], rstd[k], g, beta ? beta[c] : 0.f, act);
    dx[i] = fromf<T>(rstd[k] * (dz * g - (s1 + (v - mean[k]) * rstd[k] * s2) * rm));
  }
}

// out[j] = sum over rows of part[row][j], rows in order
__global__ __launch_bounds__(256) void gn_dparam_kernel(const float *__restrict__ part, float *__restrict__ out,
                                                        long long rows, int n) {
  const int j = blockIdx.x * 256 + threadIdx.x;
  if (j >= n) return;
  float a = 0.f;
  for (long long r = 0; r < rows; ++r) a += part[r * n + j];
  out[j] = a;
}

unsigned gn_grid(long long n) { return (unsigned)(n + 255 < 256ll * 65536 ? (n + 255) / 256 : 65536); }
}  // namespace

void launch_mx8_pack(int dt, const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st);

// dt: 0 bf16, 1 fp16, 2 fp32
long long gn_workspace_floats(int, long long B, long long, int C, int, int bwd) { return bwd ? 2 * B * C : 0; }

void launch_gn_fwd(int dt, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd,
                   uint8_t *q, uint8_t *qs, float *ws, long long B, long long S, int C, int G, float eps, int act,
                   hipStream_t st) {
  (void)ws;
  const long long n = B * S * C;
#define FWD(T)                                                                                                     \
  hipLaunchKernelGGL(gn_stats_kernel<T>, dim3((unsigned)(B * G)), dim3(256), 0, st, (const T *)x, mean, rstd, S, C, G, \
                     eps);                                                                                          \
  hipLaunchKernelGGL(gn_apply_kernel<T>, dim3(gn_grid(n)), dim3(256), 0, st, (const T *)x, gamma, beta, mean, rstd,  \
                     (T *)y, n, S *C, C, G, act)
  if (dt == 0) { FWD(bf16_t); }
  else if (dt == 1) { FWD(_Float16); }
  else { FWD(float); }
#undef FWD
  if (q) launch_mx8_pack(dt, x, q, qs, B * S, C, st);
}

void launch_gn_bwd(int dt, const void *dy, const void *x, const uint8_t *q, const uint8_t *qs, const float *gamma,
                   const float *beta, const float *mean, const float *rstd, void *dx, float *dgb, float *ws,
                   long long B, long long S, int C, int G, int act, hipStream_t st) {
  const long long n = B * S * C;
#define BWD(T)                                                                                                    \
  hipLaunchKernelGGL(gn_bwd_sums_kernel<T>, dim3((unsigned)(B * C)), dim3(256), 0, st, (const T *)dy, (const T *)x, q, \
                     qs, gamma, beta, mean, rstd, ws, S, C, G, act);                                               \
  hipLaunchKernelGGL(gn_bwd_apply_kernel<T>, dim3(gn_grid(n)), dim3(256), 0, st, (const T *)dy, (const T *)x, q, qs,  \
                     gamma, beta, mean, rstd, ws, (T *)dx, n, S, C, G, act)
  if (dt == 0) { BWD(bf16_t); }
  else if (dt == 1) { BWD(_Float16); }
  else { BWD(float); }
#undef BWD
  if (dgb) hipLaunchKernelGGL(gn_dparam_kernel, dim3((2 * C + 255) / 256), dim3(256), 0, st, ws, dgb, B, 2 * C);
}
