// 8-bit activation checkpoints (mx8.h): pack, unpack, and the weight gradient of a linear layer
// or 1x1 convolution whose input was kept as one.
#include "../mx8.h"
#include "../vec.h"

#include <algorithm>
#include <stdexcept>

namespace {
constexpr int kHalfMax = 65504;

// i / d by a multiplication while i * d < 2^32 (i is below d + 1024 here); m = ceil(2^32 / d)
struct FastDiv {
  uint32_t d, m;
  explicit FastDiv(uint32_t n) : d(n), m(n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0) {}
  PG_DEVICE uint32_t div(uint32_t i) const { return d == 1 ? i : d < 32768 ? __umulhi(i, m) : i / d; }
};

// Pack and unpack stream the matrix: V channels a thread, U of them in flight, neighbouring threads on
// neighbouring vectors of a row.  Bound by memory.
constexpr int kU = 4, kThreads = 256;

// a workgroup's U * 256 slots of a [M][slots] grid: row and slot of the u-th of this thread
struct Slots {
  long long row0;
  uint32_t rem;
  PG_DEVICE Slots(uint32_t slots) {
    const unsigned long long first = (unsigned long long)blockIdx.x * (kU * kThreads);
    row0 = (long long)(first / slots);
    rem = (uint32_t)(first % slots);
  }
  PG_DEVICE void at(int u, const FastDiv &f, long long &row, uint32_t &slot) const {
    const uint32_t local = rem + u * kThreads + threadIdx.x, q = f.div(local);
    row = row0 + q;
    slot = local - q * f.d;
  }
};

// slots of a row: its blocks' 32 / V vectors each (the last block's may lie past C)
template <class T, int V>
__global__ __launch_bounds__(kThreads) void mx8_pack_kernel(const T *__restrict__ x, uint8_t *__restrict__ q,
                                                            uint8_t *__restrict__ qs, long long M, int C, int nb,
                                                            FastDiv f) {
  typedef Vec<T, V> X;
  const Slots s(f.d);
  typename X::raw d[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {   // a slot past the end reads the matrix's first values
    long long row;
    uint32_t slot;
    s.at(u, f, row, slot);
    const bool ok = row < M && slot * V < (uint32_t)C;
    d[u] = *reinterpret_cast<const typename X::raw *>(x + (ok ? row * C + slot * V : 0));
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    long long row;
    uint32_t slot;
    s.at(u, f, row, slot);
    const bool ok = row < M && slot * V < (uint32_t)C;
    float v[V];
    X::unpack(d[u], v);
    const int e = mx8_exp(block_amax<T, V>(d[u], ok));
    if (ok) {
      *reinterpret_cast<typename Codes<V>::raw *>(q + row * C + slot * V) = Codes<V>::encode(v, mx8_inv_scale(e));
      if (slot % (kMxBlock / V) == 0) qs[row * nb + slot / (kMxBlock / V)] = (uint8_t)e;
    }
  }
}

template <class T> PG_DEVICE float mx8_hold(float v) { return v; }
// half precision ends at 65504: a value that its block's step rounds up past that stays finite (NaN stays NaN)
template <> PG_DEVICE float mx8_hold<_Float16>(float v) {
  return v > (float)kHalfMax ? (float)kHalfMax : v < -(float)kHalfMax ? -(float)kHalfMax : v;
}

template <class T, int V>
__global__ __launch_bounds__(kThreads) void mx8_unpack_kernel(const uint8_t *__restrict__ q,
                                                              const uint8_t *__restrict__ qs, T *__restrict__ x,
                                                              long long M, int C, int nb, FastDiv f) {
  const Slots s(f.d);
  typename Codes<V>::raw d[kU];
  uint8_t e[kU];
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    long long row;
    uint32_t slot;
    s.at(u, f, row, slot);
    const bool ok = row < M;
    d[u] = *reinterpret_cast<const typename Codes<V>::raw *>(q + (ok ? row * C + slot * V : 0));
    e[u] = qs[ok ? row * nb + slot * V / kMxBlock : 0];
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    long long row;
    uint32_t slot;
    s.at(u, f, row, slot);
    float v[V];
    Codes<V>::decode(d[u], mx8_scale(e[u]), v);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = mx8_hold<T>(v[j]);
    if (row < M) *reinterpret_cast<typename Vec<T, V>::raw *>(x + row * C + slot * V) = Vec<T, V>::pack(v);
  }
}

// ---------------------------------------------------------------------------
// dW[n][k] = sum_m dY[m][n] X[m][k].  The contraction runs over the rows of both operands, so both
// are read from shared memory transposed (ds_read_tr16_b64: 4 rows of a column a lane).  The codes'
// scales change with the row, so they are decoded on their way into shared memory: to bf16 exactly
// (4 significant bits), 2 an instruction.
//   tile     TN x TK outputs, 4 waves of QN x QK; 64 rows a step, two buffers: the next step's rows
//            are in registers while this one's are multiplied
//   rows     of the tile in shared memory are 32 bytes longer than the data: the 4 rows of a
//            16-lane group of a transposed read then lie in different banks
//   split    the M rows are cut into `splits` so that two workgroups a CU have work; each writes a
//            partial [N * K + N] and a second kernel adds them in order
// ---------------------------------------------------------------------------
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
constexpr int kMK = 64;

struct WgradArgs {
  const void *dy;
  const uint8_t *q, *qs;
  float *out, *db;        // splits == 1: dW, db; else partials [splits][N * K (+ N)]
  int M, N, K, nb;
  int tn, tk, splits, rows;   // tiles, row splits, rows of a split (a multiple of kMK)
  long long pitch;            // floats of a partial
};

template <class T> PG_DEVICE f32x4_t wg_mfma(s16x8_t a, s16x8_t b, f32x4_t c);
template <> PG_DEVICE f32x4_t wg_mfma<bf16_t>(s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8_t, a), __builtin_bit_cast(bf16x8_t, b), c, 0, 0, 0);
}
template <> PG_DEVICE f32x4_t wg_mfma<_Float16>(s16x8_t a, s16x8_t b, f32x4_t c) {
  return __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8_t, a), __builtin_bit_cast(f16x8_t, b), c, 0, 0, 0);
}

// 8 codes of one block -> 8 values of T
template <class T> PG_DEVICE uint4 wg_decode(uint2 c, uint8_t e) {
  const float sc = mx8_scale(e);
  uint4 r;
  if constexpr (__is_same(T, bf16_t)) {
    r.x = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, sc, false));
    r.y = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.x, sc, true));
    r.z = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, sc, false));
    r.w = __builtin_bit_cast(uint32_t, __builtin_amdgcn_cvt_scalef32_pk_bf16_fp8(c.y, sc, true));
  } else {
    float v[8];
    Codes<8>::decode(c, sc, v);
#pragma unroll
    for (int j = 0; j < 8; ++j) v[j] = mx8_hold<T>(v[j]);
    r = Vec<T, 8>::pack(v);
  }
  return r;
}

// ALN: rows of dY and of the codes begin at multiples of 8 values
template <class T, int TN, int TK, int WN, int WK, bool ALN>
__global__ __launch_bounds__(256) void mx8_wgrad_kernel(const WgradArgs a) {
  static_assert(WN * WK == 4, "4 waves");
  constexpr int QN = TN / WN, QK = TK / WK, RN = QN / 16, RK = QK / 16;
  constexpr int PA = TN * 2 + 32, PB = TK * 2 + 32;             // row pitches in bytes
  constexpr int CA = TN / 8, CB = TK / 8;                       // 8-value chunks of a row
  constexpr int NA = kMK * CA / 256, NB = (kMK * CB + 255) / 256;   // chunks a thread
  __shared__ __attribute__((aligned(16))) char smem[2][kMK * (PA + PB)];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // neighbouring tiles of one row split on one XCD, whose L2 holds the rows they share
  const int total = a.tn * a.tk * a.splits, per = total / 8;
  int id = blockIdx.x;
  if (id < per * 8) id = (id & 7) * per + (id >> 3);
  const int split = id / (a.tn * a.tk), tile = id % (a.tn * a.tk);
  const int n0 = (tile / a.tk) * TN, k0 = (tile % a.tk) * TK;
  const int mb = split * a.rows, me = min(a.M, mb + a.rows);
  const T *dy = static_cast<const T *>(a.dy);

  uint4 ra[NA];
  uint2 rb[NB];
  uint8_t re[NB];
  // chunk i of this thread: row, first column
  auto load = [&](int m0) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int s = t + i * 256, m = m0 + s / CA, n = n0 + s % CA * 8;
      if constexpr (ALN) {
        const bool ok = m < me && n < a.N;
        const uint4 v = *reinterpret_cast<const uint4 *>(dy + (ok ? (long long)m * a.N + n : 0));
        ra[i] = ok ? v : make_uint4(0, 0, 0, 0);
      } else {
        struct alignas(16) { T v[8]; } w;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool ok = m < me && n + j < a.N;
          const T v = dy[ok ? (long long)m * a.N + n + j : 0];
          w.v[j] = ok ? v : (T)0;
        }
        ra[i] = __builtin_bit_cast(uint4, w);
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int s = t + i * 256, m = m0 + s / CB, k = k0 + s % CB * 8;
      const bool row = m < me && s < kMK * CB;
      if constexpr (ALN) {
        const bool ok = row && k < a.K;
        const uint2 v = *reinterpret_cast<const uint2 *>(a.q + (ok ? (long long)m * a.K + k : 0));
        rb[i] = ok ? v : make_uint2(0, 0);
        re[i] = a.qs[ok ? (long long)m * a.nb + k / kMxBlock : 0];
      } else {
        struct alignas(8) { uint8_t v[8]; } w;
#pragma unroll
        for (int j = 0; j < 8; ++j) {
          const bool ok = row && k + j < a.K;
          const uint8_t v = a.q[ok ? (long long)m * a.K + k + j : 0];
          w.v[j] = ok ? v : 0;
        }
        rb[i] = __builtin_bit_cast(uint2, w);
        re[i] = a.qs[row && k < a.K ? (long long)m * a.nb + k / kMxBlock : 0];
      }
    }
  };
  float sum[8] = {};   // db: this thread's columns (a thread's chunks of dY are one column's, 256 % CA == 0)
  const bool bias = a.db && k0 == 0;
  auto put = [&](int buf) {
#pragma unroll
    for (int i = 0; i < NA; ++i) {
      const int s = t + i * 256;
      *reinterpret_cast<uint4 *>(smem[buf] + s / CA * PA + s % CA * 16) = ra[i];
      if (bias) {
        float v[8];
        Vec<T, 8>::unpack(ra[i], v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += v[j];
      }
    }
#pragma unroll
    for (int i = 0; i < NB; ++i) {
      const int s = t + i * 256;
      if (kMK * CB % 256 == 0 || s < kMK * CB)
        *reinterpret_cast<uint4 *>(smem[buf] + kMK * PA + s / CB * PB + s % CB * 16) = wg_decode<T>(rb[i], re[i]);
    }
  };

  f32x4_t acc[RN][RK];
#pragma unroll
  for (int i = 0; i < RN; ++i)
#pragma unroll
    for (int j = 0; j < RK; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int wn = wave / WK * QN, wk = wave % WK * QK;
  // transposed reads: lane (g = lane / 16, i = lane % 16) asks for row 8 g + i / 4 (then + 4), 8-byte
  // piece i % 4 of a 16-column block, and receives those rows of column i
  const int trow = 8 * (lane >> 4) + ((lane & 15) >> 2), tc = (lane & 3) * 8;
  auto mma = [&](int buf) {
    const char *A = smem[buf], *B = smem[buf] + kMK * PA;
#pragma unroll
    for (int sub = 0; sub < kMK / 32; ++sub) {
      s16x8_t fa[RN], fb[RK];
#pragma unroll
      for (int i = 0; i < RN; ++i) {
        const char *p = A + (sub * 32 + trow) * PA + (wn + i * 16) * 2 + tc;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * PA));
        fa[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int j = 0; j < RK; ++j) {
        const char *p = B + (sub * 32 + trow) * PB + (wk + j * 16) * 2 + tc;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * PB));
        fb[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int i = 0; i < RN; ++i)
#pragma unroll
        for (int j = 0; j < RK; ++j) acc[i][j] = wg_mfma<T>(fa[i], fb[j], acc[i][j]);
    }
  };

  if (mb < me) {
    load(mb);
    put(0);
    __syncthreads();
    int buf = 0;
    for (int m0 = mb; m0 < me; m0 += kMK, buf ^= 1) {
      const bool more = m0 + kMK < me;
      if (more) load(m0 + kMK);
      mma(buf);
      if (more) put(buf ^ 1);
      __syncthreads();
    }
  }
  float *out = a.out + (a.splits > 1 ? split * a.pitch : 0);
#pragma unroll
  for (int i = 0; i < RN; ++i)
#pragma unroll
    for (int j = 0; j < RK; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn + i * 16 + 4 * (lane >> 4) + r, k = k0 + wk + j * 16 + (lane & 15);
        if (n < a.N && k < a.K) out[(long long)n * a.K + k] = acc[i][j][r];
      }
  if (!bias) return;
  // the 256 / CA threads of a column chunk, in order
  float *sh = reinterpret_cast<float *>(smem[0]);
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[t * 8 + j] = sum[j];
  __syncthreads();
  float *db = a.splits > 1 ? out + (long long)a.N * a.K : a.db;
  if (t < TN && n0 + t < a.N) {
    float s = 0.f;
    for (int r = 0; r < 256 / CA; ++r) s += sh[(r * CA + t / 8) * 8 + t % 8];
    db[n0 + t] = s;
  }
}

// out[i] = sum over the splits of part[s][i]: 1024 / CB stripes of splits for CB groups of 4 values
template <int CB>
__global__ __launch_bounds__(1024) void mx8_join_kernel(const float *__restrict__ part, long long pitch, int splits,
                                                        long long nk, int nb, float *__restrict__ dw,
                                                        float *__restrict__ db) {
  constexpr int ST = 1024 / CB;
  __shared__ float4 sh[ST][CB];
  const int col = threadIdx.x % CB, st = threadIdx.x / CB;
  const long long i = ((long long)blockIdx.x * CB + col) * 4;
  float4 s = make_float4(0.f, 0.f, 0.f, 0.f);
  if (i < pitch)
#pragma unroll 4
    for (int r = st; r < splits; r += ST) {
      const float4 v = *reinterpret_cast<const float4 *>(part + r * pitch + i);
      s.x += v.x;
      s.y += v.y;
      s.z += v.z;
      s.w += v.w;
    }
  sh[st][col] = s;
  __syncthreads();
  if (st) return;
#pragma unroll 4
  for (int r = 1; r < ST; ++r) {
    const float4 v = sh[r][col];
    s.x += v.x;
    s.y += v.y;
    s.z += v.z;
    s.w += v.w;
  }
  const float o[4] = {s.x, s.y, s.z, s.w};
#pragma unroll
  for (int j = 0; j < 4; ++j) {
    if (i + j < nk) dw[i + j] = o[j];
    else if (i + j < nk + nb) db[i + j - nk] = o[j];
  }
}

struct WgradPlan {
  int kind;   // 0: 128 x 128, 1: 256 x 32, 2: 32 x 256, 3: 64 x 64
  int tn, tk, splits, rows;
  long long pitch;
};
const int kTileN[4] = {128, 256, 32, 64}, kTileK[4] = {128, 32, 256, 64};

WgradPlan wgrad_plan(int M, int N, int K) {
  WgradPlan p{};
  auto tiles = [&](int i) { return (long long)((N + kTileN[i] - 1) / kTileN[i]) * ((K + kTileK[i] - 1) / kTileK[i]); };
  // Narrow weights take the tile that reads the wide operand once; others the square of which less is
  // padding.
  p.kind = K <= 32 ? 1 : N <= 32 ? 2 : tiles(3) * 64 * 64 * 3 < tiles(0) * 128 * 128 * 2 ? 3 : 0;
  p.tn = (N + kTileN[p.kind] - 1) / kTileN[p.kind];
  p.tk = (K + kTileK[p.kind] - 1) / kTileK[p.kind];
  const long long t = (long long)p.tn * p.tk;
  if (t > 0x7fffffff) throw std::invalid_argument("mx8_wgrad: N * K is too large");
  const int steps = (M + kMK - 1) / kMK;
  long long s = std::max<long long>(1, std::min<long long>(512 / t, steps / 4));
  p.rows = (int)((steps + s - 1) / s) * kMK;
  p.splits = (int)(((long long)M + p.rows - 1) / p.rows);
  p.pitch = ((long long)N * K + N + 3) / 4 * 4;
  return p;
}

template <class T, bool ALN> void wgrad_go(const WgradPlan &p, const WgradArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(p.tn * p.tk * p.splits));
  if (p.kind == 0) hipLaunchKernelGGL((mx8_wgrad_kernel<T, 128, 128, 2, 2, ALN>), grid, dim3(256), 0, st, a);
  else if (p.kind == 1) hipLaunchKernelGGL((mx8_wgrad_kernel<T, 256, 32, 4, 1, ALN>), grid, dim3(256), 0, st, a);
  else if (p.kind == 2) hipLaunchKernelGGL((mx8_wgrad_kernel<T, 32, 256, 1, 4, ALN>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mx8_wgrad_kernel<T, 64, 64, 2, 2, ALN>), grid, dim3(256), 0, st, a);
}

unsigned slot_grid(long long M, long long slots) {
  const long long n = (M * slots + kU * kThreads - 1) / (kU * kThreads);
  if (n > 0x7fffffff) throw std::invalid_argument("mx8: M * C is too large");
  return (unsigned)n;
}
int vec_of(int C, int most) {
  while (C % most) most >>= 1;
  return most;
}
}  // namespace

// dt: 0 bf16, 1 fp16, 2 fp32
void launch_mx8_pack(int dt, const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st) {
  if (M <= 0) return;
  const int nb = (C + kMxBlock - 1) / kMxBlock, V = vec_of(C, dt == 2 ? 4 : 8);
  const FastDiv f((uint32_t)nb * (kMxBlock / V));
  const dim3 grid(slot_grid(M, f.d));
#define PACK(T, N) hipLaunchKernelGGL((mx8_pack_kernel<T, N>), grid, dim3(kThreads), 0, st, (const T *)x, q, qs, M, C, nb, f)
#define PACK_V(T)             \
  if (V == 4) PACK(T, 4);     \
  else if (V == 2) PACK(T, 2); \
  else PACK(T, 1)
  if (dt == 2) { PACK_V(float); }
  else if (dt == 0) { if (V == 8) PACK(bf16_t, 8); else PACK_V(bf16_t); }
  else { if (V == 8) PACK(_Float16, 8); else PACK_V(_Float16); }
#undef PACK_V
#undef PACK
}

void launch_mx8_unpack(int dt, const uint8_t *q, const uint8_t *qs, void *x, long long M, int C, hipStream_t st) {
  if (M <= 0) return;
  const int nb = (C + kMxBlock - 1) / kMxBlock, V = vec_of(C, dt == 2 ? 4 : 8);
  const FastDiv f((uint32_t)(C / V));
  const dim3 grid(slot_grid(M, f.d));
#define UNPACK(T, N) hipLaunchKernelGGL((mx8_unpack_kernel<T, N>), grid, dim3(kThreads), 0, st, q, qs, (T *)x, M, C, nb, f)
#define UNPACK_V(T)              \
  if (V == 4) UNPACK(T, 4);      \
  else if (V == 2) UNPACK(T, 2); \
  else UNPACK(T, 1)
  if (dt == 2) { UNPACK_V(float); }
  else if (dt == 0) { if (V == 8) UNPACK(bf16_t, 8); else UNPACK_V(bf16_t); }
  else { if (V == 8) UNPACK(_Float16, 8); else UNPACK_V(_Float16); }
#undef UNPACK_V
#undef UNPACK
}

long long mx8_wgrad_workspace_floats(int M, int N, int K) {
  if (M <= 0) return 0;
  const WgradPlan p = wgrad_plan(M, N, K);
  return p.splits > 1 ? p.splits * p.pitch : 0;
}

void launch_mx8_wgrad(int dt, const void *dy, const uint8_t *q, const uint8_t *qs, float *dw, float *db, float *ws,
                      int M, int N, int K, hipStream_t st) {
  const WgradPlan p = wgrad_plan(M, N, K);
  const WgradArgs a{dy, q, qs, p.splits > 1 ? ws : dw, db, M, N, K, (K + kMxBlock - 1) / kMxBlock,
                    p.tn, p.tk, p.splits, p.rows, p.pitch};
  const bool aln = N % 8 == 0 && K % 8 == 0;
  if (dt == 0) aln ? wgrad_go<bf16_t, true>(p, a, st) : wgrad_go<bf16_t, false>(p, a, st);
  else aln ? wgrad_go<_Float16, true>(p, a, st) : wgrad_go<_Float16, false>(p, a, st);
  if (p.splits == 1) return;
  const long long nk = (long long)N * K, n4 = p.pitch / 4;
  const int nb = db ? N : 0;
#define JOIN(CB)                                                                                                       \
  hipLaunchKernelGGL(mx8_join_kernel<CB>, dim3((unsigned)((n4 + CB - 1) / CB)), dim3(1024), 0, st, ws, p.pitch, p.splits, \
                     nk, nb, dw, db)
  if (n4 >= 256 * 256) JOIN(256);   // enough column blocks to fill the chip
  else if (n4 >= 64 * 256) JOIN(64);
  else JOIN(16);
#undef JOIN
}
