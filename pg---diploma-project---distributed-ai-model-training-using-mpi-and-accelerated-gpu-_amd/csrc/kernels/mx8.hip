// 8-bit activation checkpoints (mx8.h): pack, unpack, and the weight gradient of a linear layer
// or 1x1 convolution whose input was kept as one.
#include "../mx8.h"
#include "../vec.h"

#include <algorithm>
#include <stdexcept>
#include <type_traits>

namespace {
constexpr int kHalfMax = 65504;

// i / d by a multiplication while i * d < 2^32 (i is below d + 8192 here); m = ceil(2^32 / d)
struct FastDiv {
  uint32_t d, m;
  explicit FastDiv(uint32_t n) : d(n), m(n > 1 ? (uint32_t)(((1ull << 32) + n - 1) / n) : 0) {}
  PG_DEVICE uint32_t div(uint32_t i) const { return d == 1 ? i : d < 32768 ? __umulhi(i, m) : i / d; }
};

// Pack and unpack stream the matrix: V channels a thread, U of them in flight, neighbouring threads on
// neighbouring vectors of a row.  Bound by memory: pack 401408 x 144 bf16 33 us, 5.3 TB/s; unpack 100352 x 960
// bf16 50 us, 5.8 TB/s (a copy of 1 GiB: 5.1).
// ANY: rows begin anywhere, and a row's last vector may be cut short: it is read from C - V on and shifted,
// and its codes are written one by one.
constexpr int kU = 4, kThreads = 256;
// Work-items of a launch: the runtime takes 2^32 and more without a word and runs what is left modulo 2^32
constexpr long long kMostItems = 0xffffffffll, kMostWgs = kMostItems / kThreads;

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

// what V values of a row have in memory at p, at any alignment of theirs, without the first `cut` values
template <class R, class P> PG_DEVICE R load_cut(const P *p, int cut) {
  R r;
  __builtin_memcpy(&r, p, sizeof(R));
  const uint32_t s = cut * (uint32_t)sizeof(P) * 8;
  if constexpr (sizeof(R) == 16) {
    const uint64_t lo = r.x | (uint64_t)r.y << 32, hi = r.z | (uint64_t)r.w << 32, t = s & 63;
    const uint64_t l = s < 64 ? lo >> t | (t ? hi << (64 - t) : 0) : hi >> t, h = s < 64 ? hi >> t : 0;
    return make_uint4((uint32_t)l, (uint32_t)(l >> 32), (uint32_t)h, (uint32_t)(h >> 32));
  } else if constexpr (sizeof(R) == 8) {
    const uint64_t v = (r.x | (uint64_t)r.y << 32) >> s;
    return make_uint2((uint32_t)v, (uint32_t)(v >> 32));
  } else {
    return r >> s;
  }
}
// the first n of V values, at any alignment of theirs
template <int V, class R, class P> PG_DEVICE void store_cut(P *p, const R &r, int n) {
  if (n >= V) {
    __builtin_memcpy(p, &r, sizeof(R));
  } else {
    struct alignas(sizeof(R)) Parts { P v[V]; };
    const Parts a = __builtin_bit_cast(Parts, r);
#pragma unroll
    for (int j = 0; j < V; ++j)
      if (j < n) p[j] = a.v[j];
  }
}

// slots of a row: its blocks' 32 / V vectors each (the last block's may lie past C)
template <class T, int V, bool ANY>
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
    if constexpr (ANY) {
      const int cut = ok ? max(0, (int)(slot * V) + V - C) : 0;
      d[u] = load_cut<typename X::raw>(x + (ok ? row * C + slot * V - cut : 0), cut);
    } else {
      d[u] = *reinterpret_cast<const typename X::raw *>(x + (ok ? row * C + slot * V : 0));
    }
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
      const typename Codes<V>::raw c = Codes<V>::encode(v, mx8_inv_scale(e));
      if constexpr (ANY) store_cut<V>(q + row * C + slot * V, c, C - (int)(slot * V));
      else *reinterpret_cast<typename Codes<V>::raw *>(q + row * C + slot * V) = c;
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

// Rows that begin anywhere: the matrix as one run of vectors, so that codes and values are aligned.
// V neighbouring values lie in three blocks at most, whose scales are neighbours too.
template <class T, int V>
__global__ __launch_bounds__(kThreads) void mx8_unpack_run_kernel(const uint8_t *__restrict__ q,
                                                                  const uint8_t *__restrict__ qs, T *__restrict__ x,
                                                                  long long M, int C, int nb, FastDiv f) {
  const unsigned long long first = (unsigned long long)blockIdx.x * (kU * kThreads * V);
  const long long total = M * C, row0 = (long long)(first / (uint32_t)C), last = M * nb - 1;
  const uint32_t rem = (uint32_t)(first % (uint32_t)C);
  typename Codes<V>::raw d[kU];
  uint8_t e[kU][3];
  int n0[kU], n1[kU];   // values of the first and of the second block
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const uint32_t at = (u * kThreads + threadIdx.x) * V, local = rem + at, r = f.div(local), c = local - r * C;
    const long long i = (long long)first + at, k = (row0 + r) * nb + c / kMxBlock;
    const int cut = (int)min((long long)V, max(0ll, i + V - total));   // V: nothing left, the last vector is read
    d[u] = load_cut<typename Codes<V>::raw>(q + min(i, total - V), cut % V);
#pragma unroll
    for (int j = 0; j < 3; ++j) e[u][j] = qs[min(k + j, last)];
    n0[u] = min(kMxBlock - (int)(c % kMxBlock), C - (int)c);
    const int c1 = (int)c + n0[u];
    n1[u] = n0[u] + min(kMxBlock, c1 < C ? C - c1 : C);
  }
#pragma unroll
  for (int u = 0; u < kU; ++u) {
    const long long i = (long long)first + (u * kThreads + threadIdx.x) * V;
    float v[V];
    Codes<V>::decode(d[u], 1.f, v);
    const float s0 = mx8_scale(e[u][0]), s1 = mx8_scale(e[u][1]), s2 = mx8_scale(e[u][2]);
#pragma unroll
    for (int j = 0; j < V; ++j) v[j] = mx8_hold<T>(v[j] * (j < n0[u] ? s0 : j < n1[u] ? s1 : s2));
    if (i < total) store_cut<V>(x + i, Vec<T, V>::pack(v), (int)min((long long)V, total - i));
  }
}

// ---------------------------------------------------------------------------
// dW[n][k] = sum_m dY[m][n] X[m][k].  The contraction runs over the rows of both operands, so both
// are read from shared memory transposed (ds_read_tr16_b64: 4 rows of a column a lane).  The codes'
// scales change with the row, so they are decoded on their way into shared memory: to bf16 exactly
// (4 significant bits), 2 an instruction.
//   tile     W x W outputs, 4 waves of a quarter each; 64 rows a step, two buffers in shared memory and
//            two steps in registers or on their way (25088 x 1024 x 1024: kernel 85 us; 100 with one, and
//            with four the registers' moves cost more than is gained; 91 with 256 x 256 and 8 waves)
//   rows     of the tile in shared memory keep their 32-byte pieces in an order that depends on the
//            row (wg_swz), so that transposed reads meet no bank twice
//   split    the M rows are cut into `splits` so that every CU has two workgroups; each writes a
//            partial [N * K + N] and a second kernel adds them in order
// A call with its join: 25088 x 1024 x 1024 81 us, 650 TFLOP/s (a step's reads, decoding, products and barrier
// follow one another, and two workgroups a CU hide half of it); 401408 x 144 x 24 37 us, 3.4 TB/s; 128 x 1000 x
// 2048 7 us, most of it the launch and the first loads' latency.
// ---------------------------------------------------------------------------
typedef short s16x4_t __attribute__((ext_vector_type(4)));
typedef __attribute__((address_space(3))) s16x4_t lds_s16x4_t;
typedef _Float16 f16x8_t __attribute__((ext_vector_type(8)));
typedef __bf16 bf16x2_t __attribute__((ext_vector_type(2)));
constexpr int kMK = 64, kAhead = 2;

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

// What a thread holds of a chunk: itself or, where rows are not aligned, the aligned words that it lies in,
// `shift` bytes into the first.
template <bool ALN> struct WgRaw {
  typedef uint4 a;
  typedef uint2 b;
  static PG_DEVICE uint4 pack(const uint4 &v, uint32_t) { return v; }
  static PG_DEVICE uint2 pack(const uint2 &v, uint32_t) { return v; }
};
template <> struct WgRaw<false> {
  struct a { uint4 v; uint32_t more; };
  struct b { uint2 v; uint32_t more; };
  static PG_DEVICE uint4 pack(const a &x, uint32_t shift) {
    return make_uint4(__builtin_amdgcn_alignbyte(x.v.y, x.v.x, shift), __builtin_amdgcn_alignbyte(x.v.z, x.v.y, shift),
                      __builtin_amdgcn_alignbyte(x.v.w, x.v.z, shift), __builtin_amdgcn_alignbyte(x.more, x.v.w, shift));
  }
  static PG_DEVICE uint2 pack(const b &x, uint32_t shift) {
    return make_uint2(__builtin_amdgcn_alignbyte(x.v.y, x.v.x, shift), __builtin_amdgcn_alignbyte(x.more, x.v.y, shift));
  }
};

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

// Where row r of a shared tile of W columns keeps its 32-byte pieces: byte offset ^ this. A transposed
// read takes one piece of each of rows 0..3 and 8..11 (or 4 on, or 16 on) at once: they fall into
// different eighths of the 64 banks, without padding.
template <int W> PG_DEVICE int wg_swz(int r) {
  if constexpr (W == 64) return ((r >> 1 & 1) | (r >> 3 & 1) << 1) * 32;
  else return ((r & 3) | (r >> 3 & 1) << 2) * 32;
}

// ALN: rows of dY and of the codes begin at multiples of 8 values
template <class T, int W, bool ALN>
__global__ __launch_bounds__(256) void mx8_wgrad_kernel(const WgradArgs a) {
  constexpr int TH = 256;                                       // threads
  constexpr int Q = W / 2, R = Q / 16;                          // a wave's part, 16 x 16 blocks of it
  constexpr int P = W * 2;                                      // row pitch in bytes
  constexpr int CH = W / 8, RS = TH / CH;                       // 8-value chunks of a row, rows at a time
  constexpr int NC = kMK / RS;                                     // chunks a thread
  constexpr int D = kAhead;                           // steps on their way in registers
  __shared__ __attribute__((aligned(16))) char smem[2][kMK * 2 * P];
  const int t = threadIdx.x, lane = t & 63, wave = t >> 6;
  // neighbouring tiles of one row split on one XCD, whose L2 holds the rows they share
  const int total = a.tn * a.tk * a.splits, per = total / 8;
  int id = blockIdx.x;
  if (id < per * 8) id = (id & 7) * per + (id >> 3);
  const int split = id / (a.tn * a.tk), tile = id % (a.tn * a.tk);
  const int n0 = (tile / a.tk) * W, k0 = (tile % a.tk) * W;
  const int mb = split * a.rows, rows = min(a.M - mb, a.rows);
  // The split's rows through buffer descriptors: rows past its end, and columns past N or K (offset
  // kOOB), read as zeros, without a branch or a select that would wait for the load.
  // (Unaligned rows are read in whole words: the last one may reach past the end, but not into another
  // page, and a chunk's columns past N or K are another row's values, which reach only results that are
  // not written. Rows past the split's end are masked there.)
  auto bytes = [](uint32_t n) { return ALN ? n : (n + 3) & ~3u; };
  const rsrc_t ry = make_rsrc(static_cast<const T *>(a.dy) + (long long)mb * a.N, bytes((uint32_t)rows * a.N * 2u));
  const rsrc_t rq = make_rsrc(a.q + (long long)mb * a.K, bytes((uint32_t)rows * a.K));
  const rsrc_t rs = make_rsrc(a.qs + (long long)mb * a.nb, (uint32_t)rows * a.nb);

  struct Stage {
    typename WgRaw<ALN>::a a[NC];
    typename WgRaw<ALN>::b b[NC];
    uint8_t e[NC];
  };
  // Chunk i of this thread: row t / CH + i * RS of the step, column t % CH * 8 (codes alike). Its
  // offsets for the next load; from kOOB on they stay outside, a split spans less than 2^31 bytes.
  const int na = n0 + t % CH * 8, kb = k0 + t % CH * 8;
  uint32_t row = t / CH, oa = na < a.N ? (row * a.N + na) * 2u : kOOB, ob = kb < a.K ? row * a.K + kb : kOOB;
  uint32_t oe = kb < a.K ? row * a.nb + kb / kMxBlock : kOOB;
  const uint32_t sa = oa & 3u, sb = ob & 3u;   // of every chunk of this thread: RS and kMK are multiples of 4
  oa -= sa;
  ob -= sb;
  auto load = [&](Stage &g) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const uint32_t m = i * RS, da = oa + m * a.N * 2u, db = ob + m * a.K;
      if constexpr (ALN) {
        g.a[i] = bld16(ry, da);
        g.b[i] = bld8(rq, db);
      } else {
        const bool in = row + m < (uint32_t)rows;
        const uint32_t ia = in ? da : kOOB, ib = in ? db : kOOB;
        g.a[i].v = bld16(ry, ia);
        g.a[i].more = __builtin_amdgcn_raw_buffer_load_b32(ry, (int)(ia + 16), 0, 0);
        g.b[i].v = bld8(rq, ib);
        g.b[i].more = __builtin_amdgcn_raw_buffer_load_b32(rq, (int)(ib + 8), 0, 0);
      }
      g.e[i] = __builtin_amdgcn_raw_buffer_load_b8(rs, (int)(oe + m * a.nb), 0, 0);
    }
    oa += kMK * 2u * a.N;
    ob += (uint32_t)kMK * a.K;
    oe += (uint32_t)kMK * a.nb;
    row += kMK;
  };
  float sum[8] = {};   // db: this thread's columns (a thread's chunks of dY are one column's, TH % CH == 0)
  const bool bias = a.db && k0 == 0;
  auto put = [&](const Stage &g, int buf) {
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = t / CH + i * RS;
      *reinterpret_cast<uint4 *>(smem[buf] + r * P + (t % CH * 16 ^ wg_swz<W>(r))) = WgRaw<ALN>::pack(g.a[i], sa);
    }
#pragma unroll
    for (int i = 0; i < NC; ++i) {
      const int r = t / CH + i * RS;
      *reinterpret_cast<uint4 *>(smem[buf] + kMK * P + r * P + (t % CH * 16 ^ wg_swz<W>(r))) =
          wg_decode<T>(WgRaw<ALN>::pack(g.b[i], sb), g.e[i]);
    }
    if (bias)
#pragma unroll
      for (int i = 0; i < NC; ++i) {
        float v[8];
        Vec<T, 8>::unpack(WgRaw<ALN>::pack(g.a[i], sa), v);
#pragma unroll
        for (int j = 0; j < 8; ++j) sum[j] += v[j];
      }
  };

  f32x4_t acc[R][R];
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j) acc[i][j] = f32x4_t{0.f, 0.f, 0.f, 0.f};
  const int wn = wave / 2 * Q, wk = wave % 2 * Q;
  // transposed reads: lane (g = lane / 16, i = lane % 16) asks for row 8 g + i / 4 (then + 4), 8-byte
  // piece i % 4 of a 16-column block, and receives those rows of column i
  const int trow = 8 * (lane >> 4) + ((lane & 15) >> 2), tc = (lane & 3) * 8;
  auto mma = [&](int buf) {
    const char *A = smem[buf], *B = smem[buf] + kMK * P;
#pragma unroll
    for (int sub = 0; sub < kMK / 32; ++sub) {
      s16x8_t fa[R], fb[R];
#pragma unroll
      for (int i = 0; i < R; ++i) {
        const char *p = A + (sub * 32 + trow) * P + ((wn + i * 16) * 2 ^ wg_swz<W>(trow)) + tc;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * P));
        fa[i] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int j = 0; j < R; ++j) {
        const char *p = B + (sub * 32 + trow) * P + ((wk + j * 16) * 2 ^ wg_swz<W>(trow)) + tc;
        const s16x4_t lo = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)p);
        const s16x4_t hi = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lds_s16x4_t *)(p + 4 * P));
        fb[j] = __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
      }
#pragma unroll
      for (int i = 0; i < R; ++i)
#pragma unroll
        for (int j = 0; j < R; ++j) acc[i][j] = wg_mfma<T>(fa[i], fb[j], acc[i][j]);
    }
  };

  // Steps x + 1 to x + D are in registers or on their way while step x is multiplied; a turn is D
  // steps (rows past the end are zeros).
  Stage g[D];
#pragma unroll
  for (int j = 0; j < D; ++j) load(g[j]);
  put(g[0], 0);
  __syncthreads();
  const int turns = (rows + kMK * D - 1) / (kMK * D);
#pragma unroll 1
  for (int s = 0; s < turns; ++s) {
#pragma unroll
    for (int j = 0; j < D; ++j) {
      load(g[j]);
      mma(j & 1);
      put(g[(j + 1) % D], (j + 1) & 1);
      __syncthreads();
    }
  }
  float *out = a.out + (a.splits > 1 ? split * a.pitch : 0);
#pragma unroll
  for (int i = 0; i < R; ++i)
#pragma unroll
    for (int j = 0; j < R; ++j)
#pragma unroll
      for (int r = 0; r < 4; ++r) {
        const int n = n0 + wn + i * 16 + 4 * (lane >> 4) + r, k = k0 + wk + j * 16 + (lane & 15);
        if (n < a.N && k < a.K) out[(long long)n * a.K + k] = acc[i][j][r];
      }
  if (!bias) return;
  // the RS threads of a column chunk, in order
  float *sh = reinterpret_cast<float *>(smem[0]);
#pragma unroll
  for (int j = 0; j < 8; ++j) sh[t * 8 + j] = sum[j];
  __syncthreads();
  float *db = a.splits > 1 ? out + (long long)a.N * a.K : a.db;
  if (t < W && n0 + t < a.N) {
    float s = 0.f;
    for (int r = 0; r < RS; ++r) s += sh[(r * CH + t / 8) * 8 + t % 8];
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
  int W, tn, tk, splits, rows;
  long long pitch;
};

// Tiles of 64 x 64 until there is work for larger ones: four workgroups of them fit a CU, and the odd
// widths of narrow layers pad less.  Measured, 128 and 64 (us): 25088 x 1024 x 1024 81 and 113, 6272 x
// 2048 x 1024 51 and 56, 100352 x 512 x 256 51 and 60; 25088 x 512 x 512 32 and 34, 100352 x 256 x 256
// 35 and 35; 1568 x 2048 x 1000 30 and 18, 401408 x 144 x 24 49 and 31, 100352 x 192 x 192 33 and 27.
// 128 x 128 take as long as 64 x 64 where they pad to a third more.
WgradPlan wgrad_plan(int M, int N, int K) {
  WgradPlan p{};
  auto up = [](long long n, int w) { return (n + w - 1) / w; };
  const bool large = (double)M * N * K >= 8e9 && up(N, 128) * up(K, 128) * 4 * 3 <= up(N, 64) * up(K, 64) * 4;
  p.W = large ? 128 : 64;
  const long long t = up(N, p.W) * up(K, p.W);
  p.tn = (int)up(N, p.W);
  p.tk = (int)up(K, p.W);
  const long long steps = ((long long)M + kMK - 1) / kMK;
  // 512 workgroups (256: up to a fifth slower, 768 and 1024: no faster)
  long long s = std::max<long long>(1, std::min<long long>(512 / t, steps / 4));
  // whole turns; a split's rows, and as many steps on as are loaded, span less than 2^31 bytes
  long long turns = (steps + s * kAhead - 1) / (s * kAhead);
  turns = std::min<long long>(turns, 0x7fffffffll / (2ll * std::max(N, K) * kMK * kAhead) - 1);
  if (turns < 1) throw std::invalid_argument("mx8_wgrad: N or K is too large");
  p.rows = (int)(turns * kAhead * kMK);
  p.splits = (int)(((long long)M + p.rows - 1) / p.rows);
  p.pitch = ((long long)N * K + N + 3) / 4 * 4;
  // the product's grid, and the join's: a work-item for every sum, in whole workgroups of 1024
  if (t * p.splits > kMostWgs || (p.splits > 1 && p.pitch > kMostItems - 1023))
    throw std::invalid_argument("mx8_wgrad: N * K is too large");
  return p;
}

template <class T, bool ALN> void wgrad_go(const WgradPlan &p, const WgradArgs &a, hipStream_t st) {
  const dim3 grid((unsigned)(p.tn * p.tk * p.splits));
  if (p.W == 128) hipLaunchKernelGGL((mx8_wgrad_kernel<T, 128, ALN>), grid, dim3(256), 0, st, a);
  else hipLaunchKernelGGL((mx8_wgrad_kernel<T, 64, ALN>), grid, dim3(256), 0, st, a);
}

long long slot_wgs(long long M, long long slots) { return (M * slots + kU * kThreads - 1) / (kU * kThreads); }
// rows a launch: a multiple of 16, so that the next one's begin as aligned as the first's
long long slot_rows(long long slots) { return kMostWgs * (kU * kThreads) / slots / 16 * 16; }
// Values a thread (16 bytes of them, or 8 where rows are a multiple of that only), and whether rows begin
// anywhere. 400000 rows of 140, 142, 143 and 144 bf16: pack 37, 52, 55, 34 us (one and two values a thread
// took 65 for 142 and 126 for 143), unpack 32 each (45 and 78); of 142 fp32 in twos 61 and 55 (as if at
// any alignment: 69 and 71). Matrices narrower than 16 bytes go value by value.
struct Lanes {
  int V;
  bool any;
  Lanes(int C, int full) : V(C % full == full / 2 ? full / 2 : C % full == 0 || C >= full ? full : 1),
                           any(V == full && C % full != 0) {}
};
template <int FULL, class F> void with_lanes(const Lanes &l, F f) {
  typedef std::integral_constant<int, FULL> Full;
  if (l.V == 1) f(std::integral_constant<int, 1>(), std::false_type());
  else if (l.V == FULL / 2) f(std::integral_constant<int, FULL / 2>(), std::false_type());
  else if (l.any) f(Full(), std::true_type());
  else f(Full(), std::false_type());
}
}  // namespace

template <class T> static void pack_go(const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st) {
  const int nb = (C + kMxBlock - 1) / kMxBlock, full = 16 / (int)sizeof(T);
  const Lanes l(C, full);
  const FastDiv f((uint32_t)nb * (kMxBlock / l.V));
  for (long long r = 0, most = slot_rows(f.d); r < M; r += most) {
    const long long rows = std::min(most, M - r);
    const dim3 grid((unsigned)slot_wgs(rows, f.d));
    with_lanes<16 / sizeof(T)>(l, [&](auto v, auto any) {
      hipLaunchKernelGGL((mx8_pack_kernel<T, decltype(v)::value, decltype(any)::value>), grid, dim3(kThreads), 0, st,
                         (const T *)x + r * C, q + r * C, qs + r * nb, rows, C, nb, f);
    });
  }
}
template <class T> static void unpack_go(const uint8_t *q, const uint8_t *qs, void *x, long long M, int C, hipStream_t st) {
  const int nb = (C + kMxBlock - 1) / kMxBlock;
  const Lanes l(C, 16 / (int)sizeof(T));
  const FastDiv f((uint32_t)(l.any ? C : C / l.V));
  for (long long r = 0, most = slot_rows(f.d); r < M; r += most) {
    const long long rows = std::min(most, M - r);
    const dim3 grid((unsigned)(l.any ? slot_wgs(1, rows * C / l.V + 1) : slot_wgs(rows, f.d)));
    with_lanes<16 / sizeof(T)>(l, [&](auto v, auto any) {
      constexpr int V = decltype(v)::value;
      auto go = [&](auto kernel) {
        hipLaunchKernelGGL(kernel, grid, dim3(kThreads), 0, st, q + r * C, qs + r * nb, (T *)x + r * C, rows, C, nb, f);
      };
      if constexpr (decltype(any)::value) go(mx8_unpack_run_kernel<T, V>);
      else go(mx8_unpack_kernel<T, V>);
    });
  }
}

// dt: 0 bf16, 1 fp16, 2 fp32
void launch_mx8_pack(int dt, const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st) {
  if (M <= 0) return;
  (dt == 0 ? pack_go<bf16_t> : dt == 1 ? pack_go<_Float16> : pack_go<float>)(x, q, qs, M, C, st);
}
void launch_mx8_unpack(int dt, const uint8_t *q, const uint8_t *qs, void *x, long long M, int C, hipStream_t st) {
  if (M <= 0) return;
  (dt == 0 ? unpack_go<bf16_t> : dt == 1 ? unpack_go<_Float16> : unpack_go<float>)(q, qs, x, M, C, st);
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
