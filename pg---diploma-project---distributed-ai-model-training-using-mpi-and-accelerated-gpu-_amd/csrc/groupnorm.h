// Group norm with an activation over channels-last [B][S][C] tensors, forward and backward, with
// the 8-bit checkpoint of the input (mx8.h) written by the forward and read by the backward.
//
//   y = act(z), z = (x - mean) rstd gamma + beta, statistics over the S * C/G values of (b, g)
//   dz = dy act'(z), xh = (x - mean) rstd:  dgamma = sum dz xh, dbeta = sum dz,
//   dx = rstd (dz gamma - (s1 + xh s2) / m), s1 = sum_g dz gamma, s2 = sum_g dz gamma xh
//
// Both are bound by memory.  What reads a tile twice is kept close to where it was read first:
//   solo     a workgroup holds all S rows of a slab of whole groups in registers: one read
//   held     the S rows are k tiles, and all tiles of the tensor are so few that their workgroups run
//            together: each keeps its tile in registers, publishes its sums, waits for the k - 1
//            others of its image and goes on.  One read.  (96 x 784 x 192 from a checkpoint, backward: 26
//            us a call, 33 staged.  With more tiles than fit, a workgroup's chain load - sum - publish -
//            wait - join - store is not hidden behind others': 128 x 12544 x 96 backward 1129 us.)
//   staged   longer maps: the S rows are k tiles.  One launch holds a sums and a use workgroup for
//            every tile; the use of an image's tiles is queued `lead` tiles behind its sums, so
//            that it hardly ever waits for them and finds the tile in the memory-side cache
//            (256 MB).  HBM sees every value once: 128 x 12544 x 96 backward reads 607 MB and
//            writes 308 in 230 us, 4.0 TB/s; 128 x 3136 x 144 forward with checkpoint 289 MB in 75 us,
//            3.8 TB/s.  What is left of a copy's 5.1 TB/s goes to a workgroup's latencies and, as the
//            checkpointed forward's counters have it, to the issue of its vector instructions (more
//            than half of their units' time).  Not so for wide rows on long maps: a use workgroup reads all k pairs of
//            each of its groups, and a tile has few rows there (8 x 9765 x 1280 in 160 groups, backward:
//            k = 814, 1 MB of pairs for a tile of 61 KB; 2.0 ms, 117 us of it for the tensors' bytes).
//   wide     what no workgroup holds: a slab (whole groups, vectors and, where one is written, checkpoint
//            blocks) of more vectors than threads, or whose sums pass 64 KB of shared memory (backward, bf16
//            and fp16: some 1900 to 2048 channels and other slabs of that width; 625 channels in 25 groups
//            with a checkpoint).  Plain kernels (groupnorm.hip): a workgroup at a time per (image, group),
//            then one value a thread.  32 x 784 x 2048 in 32 groups, backward: 705 us; 1880 channels, staged,
//            398.
// A thread owns one vector of V channels (16 bytes where C allows) and every R-th row of the tile.
// Sums are taken in a fixed order, so results do not vary from run to run, unless a wait for other workgroups'
// sums is given up: those sums are then taken from the tensor, in another order (right, but other last bits).
#pragma once
#include "mx8.h"
#include "vec.h"

#include <cmath>
#include <type_traits>

namespace gn {
enum GnAct : int { GN_NONE = 0, GN_RELU = 1, GN_RELU6 = 2, GN_SILU = 3 };
enum GnMode : int { SOLO = 0, HELD = 1, STAGED = 2, WIDE = 3 };

// ---- tile geometry ---------------------------------------------------------------------------
struct Geo {
  long long B, S;
  int C, G, cg;
  int cs;       // channels of a slab (whole groups; the last slab may be narrower)
  int nslab;
  int CVp;      // vector columns of a tile row (padded to whole 32-channel blocks for checkpoints)
  int R;        // tile rows per sweep: blockDim / CVp
  int k;        // tiles per unit, a unit being one (image, slab)
  int gs;       // groups of a full slab
  int tiles;    // of all units
  int lead;     // tiles that sums workgroups are ahead of use workgroups: a multiple of k
  int rows;     // held: rows of a tile
  int turn;     // staged: rows of a round; round i of tile c begins at row (i k + c) turn
  int wait;     // polls after which a use workgroup takes its sums from the tensor itself
};

// this workgroup's place
struct Place {
  long long b, unit;   // image; image * nslab + slab
  int chunk, c0, csl, ng, g0;
  int col, row, c;
  bool on;             // this thread has a column
  bool use;            // staged: applies the sums (else: makes them)
};
// Staged order: `lead` sums tiles, then the remaining sums tiles alternating, 8 and 8 (one round of
// the 8 XCDs each), with the use tiles `lead` behind them, then the last `lead` use tiles.  A use
// workgroup waits only for sums workgroups of lower index, which each XCD starts first, and those
// wait for nobody.  (Handing the places out by an atomic counter makes that order certain, but one
// address takes 32 ns an increment: 128 x 12544 x 96 backward 630 us.  Should the order ever be
// another, the wait is bounded and the work is done without the peers.)
template <int V, int MODE> PG_DEVICE Place place(const Geo &g) {
  Place p;
  uint32_t id = blockIdx.x;   // the grid is below 2^31
  p.use = false;
  if constexpr (MODE == STAGED) {
    const uint32_t lead = g.lead, both = g.tiles - lead, even = both & ~7u;
    if (id >= lead) {
      id -= lead;
      if (id < 2 * even) {
        p.use = (id >> 3) & 1;
        id = (id >> 4) * 8 + (id & 7);
      } else if (id < 2 * both) {
        const uint32_t r = id - 2 * even, rest = both - even;
        p.use = r >= rest;
        id = even + (p.use ? r - rest : r);
      } else {
        p.use = true;
        id -= both;
      }
      if (!p.use) id += lead;
    }
  }
  const uint32_t unit = id / (uint32_t)g.k;
  p.chunk = id - unit * g.k;
  p.unit = unit;
  p.b = unit / (uint32_t)g.nslab;
  const int slab = unit - (uint32_t)p.b * g.nslab;
  p.c0 = slab * g.cs;
  p.csl = min(g.cs, g.C - p.c0);
  p.ng = p.csl / g.cg;
  p.g0 = p.c0 / g.cg;
  p.col = threadIdx.x % g.CVp;
  p.row = threadIdx.x / g.CVp;
  p.on = p.col < p.csl / V && p.row < g.R;
  p.c = p.on ? p.c0 + p.col * V : p.c0;
  return p;
}

// element at a byte offset from a base that is the same for the whole workgroup (a tile spans less
// than 2^31 bytes): one scalar base and one 32-bit offset register a load
template <class R> PG_DEVICE const R &at(const void *base, uint32_t off) {
  return *reinterpret_cast<const R *>(static_cast<const char *>(base) + off);
}
template <class R> PG_DEVICE R &at(void *base, uint32_t off) {
  return *reinterpret_cast<R *>(static_cast<char *>(base) + off);
}

// V values of an optional per-channel vector.  The loads are unconditional (`any` is readable memory
// of one float): behind a branch each would be waited for by itself, 0.6 us apiece.
template <int V> PG_DEVICE void channel_values(const float *v, const float *any, int c, float none, float (&out)[V]) {
  const float *src = v ? v : any;
  const uint32_t first = v ? c * 4u : 0u, step = v ? 4u : 0u;
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = at<float>(src, first + j * step);
#pragma unroll
  for (int j = 0; j < V; ++j) out[j] = v ? out[j] : none;
}

PG_DEVICE float seg_sum(float v, int W) {   // sum over aligned segments of W lanes
  for (int o = W >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o, 64);
  return v;
}
PG_DEVICE int seg_width(int n) {   // lanes that share n terms: a power of two up to 64
  int W = 64;
  while (W > 1 && (W >> 1) >= n) W >>= 1;
  return W;
}

// sums of n columns over the rows r0, r0 + step, .. < R of a [R][ld] array, four at a time
PG_DEVICE float col_sum(const float *p, int r0, int R, int step, int ld) {
  float s[4] = {0.f, 0.f, 0.f, 0.f};
  int r = r0;
  for (; r + 3 * step < R; r += 4 * step) {
#pragma unroll
    for (int u = 0; u < 4; ++u) s[u] += p[(r + u * step) * ld];
  }
  for (; r < R; r += step) s[0] += p[r * ld];
  return (s[0] + s[1]) + (s[2] + s[3]);
}

// out[g] = sum over the tile of the values of group g; acc: this thread's column sums.
// FOLD: C/G is a multiple of V, so the thread's channels are one group's and count as one column.
// Rows first (as many stripes of them as there are threads), then the stripes, then the columns.
// red: blockDim * V floats and blockDim + slab channels more.
template <int V, bool FOLD>
PG_DEVICE void group_sums(const Geo &g, const Place &p, const float (&acc)[V], float *red, float *out) {
  const int t = threadIdx.x, TH = blockDim.x;
  const int ld = FOLD ? g.CVp : g.CVp * V, width = FOLD ? g.cg / V : g.cg, n = p.ng * width, nt = TH / n;
  float *red2 = red + TH * V, *tot = red2 + TH;
  if (p.on) {
    if constexpr (FOLD) {
      float s = 0.f;
#pragma unroll
      for (int j = 0; j < V; ++j) s += acc[j];
      red[p.row * ld + p.col] = s;
    } else {
#pragma unroll
      for (int j = 0; j < V; ++j) red[p.row * ld + p.col * V + j] = acc[j];
    }
  }
  __syncthreads();
  if (nt <= 1) {
    for (int o = t; o < n; o += TH) tot[o] = col_sum(red + o, 0, g.R, 1, ld);
  } else {
    const int st = t / n, o = t - st * n;
    if (st < nt) red2[st * n + o] = col_sum(red + o, st, g.R, nt, ld);
    __syncthreads();
    if (t < n) tot[t] = col_sum(red2 + t, 0, nt, 1, n);
  }
  __syncthreads();
  const int W = seg_width(width), per = 64 / W, lane = t & 63, l = lane & (W - 1);
  for (int i = (t >> 6) * per + lane / W; i - lane / W < p.ng; i += (TH >> 6) * per) {
    float s = 0.f;
    if (i < p.ng)
      for (int c = l; c < width; c += W) s += tot[i * width + c];
    s = seg_sum(s, W);
    if (l == 0 && i < p.ng) out[i] = s;
  }
  __syncthreads();
}

// Hand-over of a unit's sums: a tile's two sums of a group are one 64-bit word, written and read in
// one piece at agent scope.  kNone, which no computed pair holds, says that they have not come.
constexpr unsigned long long kNone = ~0ull;
PG_DEVICE void pair_store(unsigned long long *p, float a, float b) {
  const unsigned ua = __float_as_uint(a), ub = __float_as_uint(b);   // a NaN of all ones: any other
  __hip_atomic_store(p, (unsigned long long)(ua == ~0u ? 0x7fc00000u : ua) | ((unsigned long long)ub << 32),
                     __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
PG_DEVICE unsigned long long pair_load(const unsigned long long *p) {
  return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
// The lane's pairs (tiles l, l + W, ..) of a group, in order; false: one of the wave's did not come.
// v: the first four, asked for by pairs_ahead when the workgroup began.
PG_DEVICE void pairs_ahead(const unsigned long long *src, int k, int l, int W, int c0, unsigned long long (&v)[4]) {
#pragma unroll
  for (int u = 0; u < 4; ++u) {
    const int ch = c0 + u * W + l;
    v[u] = pair_load(src + (ch < k ? ch : l < k ? l : 0));
  }
}
template <class F>
PG_DEVICE bool pairs(const unsigned long long *src, int k, int l, int W, int polls, unsigned long long (&v)[4], F f) {
  if (polls < 0) return false;
  for (int c0 = 0; c0 < k; c0 += 4 * W) {   // four loads in flight
    if (c0) pairs_ahead(src, k, l, W, c0, v);
    for (int i = 0;; ++i) {
      const bool none = v[0] == kNone || v[1] == kNone || v[2] == kNone || v[3] == kNone;
      const unsigned long long who = __ballot(none);
      if (!who) break;
      // One lane looks for its first missing pair until it comes, then all look again: with every lane
      // looking, the waiting waves' reads held up those that were waited for (7 x 3249 x 100
      // forward 18.8 us, not 17.7).
      if ((int)(threadIdx.x & 63) == __ffsll((long long)who) - 1) {
        const int u = v[0] == kNone ? 0 : v[1] == kNone ? 1 : v[2] == kNone ? 2 : 3, ch = c0 + u * W + l;
        for (; i < polls && pair_load(src + (ch < k ? ch : l < k ? l : 0)) == kNone; ++i) __builtin_amdgcn_s_sleep(16);
      }
      i = __builtin_amdgcn_readlane(i, __ffsll((long long)who) - 1);
      if (i >= polls) return false;
      pairs_ahead(src, k, l, W, c0, v);
    }
#pragma unroll
    for (int u = 0; u < 4; ++u) {
      const int ch = c0 + u * W + l;
      if (ch < k) f(ch, __uint_as_float((unsigned)v[u]), __uint_as_float((unsigned)(v[u] >> 32)));
    }
  }
  return true;
}

// count, mean and sum of squares about it; joined without ever forming E[x^2]
struct Moments {
  float n, m, v;
  PG_DEVICE void join(float n2, float m2, float v2) {
    const float t = n + n2, d = m2 - m, w = t > 0.f ? n2 / t : 0.f;
    m = fmaf(d, w, m);
    v += fmaf(d * d, n * w, v2);
    n = t;
  }
};

// ---- forward ---------------------------------------------------------------------------------
struct FwdArgs {
  Geo g;
  const void *x;
  const float *gamma, *beta;
  void *y;
  float *mean, *rstd;
  uint8_t *q, *qs;
  unsigned long long *part;   // [B * nslab][gs][k]: mean and sum of squares about it of every tile and group
  float eps;
  int act;
};

// NaN passes through every activation
template <int ACT> PG_DEVICE float gn_act(float z) {
  if constexpr (ACT == GN_RELU) return z < 0.f ? 0.f : z;
  else if constexpr (ACT == GN_RELU6) return z < 0.f ? 0.f : z > 6.f ? 6.f : z;
  else if constexpr (ACT == GN_SILU) return z / (1.f + __expf(-z));
  else return z;
}

// a store through a buffer descriptor: offset kOOB drops it, without a branch around it
PG_DEVICE void buf_store(rsrc_t r, uint32_t o, const uint4 &v) { bst16(r, o, v); }
PG_DEVICE void buf_store(rsrc_t r, uint32_t o, const uint2 &v) { bst8(r, o, v); }
PG_DEVICE void buf_store(rsrc_t r, uint32_t o, uint32_t v) { __builtin_amdgcn_raw_buffer_store_b32(v, r, (int)o, 0, 0); }
PG_DEVICE void buf_store(rsrc_t r, uint32_t o, uint16_t v) { __builtin_amdgcn_raw_buffer_store_b16(v, r, (int)o, 0, 0); }
PG_DEVICE void buf_store(rsrc_t r, uint32_t o, uint8_t v) { __builtin_amdgcn_raw_buffer_store_b8(v, r, (int)o, 0, 0); }

// Where a tile's or round's checkpoint goes: rows r0 .. r0 + rows, through buffer descriptors, which drop
// the masked lanes' stores without a branch.
struct CkRows {
  rsrc_t q, qs;
  PG_DEVICE CkRows(const FwdArgs &a, long long r0, int rows) {
    const int C = a.g.C, nb = (C + kMxBlock - 1) / kMxBlock;
    q = make_rsrc(a.q + r0 * C, (uint32_t)rows * C);
    qs = make_rsrc(a.qs + r0 * nb, (uint32_t)rows * nb);
  }
};
// the checkpoint of row r's V channels; 32 channels are 32 / V neighbouring lanes (CVp is a multiple of
// that), all of which come here
template <class T, int V>
PG_DEVICE void gn_checkpoint(const FwdArgs &a, const Place &p, const typename Vec<T, V>::raw &raw, const CkRows &k, int r, bool ok) {
  float f[V];
  Vec<T, V>::unpack(raw, f);
  const int e = mx8_exp(block_amax<T, V>(raw, p.on));
  const typename Codes<V>::raw c = Codes<V>::encode(f, mx8_inv_scale(e));
  const uint32_t o = ok ? (uint32_t)r * a.g.C + p.c : kOOB;
  const uint32_t os = ok && p.c % kMxBlock == 0 ? (uint32_t)r * ((a.g.C + kMxBlock - 1) / kMxBlock) + p.c / kMxBlock : kOOB;
  buf_store(k.q, o, c);
  buf_store(k.qs, os, (uint8_t)e);
}

// y of one row's V channels
template <class T, int V, int VG, int ACT>
PG_DEVICE typename Vec<T, V>::raw gn_y(const typename Vec<T, V>::raw &raw, const float (&mu)[VG], const float (&sc)[V],
                                       const float (&be)[V]) {
  float f[V];
  Vec<T, V>::unpack(raw, f);
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = gn_act<ACT>(fmaf(f[j] - mu[VG == 1 ? 0 : j], sc[j], be[j]));
  return Vec<T, V>::pack(f);
}
// the activation as a compile-time constant
template <class F> PG_DEVICE void with_act(int act, F f) {
  if (act == GN_RELU6) f(std::integral_constant<int, GN_RELU6>());
  else if (act == GN_RELU) f(std::integral_constant<int, GN_RELU>());
  else if (act == GN_SILU) f(std::integral_constant<int, GN_SILU>());
  else f(std::integral_constant<int, GN_NONE>());
}

// the statistics of the slab's groups (gm: mean, gr: rstd) as this thread's channels take them
// (sc: gamma before, gamma rstd after)
template <int V, int VG>
PG_DEVICE void fwd_constants(const int (&gi)[VG], const float *gm, const float *gr, float (&mu)[VG], float (&sc)[V]) {
#pragma unroll
  for (int j = 0; j < VG; ++j) mu[j] = gm[gi[j]];
#pragma unroll
  for (int j = 0; j < V; ++j) sc[j] *= gr[gi[VG == 1 ? 0 : j]];
}
PG_DEVICE void fwd_statistics(const FwdArgs &a, const Place &p, const float *gm, const float *gr) {
  if (p.chunk == 0)
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) {
      a.mean[p.b * a.g.G + p.g0 + i] = gm[i];
      a.rstd[p.b * a.g.G + p.g0 + i] = gr[i];
    }
}

// where the tiles are joined: W lanes a group, 4 pairs a lane
struct JoinLanes {
  const unsigned long long *in;
  int W, per, lane, l, i0;
  PG_DEVICE JoinLanes(const Geo &g, const Place &p, const unsigned long long *part)
      : in(part + p.unit * g.k * g.gs), W(seg_width((g.k + 3) / 4)), per(64 / W), lane(threadIdx.x & 63),
        l(lane & (W - 1)), i0((threadIdx.x >> 6) * per + lane / W) {}
  // the first group's pairs on their way
  PG_DEVICE void ahead(const Geo &g, const Place &p, unsigned long long (&v)[4]) const {
    pairs_ahead(in + (long long)min(i0, p.ng - 1) * g.k, g.k, l, W, 0, v);
  }
};

// rows of tile ch: staged tiles take turns of `turn` rows, held ones are in one piece
template <int MODE> PG_DEVICE float tile_rows(const Geo &g, int ch) {
  if constexpr (MODE == HELD) return (float)min((long long)g.rows, g.S - (long long)ch * g.rows);
  const long long all = (long long)g.turn * g.k, full = g.S / all, rest = g.S - full * all - (long long)ch * g.turn;
  return (float)(full * g.turn + (rest < 0 ? 0 : rest < g.turn ? rest : g.turn));
}

// gm, gr = mean, rstd of the unit's groups
template <class T, int MODE>
PG_DEVICE void fwd_join(const FwdArgs &a, const Place &p, const JoinLanes &q, unsigned long long (&pv)[4], float *gm, float *gr) {
  const Geo &g = a.g;
  for (int i = q.i0; i - q.lane / q.W < p.ng; i += (blockDim.x >> 6) * q.per) {
    Moments t{0.f, 0.f, 0.f};
    const int gc = min(i, p.ng - 1);
    const unsigned long long *in = q.in + (long long)gc * g.k;
    if (i != q.i0) pairs_ahead(in, g.k, q.l, q.W, 0, pv);
    if (!pairs(in, g.k, q.l, q.W, g.wait, pv, [&](int ch, float m, float v) {
          t.join(tile_rows<MODE>(g, ch) * (float)g.cg, m, v);
        })) {
      // without the peers: every W-th row of the group, from the tensor
      const T *base = static_cast<const T *>(a.x) + p.b * g.S * g.C + p.c0 + gc * g.cg;
      t = Moments{0.f, 0.f, 0.f};
#pragma unroll 1
      for (long long r = q.l; r < g.S; r += q.W)
#pragma unroll 1
        for (int c = 0; c < g.cg; ++c) t.join(1.f, tof(base[r * g.C + c]), 0.f);
    }
    for (int o = 1; o < q.W; o <<= 1) t.join(__shfl_xor(t.n, o, 64), __shfl_xor(t.m, o, 64), __shfl_xor(t.v, o, 64));
    if (q.l == 0 && i < p.ng) {
      gm[i] = t.m;
      gr[i] = 1.f / sqrtf(t.v / t.n + a.eps);
    }
  }
  __syncthreads();
}

// solo, held: the rows stay in NV registers a thread between the mean, the squares about it and y
template <class T, int V, int NV, int MODE, bool CK, bool FOLD>
__global__ __launch_bounds__(1024) void gn_fwd_solo_kernel(const FwdArgs a) {
  extern __shared__ float sm[];
  typedef Vec<T, V> X;
  const Geo &g = a.g;
  const Place p = place<V, MODE>(g);
  float *gm = sm, *gr = sm + g.gs, *red = sm + 2 * g.gs;
  constexpr int VG = FOLD ? 1 : V;
  int gi[VG];   // slab group of each channel (FOLD: of all)
#pragma unroll
  for (int j = 0; j < VG; ++j) gi[j] = (p.c - p.c0 + j) / g.cg;
  const long long s0 = MODE == HELD ? (long long)p.chunk * g.rows : 0, r0 = p.b * g.S + s0;
  const int nr = (int)(MODE == HELD ? min((long long)g.rows, g.S - s0) : g.S);
  const T *src = static_cast<const T *>(a.x) + r0 * g.C;
  T *dst = static_cast<T *>(a.y) + r0 * g.C;
  // rows past the end (and threads without a column) read a row that exists and are masked
  typename X::raw d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t r = min(p.row + i * g.R, nr - 1);
    d[i] = at<typename X::raw>(src, (r * g.C + p.c) * (uint32_t)sizeof(T));
  }
  float acc[V], mu[VG], sc[V], be[V];
  auto affine = [&] {
    channel_values(a.gamma, a.mean, p.c, 1.f, sc);
    channel_values(a.beta, a.mean, p.c, 0.f, be);
  };
  if constexpr (MODE == SOLO) affine();
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (p.row + i * g.R < nr) {
      float f[V];
      X::unpack(d[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) acc[j] += f[j];
    }
  group_sums<V, FOLD>(g, p, acc, red, gm);
  const float n = (float)nr * (float)g.cg;
#pragma unroll
  for (int j = 0; j < VG; ++j) mu[j] = gm[gi[j]] / n;
#pragma unroll
  for (int j = 0; j < V; ++j) acc[j] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (p.row + i * g.R < nr) {
      float f[V];
      X::unpack(d[i], f);
#pragma unroll
      for (int j = 0; j < V; ++j) {
        const float df = f[j] - mu[FOLD ? 0 : j];
        acc[j] = fmaf(df, df, acc[j]);
      }
    }
  __syncthreads();   // gm and red have been read
  for (int i = threadIdx.x; i < p.ng; i += blockDim.x) gm[i] = gm[i] / n;
  if constexpr (CK) {
    const CkRows ck(a, r0, nr);
#pragma unroll
    for (int i = 0; i < NV; ++i) gn_checkpoint<T, V>(a, p, d[i], ck, p.row + i * g.R, p.on && p.row + i * g.R < nr);
  }
  group_sums<V, FOLD>(g, p, acc, red, gr);
  if constexpr (MODE == HELD) {
    const JoinLanes jl(g, p, a.part);
    unsigned long long *out = a.part + p.unit * g.k * g.gs + p.chunk, pv[4];
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) pair_store(out + (long long)i * g.k, gm[i], gr[i]);
    __syncthreads();   // gm and gr have been read
    affine();
    jl.ahead(g, p, pv);
    fwd_join<T, MODE>(a, p, jl, pv, gm, gr);
  } else {
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) gr[i] = 1.f / sqrtf(gr[i] / n + a.eps);
    __syncthreads();
  }
  fwd_statistics(a, p, gm, gr);
  if (!p.on) return;
  fwd_constants<V, VG>(gi, gm, gr, mu, sc);
  with_act(a.act, [&](auto act) {
#pragma unroll
    for (int i = 0; i < NV; ++i)
      if (p.row + i * g.R < nr)
        at<typename X::raw>(dst, ((uint32_t)(p.row + i * g.R) * g.C + p.c) * (uint32_t)sizeof(T)) =
            gn_y<T, V, VG, decltype(act)::value>(d[i], mu, sc, be);
  });
}

// The rounds of a staged tile.  The tiles of a unit take turns, so that at any time the chip reads few
// and compact stretches of memory (128 x 12544 x 96 backward 235 us; 245 with tiles in one piece).
struct Rounds {
  long long S;
  int turn, k, c, n;
  PG_DEVICE Rounds(const Geo &g, const Place &p) : S(g.S), turn(g.turn), k(g.k), c(p.chunk) {
    const long long all = (long long)turn * k, rest = S - (long long)c * turn;
    n = (int)((rest + all - 1) / all);
  }
  PG_DEVICE long long begin(int i) const { return ((long long)i * k + c) * turn; }
  PG_DEVICE int rows(int i) const { return (int)min((long long)turn, S - begin(i)); }
};

// staged: a tile is streamed, U rows a thread at a time, the next U already on their way
template <class T, int V, bool CK, bool FOLD>
__global__ __launch_bounds__(512, 4) void gn_fwd_staged_kernel(const FwdArgs a) {
  extern __shared__ float sm[];
  typedef Vec<T, V> X;
  constexpr int U = 4, VG = FOLD ? 1 : V;
  const Geo &g = a.g;
  const Place p = place<V, STAGED>(g);
  float *gm = sm, *gr = sm + g.gs, *red = sm + 2 * g.gs;
  int gi[VG];
#pragma unroll
  for (int j = 0; j < VG; ++j) gi[j] = (p.c - p.c0 + j) / g.cg;
  const Rounds rd(g, p);
  // byte offsets of this thread's rows in a round; past the tensor's end, the last row's
  const uint32_t hop = (uint32_t)g.R * g.C * (uint32_t)sizeof(T), first = ((uint32_t)p.row * g.C + p.c) * (uint32_t)sizeof(T);
  auto load = [&](typename X::raw (&d)[U], int i) {
    const T *src = static_cast<const T *>(a.x) + (p.b * g.S + rd.begin(i)) * g.C;
    const uint32_t last = ((uint32_t)(rd.rows(i) - 1) * g.C + p.c) * (uint32_t)sizeof(T);
#pragma unroll
    for (int u = 0; u < U; ++u) d[u] = at<typename X::raw>(src, min(first + u * hop, last));
  };
  const JoinLanes jl(g, p, a.part);
  unsigned long long pv[4];
  if (p.use) jl.ahead(g, p, pv);
  typename X::raw d[U], nx[U];
  load(d, 0);
  auto stream = [&](auto f) {
    const int rounds = rd.n;
    auto work = [&](const typename X::raw (&v)[U], int i) {
      const long long r0 = p.b * g.S + rd.begin(i);
      const int nr = rd.rows(i);
#pragma unroll
      for (int u = 0; u < U; ++u) f(v[u], r0, p.row + u * g.R, nr, first + u * hop);
    };
#pragma unroll 1
    for (int i = 0; i < rounds; i += 2) {
      if (i + 1 < rounds) load(nx, i + 1);
      work(d, i);
      if (i + 1 < rounds) {
        if (i + 2 < rounds) load(d, i + 2);
        work(nx, i + 1);
      }
    }
  };
  if (!p.use) {
    // Sums of x - K and its square, K this thread's first values: nothing is lost where the mean is
    // far from 0, and a K that lies far out spoils one thread's share at most.
    float K[VG], s1[VG], s2[VG], f[V], acc[V];
    X::unpack(d[0], f);
#pragma unroll
    for (int j = 0; j < VG; ++j) {
      K[j] = f[j];
      s1[j] = s2[j] = 0.f;
    }
    if constexpr (FOLD) {
#pragma unroll
      for (int j = 1; j < V; ++j) K[0] += f[j];
      K[0] *= 1.f / V;
    }
    int rows = 0;
    stream([&](const typename X::raw &raw, long long r0, int r, int nr, uint32_t) {
      if constexpr (CK) gn_checkpoint<T, V>(a, p, raw, CkRows(a, r0, nr), r, p.on && r < nr);
      if (r < nr) {
        float v[V];
        X::unpack(raw, v);
#pragma unroll
        for (int j = 0; j < V; ++j) {
          const float df = v[j] - K[FOLD ? 0 : j];
          s1[FOLD ? 0 : j] += df;
          s2[FOLD ? 0 : j] = fmaf(df, df, s2[FOLD ? 0 : j]);
        }
        ++rows;
      }
    });
    // this thread's means, then the groups' mean, then the squares about that
    const float n = (float)(FOLD ? rows * V : rows), rn = n > 0.f ? 1.f / n : 0.f;
#pragma unroll
    for (int j = 0; j < V; ++j) acc[j] = FOLD && j ? 0.f : fmaf(n, K[FOLD ? 0 : j], s1[FOLD ? 0 : j]);
    group_sums<V, FOLD>(g, p, acc, red, gm);
    const float cn = 1.f / (tile_rows<STAGED>(g, p.chunk) * (float)g.cg);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      const int k = FOLD ? 0 : j;
      const float df = fmaf(s1[k], rn, K[k]) - gm[gi[k]] * cn;
      const float own = fmaf(-s1[k] * rn, s1[k], s2[k]);   // a NaN stays
      acc[j] = FOLD && j ? 0.f : (own < 0.f ? 0.f : own) + n * df * df;
    }
    __syncthreads();
    group_sums<V, FOLD>(g, p, acc, red, gr);
    unsigned long long *out = a.part + p.unit * g.k * g.gs + p.chunk;
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) pair_store(out + (long long)i * g.k, gm[i] * cn, gr[i]);
    return;
  }
  float mu[VG], sc[V], be[V];
  channel_values(a.gamma, a.mean, p.c, 1.f, sc);
  channel_values(a.beta, a.mean, p.c, 0.f, be);
  fwd_join<T, STAGED>(a, p, jl, pv, gm, gr);
  fwd_statistics(a, p, gm, gr);
  if (!p.on) return;
  fwd_constants<V, VG>(gi, gm, gr, mu, sc);
  with_act(a.act, [&](auto act) {
    stream([&](const typename X::raw &raw, long long r0, int r, int nr, uint32_t off) {
      const rsrc_t y = make_rsrc(static_cast<T *>(a.y) + r0 * g.C, (uint32_t)nr * g.C * (uint32_t)sizeof(T));
      buf_store(y, r < nr ? off : kOOB, gn_y<T, V, VG, decltype(act)::value>(raw, mu, sc, be));
    });
  });
}

// ---- backward --------------------------------------------------------------------------------
struct BwdArgs {
  Geo g;
  const void *dy, *x;
  const uint8_t *q, *qs;
  const float *gamma, *beta, *mean, *rstd;
  void *dx;
  unsigned long long *part;   // [B * nslab][gs][k]: s1, s2 of every tile and group
  float *dpart;   // [B * k][2][C]: dgamma, dbeta of every tile, or null
  int act;
};

// Which values of a channel relu and relu6 pass: lo < x < hi.  0 < z (and z < 6) is a condition on x
// itself, x > mean - beta / (rstd gamma) or < where gamma < 0.  The border is found in 64 bits, once a
// channel, and rounded away from the side that passes, so the comparison of x, which is exact in
// fp32, with it tells what z in 64 bits would: no rounding of z takes part.  A border that is not there is
// NaN: nothing, infinities among them, lies behind it (a NaN z, of a group with infinite values, passes).
PG_DEVICE void gn_border(int act, float mean, float rstd, float gamma, float beta, float &lo, float &hi) {
  const double k = (double)rstd * (double)gamma, b = beta;
  lo = hi = NAN;
  if (act != GN_RELU && act != GN_RELU6) return;
  if (k == 0.0) {   // z is beta everywhere
    if (beta <= 0.f || (act == GN_RELU6 && beta >= 6.f)) lo = INFINITY;
    return;
  }
  const double r = 1.0 / k, t0 = fma(-b, r, (double)mean), t6 = fma(6.0 - b, r, (double)mean);
  if (k > 0.0) {
    lo = __double2float_rd(t0);
    if (act == GN_RELU6) hi = __double2float_ru(t6);
  } else {
    hi = __double2float_ru(t0);
    if (act == GN_RELU6) lo = __double2float_rd(t6);
  }
}

// act'(z) dy.  SILU: u, v are rstd gamma and beta, and df is x - mean; otherwise the borders of x.
// NaN passes.
template <bool SILU> PG_DEVICE float gn_dz(float dy, float x, float df, float u, float v) {
  if constexpr (SILU) {
    const float z = fmaf(df, u, v), s = 1.f / (1.f + __expf(-z));
    return dy * (s * fmaf(z, 1.f - s, 1.f));
  } else {
    return x <= u || x >= v ? 0.f : dy;
  }
}

// Shared memory of a backward workgroup: what its channels need (gamma, rstd gamma, and gn_dz's u and
// v), the sums of its channels and groups, the rows of the reduction.
struct BwdShared {
  float *ga, *al, *u, *v, *tot, *g1, *g2, *red2, *red;
  PG_DEVICE BwdShared(const Geo &g, float *sm)
      : ga(sm), al(ga + g.cs), u(al + g.cs), v(u + g.cs), tot(v + g.cs), g1(tot + 2 * g.cs), g2(g1 + g.gs),
        red2(g2 + g.gs), red(red2 + 2 * blockDim.x) {}
  // one channel's values: asked for early, put down when they are here
  struct Channel { float ga[1], be[1], mean, rstd; };
  static PG_DEVICE void ask(const BwdArgs &a, const Place &p, const float *mean, const float *rstd, int c, Channel &k) {
    channel_values(a.gamma, rstd, p.c0 + c, 1.f, k.ga);
    channel_values(a.beta, rstd, p.c0 + c, 0.f, k.be);
    k.mean = at<float>(mean, (c / a.g.cg) * 4u);
    k.rstd = at<float>(rstd, (c / a.g.cg) * 4u);
  }
  template <bool SILU>
  PG_DEVICE void put(const BwdArgs &a, const Place &p, const float *mean, const float *rstd, Channel &k) const {
    for (int c = threadIdx.x; c < p.csl; c += blockDim.x) {
      if (c != (int)threadIdx.x) ask(a, p, mean, rstd, c, k);
      ga[c] = k.ga[0];
      al[c] = k.rstd * k.ga[0];
      if constexpr (SILU) {
        u[c] = al[c];
        v[c] = k.be[0];
      } else {
        gn_border(a.act, k.mean, k.rstd, k.ga[0], k.be[0], u[c], v[c]);
      }
    }
    __syncthreads();
  }
};

// what a thread needs of its channels, and the rows it reads
template <class T, int V, bool CK, bool FOLD, bool SILU> struct BwdThread {
  typedef Vec<T, V> X;
  static constexpr int VG = FOLD ? 1 : V;
  struct Row {
    typename X::raw dy;
    typename std::conditional<CK, typename Codes<V>::raw, typename X::raw>::type x;
    uint8_t sc;   // checkpoint: the scale's byte
  };
  int gi[VG];   // slab group of each channel (FOLD: of all)
  float mu[VG], rs[VG], u[V], v[V];

  PG_DEVICE void groups(const Geo &g, const Place &p, const float *mean, const float *rstd) {
#pragma unroll
    for (int j = 0; j < VG; ++j) {
      gi[j] = (p.c - p.c0 + j) / g.cg;
      mu[j] = at<float>(mean, gi[j] * 4u);
      rs[j] = at<float>(rstd, gi[j] * 4u);
    }
  }
  PG_DEVICE void channels(const Place &p, const BwdShared &m) {
#pragma unroll
    for (int j = 0; j < V; ++j) {
      u[j] = m.u[p.c - p.c0 + j];
      v[j] = m.v[p.c - p.c0 + j];
    }
  }
  // the row at element offset o (and scale offset os) of the tile that begins at row r0 of the tensor
  static PG_DEVICE void load(const BwdArgs &a, long long r0, uint32_t o, uint32_t os, Row &d) {
    const int nb = (a.g.C + kMxBlock - 1) / kMxBlock;
    d.dy = at<typename X::raw>(static_cast<const T *>(a.dy) + r0 * a.g.C, o * (uint32_t)sizeof(T));
    if constexpr (CK) {
      d.x = at<typename Codes<V>::raw>(a.q + r0 * a.g.C, o);
      d.sc = at<uint8_t>(a.qs + r0 * nb, os);
    } else {
      d.x = at<typename X::raw>(static_cast<const T *>(a.x) + r0 * a.g.C, o * (uint32_t)sizeof(T));
    }
  }
  // x - mean and dz of a row (DONE: dy holds dz)
  template <bool DONE> PG_DEVICE void row(const Row &d, float (&df)[V], float (&dz)[V]) const {
    float f[V];
    if constexpr (CK) Codes<V>::decode(d.x, mx8_scale(d.sc), f);
    else X::unpack(d.x, f);
    X::unpack(d.dy, dz);
#pragma unroll
    for (int j = 0; j < V; ++j) {
      df[j] = f[j] - mu[FOLD ? 0 : j];
      if constexpr (!DONE) dz[j] = gn_dz<SILU>(dz[j], f[j], df[j], u[j], v[j]);
    }
  }
};

// s1 = sum dz (x - mean), s0 = sum dz of the thread -> tot[c] = dgamma, tot[cs + c] = dbeta of the
// tile (and to dpart), g1, g2 = s1, s2 of its groups
template <int V>
PG_DEVICE void bwd_sums(const BwdArgs &a, const Place &p, const float *rstd, const float (&s1)[V], const float (&s0)[V],
                        const BwdShared &m) {
  const Geo &g = a.g;
  const int ld = g.CVp * V, t = threadIdx.x, n = p.csl, nt = blockDim.x / n;
  const float rs = at<float>(rstd, min(t, n - 1) / g.cg * 4u);
  float *redb = m.red + blockDim.x * V;
  if (p.on) {
#pragma unroll
    for (int j = 0; j < V; ++j) m.red[p.row * ld + p.col * V + j] = s1[j];
#pragma unroll
    for (int j = 0; j < V; ++j) redb[p.row * ld + p.col * V + j] = s0[j];
  }
  __syncthreads();
  if (nt <= 1) {
    for (int o = t; o < n; o += blockDim.x) {
      m.tot[o] = col_sum(m.red + o, 0, g.R, 1, ld) * (o == t ? rs : rstd[o / g.cg]);
      m.tot[g.cs + o] = col_sum(redb + o, 0, g.R, 1, ld);
    }
  } else {   // nt stripes of rows a channel
    const int st = t / n, o = t - st * n;
    if (st < nt) {
      m.red2[st * n + o] = col_sum(m.red + o, st, g.R, nt, ld);
      m.red2[blockDim.x + st * n + o] = col_sum(redb + o, st, g.R, nt, ld);
    }
    __syncthreads();
    if (t < n) {
      m.tot[t] = col_sum(m.red2 + t, 0, nt, 1, n) * rs;
      m.tot[g.cs + t] = col_sum(m.red2 + blockDim.x + t, 0, nt, 1, n);
    }
  }
  __syncthreads();
  if (a.dpart) {
    float *dst = a.dpart + (p.b * g.k + p.chunk) * 2 * g.C + p.c0;
    for (int j = t; j < n; j += blockDim.x) {
      dst[j] = m.tot[j];
      dst[g.C + j] = m.tot[g.cs + j];
    }
  }
  const int W = seg_width(g.cg), per = 64 / W, lane = t & 63, l = lane & (W - 1);
  for (int i = (t >> 6) * per + lane / W; i - lane / W < p.ng; i += (blockDim.x >> 6) * per) {
    float u = 0.f, v = 0.f;
    if (i < p.ng)
      for (int c = i * g.cg + l; c < (i + 1) * g.cg; c += W) {
        u = fmaf(m.ga[c], m.tot[g.cs + c], u);
        v = fmaf(m.ga[c], m.tot[c], v);
      }
    u = seg_sum(u, W);
    v = seg_sum(v, W);
    if (l == 0 && i < p.ng) {
      m.g1[i] = u;
      m.g2[i] = v;
    }
  }
  __syncthreads();
}

// dx = dz al - (k1 + (x - mean) k2)
template <class T, int V, int VG>
PG_DEVICE typename Vec<T, V>::raw gn_dx(const float (&df)[V], const float (&dz)[V], const float (&al)[V],
                                        const float (&k1)[VG], const float (&k2)[VG]) {
  float f[V];
#pragma unroll
  for (int j = 0; j < V; ++j) f[j] = fmaf(dz[j], al[j], -fmaf(df[j], k2[VG == 1 ? 0 : j], k1[VG == 1 ? 0 : j]));
  return Vec<T, V>::pack(f);
}
template <int V, int VG>
PG_DEVICE void bwd_constants(const Geo &g, const Place &p, const float (&rs)[VG], const int (&gi)[VG], const BwdShared &m,
                             float (&al)[V], float (&k1)[VG], float (&k2)[VG]) {
  const float rm = 1.f / ((float)g.S * (float)g.cg);
#pragma unroll
  for (int j = 0; j < VG; ++j) {
    k1[j] = rs[j] * m.g1[gi[j]] * rm;
    k2[j] = rs[j] * rs[j] * m.g2[gi[j]] * rm;
  }
#pragma unroll
  for (int j = 0; j < V; ++j) al[j] = m.al[p.c - p.c0 + j];
}

// g1, g2 = s1, s2 of the unit's groups
template <class T, bool CK, bool SILU>
PG_DEVICE void bwd_join(const BwdArgs &a, const Place &p, const float *mean, const float *rstd, const JoinLanes &q,
                        unsigned long long (&pv)[4], const BwdShared &m) {
  const Geo &g = a.g;
  for (int i = q.i0; i - q.lane / q.W < p.ng; i += (blockDim.x >> 6) * q.per) {
    float u = 0.f, v = 0.f;
    const int gc = min(i, p.ng - 1);
    const unsigned long long *in = q.in + (long long)gc * g.k;
    if (i != q.i0) pairs_ahead(in, g.k, q.l, q.W, 0, pv);
    if (!pairs(in, g.k, q.l, q.W, g.wait, pv, [&](int, float s1, float s2) {
          u += s1;
          v += s2;
        })) {   // as in the forward
      u = v = 0.f;
      const int nb = (g.C + kMxBlock - 1) / kMxBlock;
      const float mu = mean[gc], rs = rstd[gc];
#pragma unroll 1
      for (long long r = p.b * g.S + q.l; r < (p.b + 1) * g.S; r += q.W)
#pragma unroll 1
        for (int c = gc * g.cg; c < (gc + 1) * g.cg; ++c) {
          const long long at = r * g.C + p.c0 + c;
          float x;
          if constexpr (CK) x = mx8_dec1(a.q[at]) * mx8_scale(a.qs[r * nb + (p.c0 + c) / kMxBlock]);
          else x = tof(static_cast<const T *>(a.x)[at]);
          const float z = gn_dz<SILU>(tof(static_cast<const T *>(a.dy)[at]), x, x - mu, m.u[c], m.v[c]);
          u = fmaf(m.ga[c], z, u);
          v = fmaf(m.ga[c] * rs * (x - mu), z, v);
        }
    }
    u = seg_sum(u, q.W);
    v = seg_sum(v, q.W);
    if (q.l == 0 && i < p.ng) {
      m.g1[i] = u;
      m.g2[i] = v;
    }
  }
  __syncthreads();
}

// solo, held: as in the forward
template <class T, int V, int NV, int MODE, bool CK, bool FOLD, bool SILU>
__global__ __launch_bounds__(1024) void gn_bwd_solo_kernel(const BwdArgs a) {
  extern __shared__ float sm[];
  typedef Vec<T, V> X;
  typedef BwdThread<T, V, CK, FOLD, SILU> Th;
  const Geo &g = a.g;
  const Place p = place<V, MODE>(g);
  const BwdShared m(g, sm);
  const float *mean = a.mean + p.b * g.G + p.g0, *rstd = a.rstd + p.b * g.G + p.g0;
  const long long s0 = MODE == HELD ? (long long)p.chunk * g.rows : 0, r0 = p.b * g.S + s0;
  const int nr = (int)(MODE == HELD ? min((long long)g.rows, g.S - s0) : g.S);
  Th th;
  BwdShared::Channel own;
  th.groups(g, p, mean, rstd);
  BwdShared::ask(a, p, mean, rstd, min((int)threadIdx.x, p.csl - 1), own);
  typename Th::Row d[NV];
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const uint32_t r = min(p.row + i * g.R, nr - 1);
    Th::load(a, r0, r * g.C + p.c, r * ((g.C + kMxBlock - 1) / kMxBlock) + p.c / kMxBlock, d[i]);
  }
  m.put<SILU>(a, p, mean, rstd, own);
  th.channels(p, m);
  float s1[V], s2[V];
#pragma unroll
  for (int j = 0; j < V; ++j) s1[j] = s2[j] = 0.f;
#pragma unroll
  for (int i = 0; i < NV; ++i)
    if (p.row + i * g.R < nr) {
      float df[V], dz[V];
      th.template row<false>(d[i], df, dz);
      if constexpr (!SILU) d[i].dy = X::pack(dz);   // dy or 0: it takes dy's place for the second use
#pragma unroll
      for (int j = 0; j < V; ++j) {
        s1[j] = fmaf(dz[j], df[j], s1[j]);
        s2[j] += dz[j];
      }
    }
  bwd_sums<V>(a, p, rstd, s1, s2, m);
  if constexpr (MODE == HELD) {
    const JoinLanes jl(g, p, a.part);
    unsigned long long *out = a.part + p.unit * g.k * g.gs + p.chunk, pv[4];
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) pair_store(out + (long long)i * g.k, m.g1[i], m.g2[i]);
    __syncthreads();   // g1 and g2 have been read
    jl.ahead(g, p, pv);
    bwd_join<T, CK, SILU>(a, p, mean, rstd, jl, pv, m);
  }
  if (!p.on) return;
  float al[V], k1[Th::VG], k2[Th::VG];
  bwd_constants<V, Th::VG>(g, p, th.rs, th.gi, m, al, k1, k2);
  T *dst = static_cast<T *>(a.dx) + r0 * g.C;
#pragma unroll
  for (int i = 0; i < NV; ++i) {
    const int r = p.row + i * g.R;
    if (r < nr) {
      float df[V], dz[V];
      th.template row<!SILU>(d[i], df, dz);
      at<typename X::raw>(dst, ((uint32_t)r * g.C + p.c) * (uint32_t)sizeof(T)) = gn_dx<T, V, Th::VG>(df, dz, al, k1, k2);
    }
  }
}

template <class T, int V, bool CK, bool FOLD, bool SILU>
__global__ __launch_bounds__(256, SILU || !FOLD ? 3 : 4) void gn_bwd_staged_kernel(const BwdArgs a) {
  extern __shared__ float sm[];
  typedef Vec<T, V> X;
  typedef BwdThread<T, V, CK, FOLD, SILU> Th;
  constexpr int U = 2;
  const Geo &g = a.g;
  const Place p = place<V, STAGED>(g);
  const BwdShared m(g, sm);
  const float *mean = a.mean + p.b * g.G + p.g0, *rstd = a.rstd + p.b * g.G + p.g0;
  const Rounds rd(g, p);
  // offsets of this thread's rows in a round in elements and in scales; past the end, the last row's
  const uint32_t nb = (g.C + kMxBlock - 1) / kMxBlock, hop = (uint32_t)g.R * g.C, hops = g.R * nb;
  const uint32_t first = (uint32_t)p.row * g.C + p.c, firsts = p.row * nb + p.c / kMxBlock;
  auto load = [&](typename Th::Row (&d)[U], int i) {
    const uint32_t end = rd.rows(i) - 1, last = end * g.C + p.c, lasts = end * nb + p.c / kMxBlock;
#pragma unroll
    for (int u = 0; u < U; ++u)
      Th::load(a, p.b * g.S + rd.begin(i), min(first + u * hop, last), CK ? min(firsts + u * hops, lasts) : 0, d[u]);
  };
  const JoinLanes jl(g, p, a.part);
  unsigned long long pv[4];
  if (p.use) jl.ahead(g, p, pv);
  Th th;
  BwdShared::Channel own;
  th.groups(g, p, mean, rstd);
  BwdShared::ask(a, p, mean, rstd, min((int)threadIdx.x, p.csl - 1), own);
  typename Th::Row d[U], nx[U];
  load(d, 0);
  m.put<SILU>(a, p, mean, rstd, own);
  th.channels(p, m);
  auto stream = [&](auto f) {
    const int rounds = rd.n;
    auto work = [&](const typename Th::Row (&v)[U], int i) {
      const long long r0 = p.b * g.S + rd.begin(i);
      const int nr = rd.rows(i);
#pragma unroll
      for (int u = 0; u < U; ++u) {
        float df[V], dz[V];
        th.template row<false>(v[u], df, dz);
        f(df, dz, r0, nr, p.row + u * g.R, first + u * hop);
      }
    };
#pragma unroll 1
    for (int i = 0; i < rounds; i += 2) {
      if (i + 1 < rounds) load(nx, i + 1);
      work(d, i);
      if (i + 1 < rounds) {
        if (i + 2 < rounds) load(d, i + 2);
        work(nx, i + 1);
      }
    }
  };
  if (!p.use) {
    float s0[V], s1[V];
#pragma unroll
    for (int j = 0; j < V; ++j) s0[j] = s1[j] = 0.f;
    stream([&](const float (&df)[V], const float (&dz)[V], long long, int nr, int r, uint32_t) {
      if (r < nr) {
#pragma unroll
        for (int j = 0; j < V; ++j) {
          s1[j] = fmaf(dz[j], df[j], s1[j]);
          s0[j] += dz[j];
        }
      }
    });
    bwd_sums<V>(a, p, rstd, s1, s0, m);
    unsigned long long *out = a.part + p.unit * g.k * g.gs + p.chunk;
    for (int i = threadIdx.x; i < p.ng; i += blockDim.x) pair_store(out + (long long)i * g.k, m.g1[i], m.g2[i]);
    return;
  }
  bwd_join<T, CK, SILU>(a, p, mean, rstd, jl, pv, m);
  if (!p.on) return;
  float al[V], k1[Th::VG], k2[Th::VG];
  bwd_constants<V, Th::VG>(g, p, th.rs, th.gi, m, al, k1, k2);
  stream([&](const float (&df)[V], const float (&dz)[V], long long r0, int nr, int r, uint32_t o) {
    const rsrc_t dx = make_rsrc(static_cast<T *>(a.dx) + r0 * g.C, (uint32_t)nr * g.C * (uint32_t)sizeof(T));
    buf_store(dx, r < nr ? o * (uint32_t)sizeof(T) : kOOB, gn_dx<T, V, Th::VG>(df, dz, al, k1, k2));
  });
}

// ---- launch ------------------------------------------------------------------------------------
struct Plan {
  Geo g;
  int V, NV, TH, mode;
  long long wgs;
};

struct Fwd {
  typedef FwdArgs Args;
  template <int MODE, bool SILU> static constexpr int most = 8;   // NV at most
  template <bool CK> static constexpr bool held = !CK;
  template <class T, int V, int NV, int MODE, bool CK, bool FOLD, bool SILU> static constexpr auto solo() {
    return gn_fwd_solo_kernel<T, V, NV, MODE, CK, FOLD>;
  }
  template <class T, int V, bool CK, bool FOLD, bool SILU> static constexpr auto staged() {
    return gn_fwd_staged_kernel<T, V, CK, FOLD>;
  }
};
struct Bwd {
  typedef BwdArgs Args;
  template <int MODE, bool SILU> static constexpr int most = MODE == SOLO || SILU ? 4 : 8;
  template <bool CK> static constexpr bool held = true;
  template <class T, int V, int NV, int MODE, bool CK, bool FOLD, bool SILU> static constexpr auto solo() {
    return gn_bwd_solo_kernel<T, V, NV, MODE, CK, FOLD, SILU>;
  }
  template <class T, int V, bool CK, bool FOLD, bool SILU> static constexpr auto staged() {
    return gn_bwd_staged_kernel<T, V, CK, FOLD, SILU>;
  }
};

// the plan gives NV 2, 4 and (up to `most`) 8 to full vectors of one group each, 2 to vectors of 8 that straddle groups
// (their constants take the registers), 4 to narrower ones
template <class D, class T, int VMAX, bool CK, bool SILU>
void launch(const Plan &p, size_t lds, const typename D::Args &a, hipStream_t st) {
  auto go = [&](auto kernel) { hipLaunchKernelGGL(kernel, dim3((unsigned)p.wgs), dim3(p.TH), lds, st, a); };
  const bool full = p.V == VMAX, fold = full && p.g.cg % VMAX == 0;
  if (p.mode == STAGED) {
    if (fold) go(D::template staged<T, VMAX, CK, true, SILU>());
    else if (full) go(D::template staged<T, VMAX, CK, false, SILU>());
    else if (VMAX == 8 && p.V == 4) go(D::template staged<T, 4, CK, false, SILU>());
    else if (p.V == 2) go(D::template staged<T, 2, CK, false, SILU>());
    else go(D::template staged<T, 1, CK, false, SILU>());
    return;
  }
  auto solo = [&](auto mode) {
    constexpr int M = decltype(mode)::value;
    constexpr int most = D::template most<M, SILU>;
    if (fold && p.NV == 2) go(D::template solo<T, VMAX, 2, M, CK, true, SILU>());
    else if (fold && p.NV == most) go(D::template solo<T, VMAX, most, M, CK, true, SILU>());
    else if (fold) go(D::template solo<T, VMAX, 4, M, CK, true, SILU>());
    else if (full) go(D::template solo<T, VMAX, VMAX == 4 ? 4 : 2, M, CK, false, SILU>());
    else if (VMAX == 8 && p.V == 4) go(D::template solo<T, 4, 4, M, CK, false, SILU>());
    else if (p.V == 2) go(D::template solo<T, 2, 4, M, CK, false, SILU>());
    else go(D::template solo<T, 1, 4, M, CK, false, SILU>());
  };
  if (p.mode == SOLO) solo(std::integral_constant<int, SOLO>());
  else if constexpr (D::template held<CK>) solo(std::integral_constant<int, HELD>());
}

// one translation unit per direction and type
void fwd_bf16(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st);
void fwd_fp16(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st);
void fwd_fp32(const Plan &p, size_t lds, const FwdArgs &a, hipStream_t st);
void bwd_bf16(const Plan &p, size_t lds, const BwdArgs &a, hipStream_t st);
void bwd_fp16(const Plan &p, size_t lds, const BwdArgs &a, hipStream_t st);
void bwd_fp32(const Plan &p, size_t lds, const BwdArgs &a, hipStream_t st);
}  // namespace gn
