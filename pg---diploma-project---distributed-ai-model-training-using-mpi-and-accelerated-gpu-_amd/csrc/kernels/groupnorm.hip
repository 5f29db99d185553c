// Group norm: geometry, workspace and launches (groupnorm.h holds the kernels), and the sums over
// images and tiles that give dgamma and dbeta.
#include "../groupnorm.h"

#include <algorithm>
#include <numeric>
#include <stdexcept>

using namespace gn;

namespace {
// Work-items of a launch: the runtime takes 2^32 and more without a word and runs what is left modulo 2^32
// (gn_bwd of 2050 x 2 x 8200 left most gradients unwritten).
constexpr long long kMostItems = 0xffffffffll;
constexpr long long kMostWgs = 65536;   // of kernels that loop: more than are resident, many times over

// ---- wide: not tuned, every access one value ------------------------------------------------------
// Plain loops over memory, with grids of kMostWgs workgroups at most, for slabs that no workgroup holds: C / G of
// thousands of channels, or over a thousand of an odd number; sums past the shared memory; checkpoint blocks of odd
// widths (groupnorm.h).
PG_DEVICE float load_one(const void *x, int dt, long long i) {
  return dt == 0 ? bf2f(static_cast<const bf16_t *>(x)[i])
                 : dt == 1 ? (float)static_cast<const _Float16 *>(x)[i] : static_cast<const float *>(x)[i];
}
PG_DEVICE void store_one(void *y, int dt, long long i, float v) {
  if (dt == 0) static_cast<bf16_t *>(y)[i] = f2bf(v);
  else if (dt == 1) static_cast<_Float16 *>(y)[i] = (_Float16)v;
  else static_cast<float *>(y)[i] = v;
}
PG_DEVICE float block_sum(float v) {   // 256 threads
  __shared__ float sh[4];
  v = wave_sum(v);
  __syncthreads();
  if ((threadIdx.x & 63) == 0) sh[threadIdx.x >> 6] = v;
  __syncthreads();
  return (sh[0] + sh[1]) + (sh[2] + sh[3]);
}

__global__ __launch_bounds__(256) void gn_wide_stats_kernel(const FwdArgs a, int dt) {
  const Geo &g = a.g;
  const long long n = g.S * g.cg;
  for (long long k = blockIdx.x; k < g.B * g.G; k += gridDim.x) {
    const long long base = k / g.G * g.S * g.C + k % g.G * g.cg;
    float s = 0.f, v = 0.f;
    for (long long i = threadIdx.x; i < n; i += 256) s += load_one(a.x, dt, base + i / g.cg * g.C + i % g.cg);
    const float mu = block_sum(s) / (float)n;
    for (long long i = threadIdx.x; i < n; i += 256) {
      const float d = load_one(a.x, dt, base + i / g.cg * g.C + i % g.cg) - mu;
      v = fmaf(d, d, v);
    }
    v = block_sum(v);
    if (threadIdx.x == 0) {
      a.mean[k] = mu;
      a.rstd[k] = 1.f / sqrtf(v / (float)n + a.eps);
    }
  }
}
__global__ __launch_bounds__(256) void gn_wide_apply_kernel(const FwdArgs a, int dt) {
  const Geo &g = a.g;
  const long long n = g.B * g.S * g.C;
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const int c = (int)(i % g.C);
    const long long k = i / (g.S * g.C) * g.G + c / g.cg;
    const float z = fmaf(load_one(a.x, dt, i) - a.mean[k], a.rstd[k] * (a.gamma ? a.gamma[c] : 1.f),
                         a.beta ? a.beta[c] : 0.f);
    store_one(a.y, dt, i, a.act == GN_RELU6 ? gn_act<GN_RELU6>(z) : a.act == GN_RELU ? gn_act<GN_RELU>(z)
                              : a.act == GN_SILU ? gn_act<GN_SILU>(z) : z);
  }
}

// value i's x - mean, gamma rstd and dz
PG_DEVICE void wide_dz(const BwdArgs &a, int dt, long long r, int c, float &df, float &al, float &dz) {
  const Geo &g = a.g;
  const long long i = r * g.C + c, b = r / g.S, k = b * g.G + c / g.cg;
  const int nb = (g.C + kMxBlock - 1) / kMxBlock;
  const float x = a.q ? mx8_dec1(a.q[i]) * mx8_scale(a.qs[r * nb + c / kMxBlock]) : load_one(a.x, dt, i);
  const float ga = a.gamma ? a.gamma[c] : 1.f, be = a.beta ? a.beta[c] : 0.f, dy = load_one(a.dy, dt, i);
  df = x - a.mean[k];
  al = a.rstd[k] * ga;
  if (a.act == GN_SILU) {
    dz = gn_dz<true>(dy, x, df, al, be);
  } else {
    float lo, hi;
    gn_border(a.act, a.mean[k], a.rstd[k], ga, be, lo, hi);
    dz = gn_dz<false>(dy, x, df, lo, hi);
  }
}
// a workgroup at a time per (image, channel) -> dpart [B][2][C]
__global__ __launch_bounds__(256) void gn_wide_dsums_kernel(const BwdArgs a, int dt) {
  const Geo &g = a.g;
  for (long long k = blockIdx.x; k < g.B * g.C; k += gridDim.x) {
    const long long b = k / g.C;
    const int c = (int)(k % g.C);
    float s0 = 0.f, s1 = 0.f, df, al, dz;
    for (long long s = threadIdx.x; s < g.S; s += 256) {
      wide_dz(a, dt, b * g.S + s, c, df, al, dz);
      s0 += dz;
      s1 = fmaf(dz, df, s1);
    }
    s0 = block_sum(s0);
    s1 = block_sum(s1);
    if (threadIdx.x == 0) {
      a.dpart[b * 2 * g.C + c] = s1 * a.rstd[b * g.G + c / g.cg];
      a.dpart[(b * 2 + 1) * g.C + c] = s0;
    }
  }
}
// a workgroup at a time per (image, group) -> part [B * G][2]
__global__ __launch_bounds__(256) void gn_wide_gsums_kernel(const BwdArgs a) {
  const Geo &g = a.g;
  for (long long k = blockIdx.x; k < g.B * g.G; k += gridDim.x) {
    const long long b = k / g.G;
    const int c0 = (int)(k % g.G) * g.cg;
    float u = 0.f, v = 0.f;
    for (int c = c0 + threadIdx.x; c < c0 + g.cg; c += 256) {
      const float ga = a.gamma ? a.gamma[c] : 1.f;
      v = fmaf(ga, a.dpart[b * 2 * g.C + c], v);
      u = fmaf(ga, a.dpart[(b * 2 + 1) * g.C + c], u);
    }
    u = block_sum(u);
    v = block_sum(v);
    if (threadIdx.x == 0) pair_store(a.part + k, u, v);
  }
}
__global__ __launch_bounds__(256) void gn_wide_dx_kernel(const BwdArgs a, int dt) {
  const Geo &g = a.g;
  const long long n = g.B * g.S * g.C;
  const float rm = 1.f / ((float)g.S * (float)g.cg);
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (long long)gridDim.x * 256) {
    const long long r = i / g.C;
    const int c = (int)(i % g.C);
    float df, al, dz;
    wide_dz(a, dt, r, c, df, al, dz);
    const long long k = r / g.S * g.G + c / g.cg;
    const unsigned long long w = a.part[k];
    const float rs = a.rstd[k], s1 = __uint_as_float((unsigned)w), s2 = __uint_as_float((unsigned)(w >> 32));
    store_one(a.dx, dt, i, fmaf(dz, al, -fmaf(df, rs * rs * s2 * rm, rs * s1 * rm)));
  }
}

// ---- dgamma, dbeta: column sums of [rows][n] in a fixed order -----------------------------------
// grid (columns / 64, row splits): 64 columns x 16 stripes of rows; with one split dst is the result
__global__ __launch_bounds__(1024) void gn_dparam_kernel(const float *__restrict__ part, float *__restrict__ dst,
                                                         long long rows, int n, int split) {
  __shared__ float sh[16][64];
  const int col = threadIdx.x & 63, st = threadIdx.x >> 6;
  const long long r0 = (long long)blockIdx.y * split, r1 = min(rows, r0 + split);
#pragma unroll 1
  for (long long j = blockIdx.x * 64ll + col; j - col < n; j += gridDim.x * 64ll) {
    float s = 0.f;
    if (j < n) {   // eight rows in flight
      float v[8] = {};
      long long r = r0 + st;
      for (; r + 7 * 16 < r1; r += 8 * 16) {
#pragma unroll
        for (int u = 0; u < 8; ++u) v[u] += part[(r + u * 16) * n + j];
      }
#pragma unroll
      for (int u = 0; u < 8; ++u) v[0] += r + u * 16 < r1 ? part[(r + u * 16) * n + j] : 0.f;
#pragma unroll
      for (int u = 0; u < 8; ++u) s += v[u];
    }
    sh[st][col] = s;
    __syncthreads();
    if (st == 0 && j < n) {
      s = 0.f;
#pragma unroll
      for (int i = 0; i < 16; ++i) s += sh[i][col];
      dst[(size_t)blockIdx.y * n + j] = s;
    }
    __syncthreads();   // sh has been read
  }
}

// no pair has come yet
__global__ __launch_bounds__(256) void gn_none_kernel(unsigned long long *__restrict__ p, long long n) {
  for (long long i = blockIdx.x * 256ll + threadIdx.x; i < n; i += (long long)gridDim.x * 256) p[i] = kNone;
}

// ---- host: geometry ----------------------------------------------------------------------------
// Held: all tiles at most (two of 512 threads are resident on each of 256 CUs), and tiles of a unit.  Units
// start in order, so at any time one unit of a launch is there in part and waits, and launches on the 4
// hardware queues together never fill the chip with tiles that wait for one another.
constexpr int kHeld = 480, kHeldUnit = 96;
// Staged: tiles wanted before tiles grow (256, 512, 1024, 2048: gn_bwd 96 x 784 x 192, were it not held, 33, 33,
// 40, 70 us)
constexpr int kTiles = 512;
// rounds of a tile at most, forward and backward (1, 2, 4, 6, 8, 16: gn_fwd 128 x 3136 x 144 with checkpoint 142,
// 89, 77, 82, 89, 89 us; gn_bwd 128 x 12544 x 96 675, 340, 253, 232, 236, 305): a workgroup costs some 12 us of
// latency however little it does, and with long ones the last tiles run alone
constexpr int kRounds[2] = {4, 6};
// sums workgroups ahead of the use workgroups at least: half of what is resident (128, 256, 512, 768, 1024: gn_bwd
// 128 x 12544 x 96 297, 282, 232, 233, 260 us; gn_fwd 128 x 3136 x 144 within 5%)
constexpr int kLead = 512;
constexpr int kSplitRows = 64;     // row splits of a long dgamma / dbeta sum
// looks (about a microsecond each) after which a waiting workgroup does without its peers
int g_wait = 1 << 16;

int gcd_pow2(long long c, int most) {
  int v = most;
  while (c % v) v >>= 1;
  return v;
}

// the sums and rows that a workgroup holds in shared memory
size_t gn_lds(const Plan &p, bool bwd) {
  const size_t red = (size_t)p.TH * (p.V + 1) * (bwd ? 2 : 1);
  return sizeof(float) * (2 * (size_t)p.g.gs + (bwd ? 6 : 1) * (size_t)p.g.cs + red);
}

// ck: with a checkpoint to write (forward), or as if there were; silu: backward through it
Plan gn_plan(int dt, long long B, long long S, int C, int G, bool ck, bool bwd, bool silu) {
  if (C > 0x3fffffff) throw std::invalid_argument("group norm: C is too large");
  Plan p{};
  Geo &g = p.g;
  g.B = B;
  g.S = S;
  g.C = C;
  g.G = G;
  g.cg = C / G;
  g.wait = g_wait;
  const int elt = dt == 2 ? 4 : 2;
  const int V = gcd_pow2(C, 16 / elt);
  p.V = V;
  const int only = V * elt < 16 ? 4 : g.cg % V ? (elt == 4 ? 4 : 2) : 0;   // NV of the kinds of vector that have one
  const int Q = ck && !bwd ? kMxBlock / V : 1;   // lanes of a checkpoint block
  // a slab is made of whole groups, vectors and (where they are written) checkpoint blocks
  long long L = std::lcm<long long>(g.cg, V);
  if (ck && !bwd) L = std::lcm<long long>(L, kMxBlock);
  if (L > C) L = C;
  auto shape = [&](long long cs) {
    g.cs = (int)std::min<long long>(cs, C);
    g.nslab = (C + g.cs - 1) / g.cs;
    g.gs = g.cs / g.cg;
    g.CVp = (g.cs / V + Q - 1) / Q * Q;
  };
  auto check = [&](long long k) {   // grid and in-tile offsets
    const bool grid = p.mode == SOLO || p.wgs <= kMostItems / p.TH;   // solo: in as many launches as it takes
    if (k > 0x7fffffff || !grid || (long long)std::max(g.turn, g.R * p.NV) * C * elt > 0x7fffffff)
      throw std::invalid_argument("group norm: sizes past the kernels' 32-bit grid and tile offsets");
  };
  const int most = bwd ? 512 : 1024;
  const int nvs[3] = {2, 4, 8};
  const int nv_most = bwd ? Bwd::most<SOLO, false> : Fwd::most<SOLO, false>;
  // solo: rows of 128 bytes at least, more while the tile is small and the chip stays full
  long long cs = (128 / elt + L - 1) / L * L;
  while (cs < C && S * cs * elt < 16384 && B * ((C + 2 * cs - 1) / (2 * cs)) >= 1024) cs *= 2;
  shape(cs);
  if (g.CVp <= 1024) {
    for (int nv : nvs) {
      if (nv > nv_most) break;
      if (only && nv != only) continue;
      const long long rows = (S + nv - 1) / nv;   // sweeps of R rows each
      const long long th = (rows * g.CVp + 63) / 64 * 64;
      if (th <= std::max(most, (g.CVp + 63) / 64 * 64) && th * nv <= 4096 + 64 * nv) {
        p.NV = nv;
        p.TH = (int)th;
        g.R = p.TH / g.CVp;
        g.k = 1;
        if (gn_lds(p, bwd) > 65536) break;
        p.mode = SOLO;
        p.wgs = B * g.nslab;
        check(1);
        return p;
      }
    }
  }
  // whole rows where they fit a workgroup, the fewest slabs otherwise
  auto slabs = [&](int th) {
    p.TH = th;
    for (long long n = 1;; ++n) {
      cs = ((C + n - 1) / n + L - 1) / L * L;
      shape(cs);
      if (g.CVp <= th || cs == L) break;
    }
    g.R = th / std::max(g.CVp, 1);
    return g.CVp <= th && gn_lds(p, bwd) <= 65536;
  };
  // Held: the fewest rows a thread with which all tiles are resident together.  Calls of 96 x 784 x 192, 32 x
  // 3136 x 96 and 16 x 3136 x 144, held and staged (us): forward 23, 21, 19 and 38, 24, 23; backward from a
  // checkpoint 27, 25, 23 and 33, 29, 29, from x 30, 27, 23 and 33, 27, 27.  Where a checkpoint is written held
  // is no faster with few rows (16 and 16) and has not the registers for 8 (35, 30, 25 and 40, 25, 22); silu's
  // backward neither (52, 48 and 43, 33 with 8).
  if (!(ck && !bwd) && slabs(512)) {
    for (int nv : nvs) {
      if ((only && nv != only) || (bwd && silu && nv > Bwd::most<HELD, true>)) continue;
      const long long rows = (long long)g.R * nv, k = (S + rows - 1) / rows;
      if (k > kHeldUnit || B * g.nslab * k > kHeld) continue;
      p.NV = nv;
      g.rows = (int)rows;
      g.k = (int)k;
      p.mode = HELD;
      p.wgs = B * g.nslab * k;
      check(k);
      return p;
    }
  }
  if (!slabs(bwd ? 256 : 512)) {
    p.mode = WIDE;
    g.k = 1;
    g.nslab = G;   // sums per (image, group)
    g.gs = 1;
    return p;
  }
  // tiles of up to kRounds rounds, fewer while the tiles do not fill the chip several times
  const long long round = (long long)g.R * (bwd ? 2 : 4), all = (S + round - 1) / round;
  const long long it = std::clamp<long long>(B * g.nslab * all / kTiles, 1, kRounds[bwd]);
  const long long k = (all + it - 1) / it;
  p.NV = 1;
  g.turn = (int)round;
  g.k = (int)k;
  p.mode = STAGED;
  g.tiles = (int)std::min<long long>(B * g.nslab * k, 0x7fffffff);
  g.lead = (int)std::min<long long>(std::min((kLead + k - 1) / k, B * g.nslab) * k, 0x7fffffff);
  p.wgs = 2 * B * g.nslab * k;
  check(k);
  return p;
}

struct Ws {
  long long part, dpart, lvl, total;   // offsets in floats
};
long long up4(long long n) { return (n + 3) / 4 * 4; }
Ws gn_ws(const Plan &p, bool bwd) {
  Ws w{};
  const Geo &g = p.g;
  if (p.mode != SOLO) {
    w.dpart = up4(g.B * g.nslab * g.k * g.gs * 2);
  }
  w.lvl = w.dpart;
  if (bwd) {
    const long long rows = g.B * g.k;
    w.lvl = w.dpart + rows * 2 * g.C;
    w.total = w.lvl + (rows > 16 * kSplitRows ? (long long)kSplitRows * 2 * g.C : 0);
  } else {
    w.total = w.lvl;
  }
  return w;
}

dim3 looped(long long wgs) { return dim3((unsigned)std::min(wgs, kMostWgs)); }

// one launch, or (solo, whose images have nothing to do with one another) as many as the grid needs: f(plan of the
// launch, its first image)
template <class F> void launches(const Plan &p, F f) {
  if (p.mode != SOLO) return f(p, 0);
  const long long most = std::max<long long>(1, kMostItems / p.TH / p.g.nslab);
  for (long long b = 0; b < p.g.B; b += most) {
    Plan part = p;
    part.wgs = std::min(most, p.g.B - b) * p.g.nslab;
    f(part, b);
  }
}

void gn_none(const Plan &p, unsigned long long *part, hipStream_t st) {
  if (p.mode != STAGED && p.mode != HELD) return;
  const long long n = p.g.B * p.g.nslab * p.g.k * p.g.gs;
  hipLaunchKernelGGL(gn_none_kernel, dim3((unsigned)std::min<long long>((n + 255) / 256, 2048)), dim3(256), 0, st, part, n);
}
}  // namespace

void launch_mx8_pack(int dt, const void *x, uint8_t *q, uint8_t *qs, long long M, int C, hipStream_t st);

// tests: -1, what has come is not looked at
void gn_set_wait(int polls) { g_wait = polls; }
// tests: the form (GnMode) that a call of these sizes takes
int gn_form(int dt, long long B, long long S, int C, int G, int ck, int bwd, int act) {
  return gn_plan(dt, B, S, C, G, ck && !bwd, bwd, bwd && act == GN_SILU).mode;
}

// dt: 0 bf16, 1 fp16, 2 fp32.  With and without a checkpoint (forward) or silu (backward): the largest.
long long gn_workspace_floats(int dt, long long B, long long S, int C, int G, int bwd) {
  if (B * S <= 0) return 0;
  return std::max(gn_ws(gn_plan(dt, B, S, C, G, false, bwd, false), bwd).total,
                  gn_ws(gn_plan(dt, B, S, C, G, true, bwd, true), bwd).total);
}

void launch_gn_fwd(int dt, const void *x, const float *gamma, const float *beta, void *y, float *mean, float *rstd,
                   uint8_t *q, uint8_t *qs, float *ws, long long B, long long S, int C, int G, float eps, int act,
                   int as_ckpt8, hipStream_t st) {
  const Plan p = gn_plan(dt, B, S, C, G, q != nullptr || as_ckpt8, false, false);
  const Ws w = gn_ws(p, false);
  const FwdArgs a{p.g, x, gamma, beta, y, mean, rstd, q, qs, reinterpret_cast<unsigned long long *>(ws + w.part), eps, act};
  gn_none(p, a.part, st);
  if (p.mode == WIDE) {
    hipLaunchKernelGGL(gn_wide_stats_kernel, looped(B * G), dim3(256), 0, st, a, dt);
    hipLaunchKernelGGL(gn_wide_apply_kernel, looped((B * S * C + 255) / 256), dim3(256), 0, st, a, dt);
    if (q) launch_mx8_pack(dt, x, q, qs, B * S, C, st);
    return;
  }
  const long long e = dt == 2 ? 4 : 2, nb = (C + kMxBlock - 1) / kMxBlock;
  launches(p, [&](const Plan &part, long long b) {
    FwdArgs t = a;
    t.x = static_cast<const char *>(x) + b * S * C * e;
    t.y = static_cast<char *>(y) + b * S * C * e;
    t.mean += b * G;
    t.rstd += b * G;
    if (q) {
      t.q += b * S * C;
      t.qs += b * S * nb;
    }
    (dt == 0 ? fwd_bf16 : dt == 1 ? fwd_fp16 : fwd_fp32)(part, gn_lds(p, false), t, st);
  });
}

void launch_gn_bwd(int dt, const void *dy, const void *x, const uint8_t *q, const uint8_t *qs, const float *gamma,
                   const float *beta, const float *mean, const float *rstd, void *dx, float *dgb, float *ws,
                   long long B, long long S, int C, int G, int act, hipStream_t st) {
  const Plan p = gn_plan(dt, B, S, C, G, false, true, act == GN_SILU);
  const Ws w = gn_ws(p, true);
  const BwdArgs a{p.g, dy, x, q, qs, gamma, beta, mean, rstd, dx, reinterpret_cast<unsigned long long *>(ws + w.part),
                  dgb || p.mode == WIDE ? ws + w.dpart : nullptr, act};
  gn_none(p, a.part, st);
  if (p.mode == WIDE) {
    hipLaunchKernelGGL(gn_wide_dsums_kernel, looped(B * C), dim3(256), 0, st, a, dt);
    hipLaunchKernelGGL(gn_wide_gsums_kernel, looped(B * G), dim3(256), 0, st, a);
    hipLaunchKernelGGL(gn_wide_dx_kernel, looped((B * S * C + 255) / 256), dim3(256), 0, st, a, dt);
  } else {
    const long long e = dt == 2 ? 4 : 2, nb = (C + kMxBlock - 1) / kMxBlock;
    launches(p, [&](const Plan &part, long long b) {
      BwdArgs t = a;
      t.dy = static_cast<const char *>(dy) + b * S * C * e;
      t.dx = static_cast<char *>(dx) + b * S * C * e;
      if (q) {
        t.q += b * S * C;
        t.qs += b * S * nb;
      } else {
        t.x = static_cast<const char *>(x) + b * S * C * e;
      }
      t.mean += b * G;
      t.rstd += b * G;
      if (t.dpart) t.dpart += b * 2 * C;
      (dt == 0 ? bwd_bf16 : dt == 1 ? bwd_fp16 : bwd_fp32)(part, gn_lds(p, true), t, st);
    });
  }
  if (!dgb) return;
  const long long rows = B * p.g.k;
  const unsigned nb = looped((2ll * C + 63) / 64).x;
  if (rows > 16 * kSplitRows) {
    const int split = (int)((rows + kSplitRows - 1) / kSplitRows), ns = (int)((rows + split - 1) / split);
    hipLaunchKernelGGL(gn_dparam_kernel, dim3(nb, ns), dim3(1024), 0, st, ws + w.dpart, ws + w.lvl, rows, 2 * C, split);
    hipLaunchKernelGGL(gn_dparam_kernel, dim3(nb), dim3(1024), 0, st, ws + w.lvl, dgb, (long long)ns, 2 * C, ns);
  } else {
    hipLaunchKernelGGL(gn_dparam_kernel, dim3(nb), dim3(1024), 0, st, ws + w.dpart, dgb, rows, 2 * C, (int)rows);
  }
}
