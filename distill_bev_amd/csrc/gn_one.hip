// Group norm + activation in ONE pass over the data (forward: x read once; backward: gy and x, or its checkpoint, read once) for batches that
// are large against the chip while an image is small against it.  The two launches of gn_act.hip read the data twice, and the backward
// evaluates the activation's derivative twice.
//
// A workgroup of 256 threads keeps a tile of one image in registers (R rows x 16 bytes a thread, 64 KB a workgroup, four workgroups a CU:
// 64 MB on the chip), reduces it to one pair of numbers per group, publishes them, waits for its image's totals, and finishes from the
// registers.  The image's last tiles collect, four groups a workgroup: all T pairs of a group in fp64 in a fixed order, and publish the totals.
//
// Measured at 48 x 256 x 64 x 176 (forward / backward, us; in brackets the two launches a direction of gn_act.hip):
//   fp32                 no activation 229 / 388 (300 / 481)   SiLU 228 / 451 (299 / 484)   GELU 236 / 471 (308 / 488)
//   fp32, int8 kept      no activation 241 / 301 (327 / 334)   SiLU 249 / 314 (328 / 342)   GELU 262 / 333 (331 / 347)
//   bf16 (forward only)  no activation 142 (166)   SiLU 145 (163)   GELU 160 (179); int8 kept 154 (187)   162 (190)   179 (201)
// i.e. the forward moves its floor of 2 n es (+ 1.03 n) bytes at 4.7 to 5.1 TB/s in fp32 where a copy reaches 5.3, the backward at 3.5 to 4.3;
// GELU in bf16 (3.5) and the backward are held by VALU work (some 30 instructions an element) that a workgroup's phases overlap with the
// transfers only in part.
//
// These tensors are as large as the memory-side cache or larger: they are read and written past it (nontemporal).  With an operator that
// writes x and one that reads y around the SiLU forward, us kept / past: fp32 138 MB 142 / 145, 277 MB 312 / 275, 553 MB 620 / 559; bf16 138
// MB 160 / 160, 277 MB 324 / 298; int8 backward 185 / 181, 382 / 362, 742 / 705.
//
// Every published pair is ONE 64-bit word, written and read with relaxed agent-scope atomics and empty (all ones) before: a word is its own
// flag, nothing else has to be ordered or visible, no fence writes an L2 back.  A NaN is published with the usual quiet pattern, never as
// all ones.
//
// Every wait is bounded: a workgroup that has polled `polls` times (about 10 ms) without its words -- other streams' kernels may keep the
// tiles that it waits for from starting -- notes its tile as not finished and ends; so the grid drains whatever else runs.  All
// workgroups publish before they wait, so behind this launch every pair is there: gn_one_*_rest, launched always, finishes the noted tiles
// from memory with the same sums in the same order (the same bits), and returns at once when there are none.
//
// Launches: fill (empty words), main, rest [, sums of the parameter gradients].
#include "gn_act.h"
#include "gn_one.h"

#include <atomic>
#include <type_traits>

namespace {

typedef unsigned long long ull;
constexpr ull GN_EMPTY = ~0ull;

struct GnOneBufs { ull *part, *fin; int *todo, *undone; float2* pc; double2* ps; };
struct GnOneArgs { GnArgs a; int T, polls; GnOneBufs b; };

__device__ __forceinline__ void gn_publish(ull* p, float x, float y) {
  const unsigned u = x == x ? __float_as_uint(x) : 0x7fc00000u, v = y == y ? __float_as_uint(y) : 0x7fc00000u;
  __hip_atomic_store(p, (static_cast<ull>(v) << 32) | u, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}
__device__ __forceinline__ ull gn_peek(const ull* p) { return __hip_atomic_load(p, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT); }

__global__ __launch_bounds__(256) void gn_one_fill(ull* __restrict__ words, long long nwords, int* __restrict__ ints, long long nints) {
  const long long i = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  if (i < nwords) words[i] = GN_EMPTY;
  if (i < nints) ints[i] = 0;
}

// An image is at most 512 tiles of 64 KB: addresses are a uniform image base + 32-bit offsets.  `nv`: rows of this thread inside the image.
struct GnOnePos { int n, t, rp, lane, col, nv; bool on; unsigned at; };
template <int V, int R>
__device__ __forceinline__ GnOnePos gn_one_pos(const GnOneArgs& o, int tile) {
  GnOnePos p;
  p.n = tile / o.T;
  p.t = tile - p.n * o.T;
  p.rp = threadIdx.x / o.a.t.CH;
  p.lane = threadIdx.x - p.rp * o.a.t.CH;
  p.col = p.lane;
  p.on = p.rp < o.a.t.RP && p.col < o.a.cv;
  const int r0 = p.t * (o.a.t.RP * R) + p.rp, left = static_cast<int>(o.a.S) - r0;
  p.nv = p.rp < o.a.t.RP && left > 0 ? min(R, (left + o.a.t.RP - 1) / o.a.t.RP) : 0;
  p.at = static_cast<unsigned>(r0) * o.a.C + p.col * V;       // element of the first row, in the image
  return p;
}
// The compiler would keep what it derived from these registers -- converted values, addresses -- alive from one phase to the next; behind this
// it derives them again
template <typename X>
__device__ __forceinline__ void gn_opaque(X& v) { asm volatile("" : "+v"(v)); }
template <typename T>
__device__ __forceinline__ T* gn_at(T* image, unsigned bytes) {
  return reinterpret_cast<T*>(reinterpret_cast<char*>(const_cast<typename std::remove_const<T>::type*>(image)) + bytes);
}
// groups of a thread's V channels: one division where groups are whole vectors
template <int V>
__device__ __forceinline__ void gn_groups(const GnArgs& a, const GnOnePos& p, int* g) {
  const int first = p.on ? p.col * V : 0;
  if (a.cpg % V == 0) {
    g[0] = first / a.cpg;
#pragma unroll
    for (int i = 1; i < V; ++i) g[i] = g[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) g[i] = (first + i) / a.cpg;
  }
}
template <typename T, int V> struct GnRaw {                   // one 16-byte vector as dwords
  typedef unsigned type __attribute__((ext_vector_type(4)));
  static __device__ __forceinline__ void get(type t, float* v) { A8Vec<T, V>::get(__builtin_bit_cast(typename A8Vec<T, V>::Raw, t), v); }
};

// per-thread column sums -> per channel in sh[0 .. CH V); one or two arrays (the second behind the first)
template <int V, int ARRAYS>
__device__ __forceinline__ void gn_one_fold(float* sh, const GnArgs& a, const GnOnePos& p, const float* s, const float* q) {
  const int w = a.t.CH * V;
  float* t = sh + ARRAYS * w;                                 // [ARRAYS][RP][CH V]
  __syncthreads();
  if (p.rp < a.t.RP) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      t[p.rp * w + p.lane * V + i] = s[i];
      if (ARRAYS == 2) t[(a.t.RP + p.rp) * w + p.lane * V + i] = q[i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < w; c += blockDim.x) {
#pragma unroll
    for (int k = 0; k < ARRAYS; ++k) {
      float sum = 0.f;
      for (int r = 0; r < a.t.RP; ++r) sum += t[(k * a.t.RP + r) * w + c];
      sh[k * w + c] = sum;
    }
  }
  __syncthreads();
}

// Groups [ga, gb) of one image: its T words per group added in fp64 into out[2 g], out[2 g + 1] (LDS).  A wave takes a group, its lanes the tiles
// (T <= 512: eight words a lane, all loads at once), a shuffle tree adds them: the same order whoever does it.
// POLL: words may still be empty, `polls` looks in all; returns (for the whole workgroup) whether all were there.
// STATS: (mean, M2) -> (mean, rstd): from sum n m and sum (M2 + n m^2), the cancellation costs (mean / spread)^2 of 2^-53; else (A, B) ->
// (A / D, B / D)
template <bool STATS, bool POLL, int R>
__device__ __forceinline__ bool gn_one_collect(float* out, const GnOneArgs& o, int n, int ga, int gb, float eps) {
  const GnArgs& a = o.a;
  const double D = static_cast<double>(a.S) * a.cpg;
  const int tile_rows = a.t.RP * R, last_rows = static_cast<int>(a.S) - (o.T - 1) * tile_rows;
  const int lane = threadIdx.x & 63, nwave = blockDim.x >> 6;
  int polls = o.polls;
  bool ok = true;
  for (int g = ga + static_cast<int>(threadIdx.x >> 6); g < gb; g += nwave) {
    const ull* words = o.b.part + (static_cast<size_t>(n) * a.G + g) * o.T;
    ull w[8];
    bool all;
    do {
      all = true;
#pragma unroll
      for (int j = 0; j < 8; ++j) w[j] = lane + 64 * j < o.T ? gn_peek(words + lane + 64 * j) : 0ull;
#pragma unroll
      for (int j = 0; j < 8; ++j) all = all && w[j] != GN_EMPTY;
      if (POLL && !all) __builtin_amdgcn_s_sleep(4);
    } while (POLL && !all && --polls > 0);
    ok = ok && all;
    double s0 = 0.0, s1 = 0.0;
#pragma unroll
    for (int j = 0; j < 8; ++j) {
      const int k = lane + 64 * j;
      const double x = __uint_as_float(static_cast<unsigned>(w[j])), y = __uint_as_float(static_cast<unsigned>(w[j] >> 32));
      if (k >= o.T) break;
      if (STATS) {
        const double cnt = static_cast<double>(k == o.T - 1 ? last_rows : tile_rows) * a.cpg;
        s0 += cnt * x;
        s1 += y + cnt * x * x;
      } else {
        s0 += x;
        s1 += y;
      }
    }
    s0 = gn_lane_sum(s0, 64) / D;
    s1 = gn_lane_sum(s1, 64) / D;
    if (STATS) {
      const double var = s1 - s0 * s0;
      s1 = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + static_cast<double>(eps));
    }
    if (lane == 0) {
      out[2 * g] = static_cast<float>(s0);
      out[2 * g + 1] = static_cast<float>(s1);
    }
  }
  return __syncthreads_and(ok) != 0;
}

// The image's last tiles collect: one workgroup per four groups (a group a wave), so that the totals are one look at the words away
__device__ __forceinline__ int gn_one_collectors(const GnOneArgs& o) { return min(o.T, (o.a.G + 3) / 4); }
__device__ __forceinline__ int gn_one_share(const GnOneArgs& o) { const int nc = gn_one_collectors(o); return (o.a.G + nc - 1) / nc; }

// the totals of this tile's image in out[]; false: not there in time
template <bool STATS, int R>
__device__ __forceinline__ bool gn_one_totals(float* out, const GnOneArgs& o, const GnOnePos& p, float eps, float* mean, float* rstd) {
  const GnArgs& a = o.a;
  ull* fin = o.b.fin + static_cast<size_t>(p.n) * a.G;
  bool ok = true;
  const int share = gn_one_share(o), ga = min(a.G, (o.T - 1 - p.t) * share), gb = min(a.G, ga + share);
  if (ga < gb) {                                              // (uniform)
    ok = gn_one_collect<STATS, true, R>(out, o, p.n, ga, gb, eps);
    if (ok)
      for (int g = ga + threadIdx.x; g < gb; g += blockDim.x) {
        gn_publish(fin + g, out[2 * g], out[2 * g + 1]);
        if (STATS && mean != nullptr) {
          mean[static_cast<size_t>(p.n) * a.G + g] = out[2 * g];
          rstd[static_cast<size_t>(p.n) * a.G + g] = out[2 * g + 1];
        }
      }
  }
  int polls = o.polls;
  for (int g = threadIdx.x; g < a.G && ok; g += blockDim.x) {
    if (g >= ga && g < gb) continue;
    ull w = gn_peek(fin + g);
    while (w == GN_EMPTY && --polls > 0) {
      __builtin_amdgcn_s_sleep(4);
      w = gn_peek(fin + g);
    }
    ok = w != GN_EMPTY;
    out[2 * g] = __uint_as_float(static_cast<unsigned>(w));
    out[2 * g + 1] = __uint_as_float(static_cast<unsigned>(w >> 32));
  }
  ok = __syncthreads_and(ok) != 0;
  if (!ok && threadIdx.x == 0) {
    o.b.todo[static_cast<size_t>(p.n) * o.T + p.t] = 1;
    atomicAdd(o.b.undone, 1);
  }
  return ok;
}

template <int V>
__device__ __forceinline__ float* gn_one_out(float* sh, const GnArgs& a) {      // behind the fold's scratch
  return sh + 2 * a.t.CH * V * (1 + a.t.RP);
}

// y (and the checkpoint) of one tile from the values in `raw`
template <typename T, int V, int R, int FMT, int ACT, bool NT>
__device__ __forceinline__ void gn_one_write(const typename GnRaw<T, V>::type* raw, const float* out, const GnOneArgs& o, GnOnePos p,
                                             const float* gamma, const float* beta, T* y, uint8_t* codes, uint8_t* scales) {
  constexpr int LB = 32 / V;
  const GnArgs& a = o.a;
  float sc[V], bt[V];
  int gr[V];
  gn_groups<V>(a, p, gr);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = p.on ? p.col * V + i : i;
    sc[i] = out[2 * gr[i] + 1] * (gamma != nullptr ? gamma[c] : 1.f);
    bt[i] = fmaf(-out[2 * gr[i]], sc[i], beta != nullptr ? beta[c] : 0.f);
  }
  const size_t image = static_cast<size_t>(p.n) * a.S;
  T* yi = y + image * a.C;
  uint8_t* ci = FMT != DBEV_ACT8_NONE ? codes + image * a.C : nullptr;
  uint8_t* si = FMT != DBEV_ACT8_NONE ? scales + image * a.nb : nullptr;
  unsigned at = p.at, sat = static_cast<unsigned>(p.t * (a.t.RP * R) + p.rp) * a.nb + p.col / LB;
  gn_opaque(at);
#pragma unroll
  for (int u = 0; u < R; ++u) {
    if (u < p.nv) {                                           // all lanes of a block are on the same pixel
      float v[V];
      GnRaw<T, V>::get(raw[u], v);
      if (FMT != DBEV_ACT8_NONE) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        const unsigned b = a8_scale_byte<FMT>(a8_block_max<V>(m));
        if (p.on) {
          *reinterpret_cast<typename A8Bytes<V>::type*>(gn_at(ci, at)) = a8_encode<FMT, V>(v, b);
          if (p.col % LB == 0) *gn_at(si, sat) = static_cast<uint8_t>(b);
        }
      }
      if (p.on) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = a8_act<ACT>(fmaf(v[i], sc[i], bt[i]));
        A8Vec<T, V>::template store<NT>(gn_at(yi, at * static_cast<unsigned>(sizeof(T))), v);
      }
    }
    at += a.t.RP * a.C;
    sat += a.t.RP * a.nb;
  }
}

template <typename T, int V, int R, bool NT>
__device__ __forceinline__ void gn_one_load(typename GnRaw<T, V>::type* raw, const T* x, const GnArgs& a, const GnOnePos& p) {
  typedef typename GnRaw<T, V>::type dw;
  const T* xi = x + static_cast<size_t>(p.n) * a.S * a.C;
  unsigned at = p.at * static_cast<unsigned>(sizeof(T));
#pragma unroll
  for (int u = 0; u < R; ++u) {
    if (p.on && u < p.nv) raw[u] = NT ? __builtin_nontemporal_load(reinterpret_cast<const dw*>(gn_at(xi, at))) : *reinterpret_cast<const dw*>(gn_at(xi, at));
    else raw[u] = dw{0, 0, 0, 0};
    at += a.t.RP * a.C * static_cast<unsigned>(sizeof(T));
  }
}

// the tile's mean per group, then the squares about it, both from the registers: done(g, mean, M2) by one thread a group, out[2 g] = mean.  x0: the
// tile's first pixel.  Its value in a group's first channel is taken off every thread's sum, so that the sums over threads are of numbers of the
// spread's size whatever offset the data have: an offset of 1000 spreads costs the mean its last rounding (and every thread's sum of 16
// rows, which averages out), not those of a sum over all
template <typename T, int V, int R, typename F>
__device__ __forceinline__ void gn_one_stats(typename GnRaw<T, V>::type* raw, const T* x0, float* sh, float* out, const GnArgs& a, const GnOnePos& p,
                                             int rows, F done) {
  const int lanes = gn_lanes(a.G), sub = threadIdx.x % lanes;
  float s[V], ref[V];
  int gr[V];
  gn_groups<V>(a, p, gr);
  if (a.cpg % V == 0) {
    ref[0] = static_cast<float>(x0[gr[0] * a.cpg]);
#pragma unroll
    for (int i = 1; i < V; ++i) ref[i] = ref[0];
  } else {
#pragma unroll
    for (int i = 0; i < V; ++i) ref[i] = static_cast<float>(x0[gr[i] * a.cpg]);
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = 0.f;
#pragma unroll
  for (int u = 0; u < R; u += 2) {                            // (rows past the end are zeros)
    float v[V], v2[V];
    GnRaw<T, V>::get(raw[u], v);
    GnRaw<T, V>::get(raw[u + 1], v2);
#pragma unroll
    for (int i = 0; i < V; ++i) s[i] += v[i] + v2[i];
  }
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = fmaf(-static_cast<float>(p.nv), ref[i], s[i]);
  if (p.on && p.rp == 0) {                                    // for the group's mean below, without another load
#pragma unroll
    for (int i = 0; i < V; ++i)
      if (p.col * V + i == gr[i] * a.cpg) out[2 * gr[i] + 1] = ref[i];
  }
  gn_one_fold<V, 1>(sh, a, p, s, s);
  for (int g = threadIdx.x / lanes; g < a.G; g += blockDim.x / lanes) {
    float m = 0.f;
    for (int c = sub; c < a.cpg; c += lanes) m += sh[g * a.cpg + c];
    m = gn_lane_sum(m, lanes);
    if (sub == 0) out[2 * g] = out[2 * g + 1] + m / (static_cast<float>(rows) * static_cast<float>(a.cpg));
  }
  __syncthreads();
  float mu[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    mu[i] = out[2 * gr[i]];
    s[i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < R; ++u) {
    gn_opaque(raw[u]);
    if (u < p.nv) {
      float v[V];
      GnRaw<T, V>::get(raw[u], v);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float d = v[i] - mu[i];
        s[i] = fmaf(d, d, s[i]);
      }
    }
  }
  gn_one_fold<V, 1>(sh, a, p, s, s);
  for (int g = threadIdx.x / lanes; g < a.G; g += blockDim.x / lanes) {
    float m2 = 0.f;
    for (int c = sub; c < a.cpg; c += lanes) m2 += sh[g * a.cpg + c];
    m2 = gn_lane_sum(m2, lanes);
    if (sub == 0) done(g, out[2 * g], m2);
  }
  __syncthreads();                                            // out[] is read above and written below
}

template <typename T, int V, int R, int FMT, int ACT>
__global__ __launch_bounds__(256, 4) void gn_one_fwd(const T* __restrict__ x, GnOneArgs o, const float* __restrict__ gamma, const float* __restrict__ beta,
                                                     float eps, T* __restrict__ y, float* __restrict__ mean, float* __restrict__ rstd,
                                                     uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  extern __shared__ float sh[];
  const GnArgs& a = o.a;
  const GnOnePos p = gn_one_pos<V, R>(o, blockIdx.x);
  float* out = gn_one_out<V>(sh, a);
  typename GnRaw<T, V>::type raw[R];
  gn_one_load<T, V, R, true>(raw, x, a, p);
  const int r0 = p.t * (a.t.RP * R);
  gn_one_stats<T, V, R>(raw, x + (static_cast<size_t>(p.n) * a.S + r0) * a.C, sh, out, a, p, min(a.t.RP * R, static_cast<int>(a.S) - r0),
                        [&](int g, float m, float m2) { gn_publish(o.b.part + (static_cast<size_t>(p.n) * a.G + g) * o.T + p.t, m, m2); });
  if (!gn_one_totals<true, R>(out, o, p, eps, mean, rstd)) return;
#pragma unroll
  for (int u = 0; u < R; ++u) gn_opaque(raw[u]);
  gn_one_write<T, V, R, FMT, ACT, true>(raw, out, o, p, gamma, beta, y, codes, scales);
}

// Small images, forward: one workgroup holds all pixels of W channels of an image (whole groups, a multiple of 32 or all) in registers.  One
// launch, nothing exchanged; bound by the latency of load -> two LDS folds -> store.  The helpers see the image's W channels through
// shifted pointers.
template <typename T, int V, int R, int FMT, int ACT>
__global__ __launch_bounds__(256, 4) void gn_small_fwd(const T* __restrict__ x, GnOneArgs o, int W, int nblk, const float* __restrict__ gamma,
                                                       const float* __restrict__ beta, float eps, T* __restrict__ y, float* __restrict__ mean,
                                                       float* __restrict__ rstd, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  extern __shared__ float sh[];
  const int n = blockIdx.x / nblk, c0 = (blockIdx.x - n * nblk) * W, w = min(W, o.a.C - c0);
  const size_t first = static_cast<size_t>(n) * o.a.G + c0 / o.a.cpg;
  o.a.cv = w / V;
  o.a.G = w / o.a.cpg;
  const GnArgs& a = o.a;
  const GnOnePos p = gn_one_pos<V, R>(o, n);
  float* out = gn_one_out<V>(sh, a);
  typename GnRaw<T, V>::type raw[R];
  gn_one_load<T, V, R, false>(raw, x + c0, a, p);
  const double D = static_cast<double>(a.S) * a.cpg;
  gn_one_stats<T, V, R>(raw, x + c0 + static_cast<size_t>(n) * a.S * a.C, sh, out, a, p, static_cast<int>(a.S), [&](int g, float m, float m2) {
    const float r = static_cast<float>(1.0 / sqrt(m2 / D + static_cast<double>(eps)));
    out[2 * g + 1] = r;
    if (mean != nullptr) {
      mean[first + g] = m;
      rstd[first + g] = r;
    }
  });
#pragma unroll
  for (int u = 0; u < R; ++u) gn_opaque(raw[u]);
  gn_one_write<T, V, R, FMT, ACT, false>(raw, out, o, p, gamma == nullptr ? nullptr : gamma + c0, beta == nullptr ? nullptr : beta + c0, y + c0,
                                         FMT == DBEV_ACT8_NONE ? nullptr : codes + c0, FMT == DBEV_ACT8_NONE ? nullptr : scales + c0 / 32);
}

// the tiles that gave up waiting, from memory
template <typename T, int V, int R, int FMT, int ACT>
__global__ __launch_bounds__(256, 2) void gn_one_fwd_rest(const T* __restrict__ x, GnOneArgs o, int tiles, const float* __restrict__ gamma,
                                                          const float* __restrict__ beta, float eps, T* __restrict__ y, float* __restrict__ mean,
                                                          float* __restrict__ rstd, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  extern __shared__ float sh[];
  if (*o.b.undone == 0) return;
  const GnArgs& a = o.a;
  float* out = gn_one_out<V>(sh, a);
  for (int tile = blockIdx.x; tile < tiles; tile += gridDim.x) {
    if (o.b.todo[tile] == 0) continue;                        // (uniform)
    const GnOnePos p = gn_one_pos<V, R>(o, tile);
    gn_one_collect<true, false, R>(out, o, p.n, 0, a.G, eps);
    if (mean != nullptr)                                      // (a collector that gave up has not written its groups; others write the same)
      for (int g = threadIdx.x; g < a.G; g += blockDim.x) {
        mean[static_cast<size_t>(p.n) * a.G + g] = out[2 * g];
        rstd[static_cast<size_t>(p.n) * a.G + g] = out[2 * g + 1];
      }
    typename GnRaw<T, V>::type raw[R];
    gn_one_load<T, V, R, true>(raw, x, a, p);
    gn_one_write<T, V, R, FMT, ACT, true>(raw, out, o, p, gamma, beta, y, codes, scales);
    __syncthreads();
  }
}

// the other operand of the backward, as loaded: 16 bytes of x, or V codes (the scale byte is read again where it is needed)
template <typename T, int V, int FMT> struct GnKept {
  typedef typename GnRaw<T, V>::type type;
  static __device__ __forceinline__ type load(const T* xi, const uint8_t*, unsigned at) {
    return *reinterpret_cast<const type*>(gn_at(xi, at * static_cast<unsigned>(sizeof(T))));
  }
  static __device__ __forceinline__ void get(const type& t, const uint8_t*, unsigned, float* v) { GnRaw<T, V>::get(t, v); }
};
template <typename T, int V> struct GnKept8 {
  typedef typename A8Bytes<V>::type type;
  static __device__ __forceinline__ type load(const T*, const uint8_t* ci, unsigned at) { return *reinterpret_cast<const type*>(gn_at(ci, at)); }
};
template <typename T, int V> struct GnKept<T, V, DBEV_ACT8_INT8> : GnKept8<T, V> {
  static __device__ __forceinline__ void get(const typename A8Bytes<V>::type& t, const uint8_t* si, unsigned sat, float* v) {
    a8_decode<DBEV_ACT8_INT8, V>(t, a8_scale(*gn_at(si, sat)), v);
  }
};
template <typename T, int V> struct GnKept<T, V, DBEV_ACT8_E4M3> : GnKept8<T, V> {
  static __device__ __forceinline__ void get(const typename A8Bytes<V>::type& t, const uint8_t* si, unsigned sat, float* v) {
    a8_decode<DBEV_ACT8_E4M3, V>(t, a8_scale(*gn_at(si, sat)), v);
  }
};

struct GnImage { size_t row; unsigned at, sat, step, sstep; };          // image's first row; this thread's first element and scale byte, distances
template <int V, int R>
__device__ __forceinline__ GnImage gn_image(const GnArgs& a, const GnOnePos& p) {
  GnImage m;
  m.row = static_cast<size_t>(p.n) * a.S;
  m.at = p.at;
  m.sat = static_cast<unsigned>(p.t * (a.t.RP * R) + p.rp) * a.nb + p.col / (32 / V);
  gn_opaque(m.at);
  gn_opaque(m.sat);
  m.step = a.t.RP * a.C;
  m.sstep = a.t.RP * a.nb;
  return m;
}

// backward: g = gy act'(z) of one tile into registers, its sums per column
template <typename T, int V, int R, int FMT, int ACT>
__device__ __forceinline__ void gn_one_grad(float (*g)[V], typename GnKept<T, V, FMT>::type* kept, float* s, float* q, const T* gy, const T* x,
                                            const uint8_t* codes, const uint8_t* scales, const GnOneArgs& o, const GnOnePos& p, const GnCoef& k) {
  typedef typename GnRaw<T, V>::type dw;
  const GnArgs& a = o.a;
  const GnImage m = gn_image<V, R>(a, p);
  const T* gi = gy + m.row * a.C;
  const T* xi = FMT == DBEV_ACT8_NONE ? x + m.row * a.C : nullptr;
  const uint8_t* ci = FMT == DBEV_ACT8_NONE ? nullptr : codes + m.row * a.C;
  const uint8_t* si = FMT == DBEV_ACT8_NONE ? nullptr : scales + m.row * a.nb;
  dw raw[R];
#pragma unroll
  for (int u = 0; u < R; ++u)
    if (p.on && u < p.nv) {
      raw[u] = __builtin_nontemporal_load(reinterpret_cast<const dw*>(gn_at(gi, (m.at + u * m.step) * static_cast<unsigned>(sizeof(T)))));
      kept[u] = GnKept<T, V, FMT>::load(xi, ci, m.at + u * m.step);
    }
  float mu[V], rs[V], sc[V], bt[V];
  int gr[V];
  gn_groups<V>(a, p, gr);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = p.on ? p.col * V + i : i;
    mu[i] = k.mean[static_cast<size_t>(p.n) * a.G + gr[i]];
    rs[i] = k.rstd[static_cast<size_t>(p.n) * a.G + gr[i]];
    sc[i] = rs[i] * (k.gamma != nullptr ? k.gamma[c] : 1.f);
    bt[i] = k.beta != nullptr ? k.beta[c] : 0.f;
    s[i] = q[i] = 0.f;
  }
#pragma unroll
  for (int u = 0; u < R; ++u)
    if (p.on && u < p.nv) {
      float v[V], d[V];
      GnKept<T, V, FMT>::get(kept[u], si, m.sat + u * m.sstep, v);
      GnRaw<T, V>::get(raw[u], d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dev = v[i] - mu[i];
        g[u][i] = a8_act_grad<ACT>(d[i], fmaf(dev, sc[i], bt[i]));
        s[i] += g[u][i];
        q[i] = fmaf(g[u][i], dev, q[i]);
      }
    }
#pragma unroll
  for (int i = 0; i < V; ++i) q[i] *= rs[i];
}

template <typename T, int V, int R, int FMT>
__device__ __forceinline__ void gn_one_dx(const float (*g)[V], typename GnKept<T, V, FMT>::type* kept, const float* out, const uint8_t* scales,
                                          const GnOneArgs& o, const GnOnePos& p, const GnCoef& k, T* dx) {
  const GnArgs& a = o.a;
  if (!p.on) return;
  const GnImage m = gn_image<V, R>(a, p);
  T* di = dx + m.row * a.C;
  const uint8_t* si = FMT == DBEV_ACT8_NONE ? nullptr : scales + m.row * a.nb;
  float mu[V], sc[V], A[V], B[V];                             // dx = sc g - (rstd A) - (x - mean) (rstd^2 B), sc = rstd gamma
  int gr[V];
  gn_groups<V>(a, p, gr);
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = p.col * V + i;
    const float rs = k.rstd[static_cast<size_t>(p.n) * a.G + gr[i]];
    mu[i] = k.mean[static_cast<size_t>(p.n) * a.G + gr[i]];
    sc[i] = rs * (k.gamma != nullptr ? k.gamma[c] : 1.f);
    A[i] = rs * out[2 * gr[i]];
    B[i] = rs * rs * out[2 * gr[i] + 1];
  }
#pragma unroll
  for (int u = 0; u < R; ++u) {
    gn_opaque(kept[u]);
    if (u < p.nv) {
      float v[V];
      GnKept<T, V, FMT>::get(kept[u], si, m.sat + u * m.sstep, v);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = fmaf(sc[i], g[u][i], -fmaf(v[i] - mu[i], B[i], A[i]));
      A8Vec<T, V>::template store<true>(gn_at(di, (m.at + u * m.step) * static_cast<unsigned>(sizeof(T))), v);
    }
  }
}

template <typename T, int V, int R, int FMT, int ACT>
__global__ __launch_bounds__(256, 3) void gn_one_bwd(const T* __restrict__ gy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, GnOneArgs o, GnCoef k, T* __restrict__ dx) {
  extern __shared__ float sh[];
  const GnArgs& a = o.a;
  const GnOnePos p = gn_one_pos<V, R>(o, blockIdx.x);
  float* out = gn_one_out<V>(sh, a);
  float g[R][V], s[V], q[V];
  typename GnKept<T, V, FMT>::type kept[R];
  gn_one_grad<T, V, R, FMT, ACT>(g, kept, s, q, gy, x, codes, scales, o, p, k);
  gn_one_fold<V, 2>(sh, a, p, s, q);
  const int w = a.t.CH * V, lanes = gn_lanes(a.G), sub = threadIdx.x % lanes;
  for (int gr = threadIdx.x / lanes; gr < a.G; gr += blockDim.x / lanes) {
    float A = 0.f, B = 0.f;
    for (int c = gr * a.cpg + sub; c < (gr + 1) * a.cpg; c += lanes) {
      const float gc = k.gamma != nullptr ? k.gamma[c] : 1.f;
      A = fmaf(gc, sh[c], A);
      B = fmaf(gc, sh[w + c], B);
    }
    A = gn_lane_sum(A, lanes);
    B = gn_lane_sum(B, lanes);
    if (sub == 0) gn_publish(o.b.part + (static_cast<size_t>(p.n) * a.G + gr) * o.T + p.t, A, B);
  }
  if (o.b.pc != nullptr) {
    float2* row = o.b.pc + (static_cast<size_t>(p.n) * o.T + p.t) * a.C;
    for (int c = threadIdx.x; c < a.C; c += blockDim.x) row[c] = make_float2(sh[c], sh[w + c]);
  }
  __syncthreads();
  if (!gn_one_totals<false, R>(out, o, p, 0.f, nullptr, nullptr)) return;
  gn_one_dx<T, V, R, FMT>(g, kept, out, scales, o, p, k, dx);
}

constexpr int GN_PS = 16;                                     // slices of the tile rows for the parameter gradients: C / 8 * 16 workgroups

// workgroups [0, npar): one slice's sums of 8 channels; the others: tiles that gave up waiting
template <typename T, int V, int R, int FMT, int ACT>
__global__ __launch_bounds__(256, 2) void gn_one_bwd_rest(const T* __restrict__ gy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                          const uint8_t* __restrict__ scales, GnOneArgs o, int tiles, int npar, GnCoef k,
                                                          T* __restrict__ dx) {
  extern __shared__ float sh[];
  const GnArgs& a = o.a;
  if (static_cast<int>(blockIdx.x) < npar) {
    double* sd = reinterpret_cast<double*>(sh);
    const int slice = blockIdx.x % GN_PS, c = blockIdx.x / GN_PS * 8 + threadIdx.x % 8, ph = threadIdx.x / 8, np = blockDim.x / 8;
    const long long per = (tiles + GN_PS - 1) / GN_PS, r0 = slice * per, r1 = min(static_cast<long long>(tiles), r0 + per);
    double s = 0.0, q = 0.0;
    if (c < a.C) {
#pragma unroll 8
      for (long long r = r0 + ph; r < r1; r += np) {
        const float2 e = o.b.pc[r * a.C + c];
        s += e.x;
        q += e.y;
      }
    }
    sd[2 * threadIdx.x] = s;
    sd[2 * threadIdx.x + 1] = q;
    __syncthreads();
    if (ph == 0 && c < a.C) {
      for (int i = 1; i < np; ++i) {
        s += sd[2 * (threadIdx.x + 8 * i)];
        q += sd[2 * (threadIdx.x + 8 * i) + 1];
      }
      o.b.ps[static_cast<size_t>(slice) * a.C + c] = make_double2(s, q);
    }
    return;
  }
  if (*o.b.undone == 0) return;
  float* out = gn_one_out<V>(sh, a);
  for (int tile = blockIdx.x - npar; tile < tiles; tile += gridDim.x - npar) {
    if (o.b.todo[tile] == 0) continue;
    const GnOnePos p = gn_one_pos<V, R>(o, tile);
    gn_one_collect<false, false, R>(out, o, p.n, 0, a.G, 0.f);
    float g[R][V], s[V], q[V];
    typename GnKept<T, V, FMT>::type kept[R];
    gn_one_grad<T, V, R, FMT, ACT>(g, kept, s, q, gy, x, codes, scales, o, p, k);
    gn_one_dx<T, V, R, FMT>(g, kept, out, scales, o, p, k, dx);
    __syncthreads();
  }
}

__global__ __launch_bounds__(64) void gn_one_params(const double2* __restrict__ ps, int C, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int c = blockIdx.x * 64 + threadIdx.x;
  if (c >= C) return;
  double s = 0.0, q = 0.0;
#pragma unroll
  for (int i = 0; i < GN_PS; ++i) {
    s += ps[static_cast<size_t>(i) * C + c].x;
    q += ps[static_cast<size_t>(i) * C + c].y;
  }
  if (dbeta != nullptr) dbeta[c] = static_cast<float>(s);
  if (dgamma != nullptr) dgamma[c] = static_cast<float>(q);
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
std::atomic<int> g_polls{10000};

// Rows per thread.  Forward 16: 64 registers of data (with 8 or 12 the waits weigh more: 870 and 723 us against 720, 48 x 256 x 64 x 176 fp32
// forward + backward).  Backward, fp32 gradients and the other operand: 12 beside codes, 8 beside x itself.
constexpr int GN_RF = 16;
constexpr int gn_rb(int fmt) { return fmt == DBEV_ACT8_NONE ? 8 : 12; }

// CUs of the current device (a partition of the chip has fewer), 0 without one
int gn_one_cus() {
  static std::atomic<int> known[16];
  int dev = 0, n = 0;
  if (hipGetDevice(&dev) != hipSuccess || dev < 0) return 0;
  if (dev < 16 && (n = known[dev].load(std::memory_order_relaxed)) != 0) return n;
  if (hipDeviceGetAttribute(&n, hipDeviceAttributeMultiprocessorCount, dev) != hipSuccess) return 0;
  if (dev < 16) known[dev].store(n, std::memory_order_relaxed);
  return n;
}

// One pass where it is the faster way: rows wide enough to fill a workgroup, an image of 2 to 512 tiles and at most half of what the device
// holds (four a CU), so that another image's transfer covers one's wait, and 2048 tiles or more in all: below, the two extra launches eat
// the gain (8 x 128 x 128 x 128 fp32, 1024 tiles: forward 41 us against 50 of GPU time but two launches more for the host, backward 63
// against 56).
bool gn_one_plan(int dtype, int N, long long S, int C, int vec, int R, GnArgs* a, int* T) {
  const int wide = dtype == DBEV_DT_F32 ? 4 : 8;
  if (vec != wide) return false;
  a->t = a8_tile(C, wide);
  if (a->t.ncol != 1 || a->t.CH * a->t.RP < 192) return false;
  const long long rows = static_cast<long long>(a->t.RP) * R, tiles = (S + rows - 1) / rows;
  if (tiles < 2 || tiles > 512 || tiles * N < 2048 || tiles * N > (1 << 22) || tiles > 2LL * gn_one_cus()) return false;
  *T = static_cast<int>(tiles);
  return true;
}

GnArgs gn_one_args(GnArgs a, long long S, int C, int G, int vec) {
  a.S = S;
  a.C = C;
  a.cv = C / vec;
  a.G = G;
  a.cpg = C / G;
  a.nb = (C + 31) / 32;
  a.nchunk = a.tiles_each = a.extra = a.last = a.lack = 0;
  return a;
}

size_t gn_one_layout(int N, int T, int C, int G, bool params, char* base, GnOneBufs* b) {
  size_t at = 0;
  auto take = [&](size_t bytes) {
    char* p = base + at;
    at += (bytes + 15) / 16 * 16;
    return p;
  };
  GnOneBufs l;
  l.part = reinterpret_cast<ull*>(take(static_cast<size_t>(N) * T * G * 8));
  l.fin = reinterpret_cast<ull*>(take(static_cast<size_t>(N) * G * 8));
  l.todo = reinterpret_cast<int*>(take((static_cast<size_t>(N) * T + 1) * 4));
  l.undone = l.todo + static_cast<size_t>(N) * T;
  l.pc = params ? reinterpret_cast<float2*>(take(static_cast<size_t>(N) * T * C * 8)) : nullptr;
  l.ps = params ? reinterpret_cast<double2*>(take(static_cast<size_t>(GN_PS) * C * 16)) : nullptr;
  if (b != nullptr) *b = l;
  return at;
}

template <int V>
size_t gn_one_lds(const GnArgs& a) {
  return (static_cast<size_t>(2) * a.t.CH * V * (1 + a.t.RP) + 2 * static_cast<size_t>(a.G)) * sizeof(float);
}

void gn_one_clear(const GnOneArgs& o, int N, hipStream_t st) {
  // part and fin are neighbours (sizes padded to 16 bytes): cleared as one range
  const long long words = (reinterpret_cast<char*>(o.b.fin) - reinterpret_cast<char*>(o.b.part)) / 8 + static_cast<long long>(N) * o.a.G;
  const long long ints = static_cast<long long>(N) * o.T + 1, n = words > ints ? words : ints;
  hipLaunchKernelGGL(gn_one_fill, dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, o.b.part, words, o.b.todo, ints);
}

}  // namespace

extern "C" int dbev_gn_act_poll_limit(int polls) {
  const int old = g_polls.load();
  if (polls >= 0) g_polls.store(polls);
  return old;
}

size_t gn_one_bytes(int N, long long S, int C, int G) {
  size_t m = 0;
  for (int dtype : {DBEV_DT_F32, DBEV_DT_BF16})
    for (int R : {gn_rb(DBEV_ACT8_NONE), gn_rb(DBEV_ACT8_INT8), GN_RF}) {
      GnArgs a;
      int T;
      const int vec = dtype == DBEV_DT_F32 ? 4 : 8;
      if (C % vec == 0 && gn_one_plan(dtype, N, S, C, vec, R, &a, &T)) {
        const size_t b = gn_one_layout(N, T, C, G, true, nullptr, nullptr);
        m = b > m ? b : m;
      }
    }
  return m;
}

#define GN_ONE_TYPES(dtype_, ...)                                            \
  switch (dtype_) {                                                          \
    case DBEV_DT_F32: { typedef float T; constexpr int V = 4; __VA_ARGS__; break; }     \
    case DBEV_DT_BF16: { typedef a8_bf16 T; constexpr int V = 8; __VA_ARGS__; break; }  \
    default: { typedef a8_f16 T; constexpr int V = 8; __VA_ARGS__; break; }             \
  }

// Small images: W channels (whole groups, whole blocks of 32, or all of them), at most GN_RF rows a thread (fp32, 32 channels: 512 pixels); wider
// while every thread still has a row of its own, and, with several rows a thread, while two workgroups a CU remain (5000 x 256 x 4 x 4, fp32 /
// bf16: 109 / 112 us with 64 channels a workgroup, 37 / 62 with all; 500 x 256 x 8 x 8 27 / 43 -> 14 / 17).  Against the two launches, without an
// activation, us a call: fp32 6 x 256 x 8 x 22 13 (16), 48 x 512 x 22 x 22 18 (34), 200 x 256 x 16 x 32 35 (60), 1000 x 256 x 4 x 4 13 (17), 5000 x 256 x 4 x 4
// 38 (58), 40000 images of one pixel 227 (287); bf16 13 (16), 19 (27), 22 (48), 15 (22), 60 (84), 424 (481)
bool gn_small_plan(int dtype, int N, long long S, int C, int G, int vec, GnArgs* a, int* W) {
  const int wide = dtype == DBEV_DT_F32 ? 4 : 8, cpg = C / G;
  if (vec != wide || S > 256 * GN_RF) return false;
  int unit = cpg;
  while (unit % 32 != 0 && unit < C) unit += cpg;
  if (unit > C) unit = C;
  for (int w = unit;; w = 2 * w < C ? 2 * w : C) {
    const A8Tile t = a8_tile(w, wide);
    const bool many = static_cast<long long>(N) * ((C + w - 1) / w) >= 512;
    if (t.ncol != 1 || S > static_cast<long long>(t.RP) * (w == unit || many ? GN_RF : 1)) break;
    a->t = t;
    *W = w;
    if (w == C) return true;
  }
  return a8_tile(unit, wide).ncol == 1 && S <= static_cast<long long>(a8_tile(unit, wide).RP) * GN_RF;
}

static int gn_one_vec(int dtype, int C) {
  const int wide = dtype == DBEV_DT_F32 ? 4 : 8;
  return C % wide == 0 ? wide : 0;
}
bool gn_small_takes(int dtype, int N, long long S, int C, int G) {
  GnArgs a;
  int W;
  return gn_small_plan(dtype, N, S, C, G, gn_one_vec(dtype, C), &a, &W) && static_cast<long long>(N) * ((C + W - 1) / W) * a.t.threads < (1LL << 32);
}
bool gn_one_takes(int dtype, int N, long long S, int C, int fmt, bool backward) {
  GnArgs a;
  int T;
  return !(backward && dtype != DBEV_DT_F32) && gn_one_plan(dtype, N, S, C, gn_one_vec(dtype, C), backward ? gn_rb(fmt) : GN_RF, &a, &T);
}

bool gn_small_forward(const void* x, int dtype, int vec, int N, long long S, int C, int G, const float* gamma, const float* beta, float eps, int act,
                      void* y, float* mean, float* rstd, int fmt, uint8_t* codes, uint8_t* scales, hipStream_t st) {
  GnOneArgs o;
  int W;
  if (!gn_small_plan(dtype, N, S, C, G, vec, &o.a, &W)) return false;
  const int nblk = (C + W - 1) / W;
  if (static_cast<long long>(N) * nblk * o.a.t.threads >= (1LL << 32)) return false;
  o.a = gn_one_args(o.a, S, C, G, vec);
  o.T = 1;
  o.polls = 0;
  o.b = GnOneBufs{};
  GnArgs local = o.a;
  local.G = W / o.a.cpg;
  GN_ONE_TYPES(dtype, A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
    hipLaunchKernelGGL((gn_small_fwd<T, V, GN_RF, FMT, ACT>), dim3(static_cast<unsigned>(N) * nblk), dim3(o.a.t.threads), gn_one_lds<V>(local), st,
                       static_cast<const T*>(x), o, W, nblk, gamma, beta, eps, static_cast<T*>(y), mean, rstd, codes, scales);
  })));
  return true;
}

bool gn_one_forward(const void* x, int dtype, int vec, int N, long long S, int C, int G, const float* gamma, const float* beta, float eps, int act, void* y,
                    float* mean, float* rstd, int fmt, uint8_t* codes, uint8_t* scales, void* ws, hipStream_t st) {
  GnOneArgs o;
  if (!gn_one_plan(dtype, N, S, C, vec, GN_RF, &o.a, &o.T)) return false;
  o.a = gn_one_args(o.a, S, C, G, vec);
  o.polls = g_polls.load();
  gn_one_layout(N, o.T, C, G, false, static_cast<char*>(ws), &o.b);
  const int tiles = N * o.T;
  gn_one_clear(o, N, st);
  GN_ONE_TYPES(dtype, A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
    constexpr int R = GN_RF;
    const size_t lds = gn_one_lds<V>(o.a);
    hipLaunchKernelGGL((gn_one_fwd<T, V, R, FMT, ACT>), dim3(tiles), dim3(o.a.t.threads), lds, st, static_cast<const T*>(x), o, gamma, beta, eps,
                       static_cast<T*>(y), mean, rstd, codes, scales);
    hipLaunchKernelGGL((gn_one_fwd_rest<T, V, R, FMT, ACT>), dim3(512), dim3(o.a.t.threads), lds, st, static_cast<const T*>(x), o, tiles, gamma, beta,
                       eps, static_cast<T*>(y), mean, rstd, codes, scales);
  })));
  return true;
}

// fp32 only: the 16-bit types would hold their gradients in twice the registers that they were read in, and the two launches are faster
// (48 x 256 x 64 x 176 bf16, SiLU: 365 us against 296; int8 checkpoint 340 against 251; the two launches with nontemporal accesses: 260 and 228)
bool gn_one_backward(const void* gy, int dtype, int vec, const void* x, int fmt, const uint8_t* codes, const uint8_t* scales, int N, long long S, int C,
                     int G, const float* gamma, const float* beta, const float* mean, const float* rstd, int act, void* dx, float* dgamma, float* dbeta,
                     void* ws, hipStream_t st) {
  GnOneArgs o;
  if (dtype != DBEV_DT_F32 || !gn_one_plan(dtype, N, S, C, vec, gn_rb(fmt), &o.a, &o.T)) return false;
  o.a = gn_one_args(o.a, S, C, G, vec);
  o.polls = g_polls.load();
  const bool params = dgamma != nullptr || dbeta != nullptr;
  gn_one_layout(N, o.T, C, G, params, static_cast<char*>(ws), &o.b);
  const int tiles = N * o.T, npar = params ? (C + 7) / 8 * GN_PS : 0;
  const GnCoef k = {gamma, beta, mean, rstd};
  const size_t lds = gn_one_lds<4>(o.a);
  const float *gyf = static_cast<const float*>(gy), *xf = static_cast<const float*>(x);
  float* dxf = static_cast<float*>(dx);
  gn_one_clear(o, N, st);
  A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
    constexpr int R = gn_rb(FMT);
    hipLaunchKernelGGL((gn_one_bwd<float, 4, R, FMT, ACT>), dim3(tiles), dim3(o.a.t.threads), lds, st, gyf, xf, codes, scales, o, k, dxf);
    hipLaunchKernelGGL((gn_one_bwd_rest<float, 4, R, FMT, ACT>), dim3(512 + npar), dim3(o.a.t.threads), lds, st, gyf, xf, codes, scales, o, tiles, npar,
                       k, dxf);
  }));
  if (params) hipLaunchKernelGGL(gn_one_params, dim3((C + 63) / 64), dim3(64), 0, st, o.b.ps, C, dgamma, dbeta);
  return true;
}
