// Shared parts of the group norm's kernels: gn_act.hip (two launches a direction) and gn_one.hip (one pass over the data).
#pragma once
#include "act8.h"

namespace {

constexpr int GN_U = 4;                                       // rows in flight per thread
constexpr int GN_BLOCKS = 4096;                               // workgroups of a launch that the chunking aims at

struct GnArgs {
  long long S;                                                // pixels of an image
  int C, cv, G, cpg, nb;                                      // channels, vector columns, groups, channels a group, blocks of 32 a row
  // an image's pixels in tiles of RP * GN_U; chunk k takes the tiles k, k + nchunk, ...: the workgroups of an image sweep its memory side by
  // side, as one front (3 % faster than with a region of its own for each)
  int nchunk;
  int tiles_each, extra, last;                                // tiles of a chunk, chunks with one more, the chunk that holds the image's last tile
  int lack;                                                   // pixels missing from that tile
  A8Tile t;
};
// Entries of a chunk's row of per-group numbers: a group that crosses a border of column ranges has one in each.  Entry g + cc for group g in
// range cc: neighbouring ranges share at most their border's group, so that no two are the same
__host__ __device__ __forceinline__ int gn_row(const GnArgs& a) { return a.G + a.t.ncol - 1; }
__host__ __device__ __forceinline__ long long gn_tile(const GnArgs& a) { return static_cast<long long>(a.t.RP) * GN_U; }
// pixels of a chunk
__device__ __forceinline__ int gn_rows(const GnArgs& a, int chunk) {
  return (a.tiles_each + (chunk < a.extra ? 1 : 0)) * (a.t.RP * GN_U) - (chunk == a.last ? a.lack : 0);
}

// ... of them, those of row phase rp
__device__ __forceinline__ int gn_phase_rows(const GnArgs& a, int chunk, int rp) {
  const int n = (a.tiles_each + (chunk < a.extra ? 1 : 0)) * GN_U;
  if (chunk != a.last) return n;
  const int left = a.t.RP * GN_U - a.lack - rp;               // pixels of the image's last tile from this phase on
  return n - GN_U + (left > 0 ? (left + a.t.RP - 1) / a.t.RP : 0);
}

// (image, pixel chunk, column range) of this workgroup
struct GnPos { int n, chunk, cc, col, c0, c1, g0, g1, rp; bool on; long long r0, step; };
__device__ __forceinline__ GnPos gn_pos(const GnArgs& a, int block, int V) {
  GnPos p;
  p.cc = block % a.t.ncol;
  const int b = block / a.t.ncol;
  p.chunk = b % a.nchunk;
  p.n = b / a.nchunk;
  p.rp = threadIdx.x / a.t.CH;
  p.col = p.cc * a.t.CH + (threadIdx.x - p.rp * a.t.CH);
  p.on = p.rp < a.t.RP && p.col < a.cv;
  p.c0 = p.cc * a.t.CH * V;
  p.c1 = min(a.C, p.c0 + a.t.CH * V);
  p.g0 = p.c0 / a.cpg;
  p.g1 = (p.c1 - 1) / a.cpg + 1;
  p.r0 = p.chunk * gn_tile(a);
  p.step = a.nchunk * gn_tile(a);
  return p;
}

// lanes that share one group's work: the workgroup's threads spread over its groups, at most a wave each
__device__ __forceinline__ int gn_lanes(int ng) {
  int l = 64;
  while (l > 1 && ng * l > static_cast<int>(blockDim.x)) l >>= 1;
  return l;
}
template <typename F>
__device__ __forceinline__ F gn_lane_sum(F v, int lanes) {
  for (int o = lanes >> 1; o > 0; o >>= 1) v += __shfl_xor(v, o);
  return v;
}

// the two per-thread sums of every column -> per channel in sh[0 .. CH V), sh[CH V ..): row phases added in order
template <int V>
__device__ __forceinline__ void gn_fold(float* sh, const GnArgs& a, const GnPos& p, const float* s, const float* q) {
  const int w = a.t.CH * V, lane = threadIdx.x - p.rp * a.t.CH;
  float* t1 = sh + 2 * w;                                     // [RP][CH V] twice
  float* t2 = t1 + a.t.RP * w;
  if (p.rp < a.t.RP) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      t1[p.rp * w + lane * V + i] = s[i];
      t2[p.rp * w + lane * V + i] = q[i];
    }
  }
  __syncthreads();
  for (int c = threadIdx.x; c < w; c += blockDim.x) {
    float a1 = 0.f, a2 = 0.f;
    for (int r = 0; r < a.t.RP; ++r) {
      a1 += t1[r * w + c];
      a2 += t2[r * w + c];
    }
    sh[c] = a1;
    sh[w + c] = a2;
  }
  __syncthreads();
}

// one vector of the backward pass's view of x: x itself or its checkpoint
template <typename T, int V, int FMT>
struct GnX {
  typename A8Bytes<V>::type c;
  unsigned b;
  typename A8Vec<T, V>::Raw v;
  template <bool NT = false>
  __device__ __forceinline__ void load(const T* x, const uint8_t* codes, const uint8_t* scales, size_t row, int C, int nb, int col) {
    if (FMT == DBEV_ACT8_NONE) v = A8Vec<T, V>::template load<NT>(x + row * C + static_cast<size_t>(col) * V);
    else {
      c = *reinterpret_cast<const typename A8Bytes<V>::type*>(codes + row * C + static_cast<size_t>(col) * V);
      b = scales[row * nb + col / (32 / V)];
    }
  }
  __device__ __forceinline__ void get(float* o) const {
    if (FMT == DBEV_ACT8_NONE) A8Vec<T, V>::get(v, o);
    else a8_decode<FMT, V>(c, a8_scale(b), o);
  }
};

struct GnCoef { const float *gamma, *beta, *mean, *rstd; };

}  // namespace
