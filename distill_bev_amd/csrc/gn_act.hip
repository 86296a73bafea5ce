// Group norm + activation, channels-last: y = act((x - mean_g) rstd_g gamma + beta), statistics per (image, group) over S pixels x C / G
// channels; forward (training or inference, optionally with an 8-bit checkpoint of x, act8.h) and backward (from x or the checkpoint).
//
// (Small images go through gn_small_fwd, large batches through gn_one_*, gn_one.hip.)
// Forward, two launches, no finalize launch between them:
//   gn_stats   a workgroup owns a chunk of one image's pixels x a range of channels, a thread one vector column: (mean, M2) of x - K_c, K_c
//              the chunk's first pixel, so that an offset of the data costs no digits.  Four rows at a time: their own mean, the squares
//              about it, merged with those before (M2 += M2_4 + delta^2 n 4 / (n + 4)): M2 is a sum of positive terms, wherever K_c and
//              outliers are.  Reduced to (mean, M2) per group and chunk in LDS.
//   gn_apply   every workgroup merges its image's chunk statistics itself -- a few KB from L2 against its share of x -- in fp64
//              (M2 = sum of M2_i + n_i (mean_i - mean)^2), then y, and the checkpoint from the same registers.
// Backward, two launches, xh = (x - mean) rstd, g = dy act'(gamma xh + beta):
//   gn_bwd_reduce   per chunk: sums of g and g xh per channel (for dbeta, dgamma), weighted with gamma per group (A, B)
//   gn_bwd_dx       dx = rstd (gamma g - A / D - xh B / D), D = S C / G; its first workgroups add the per-channel rows up instead
// Bound by HBM: 3 n es forward and 5 n es backward (n es = bytes of x; with a checkpoint the two reads of x in the backward are 1.03
// bytes a value).  All sums have a fixed order: run-to-run bit-identical, no atomics.
// Measured, fp32, SiLU: 1 x 128 x 1024 x 1024 forward 290 us (1.6 GB in three passes: 5.6 TB/s, part of the second read comes from the
// memory-side cache), backward 446; 8 x 128 x 128 x 128, int8 kept: 22 + 28 and 24 + 27 us, half of it cache; 6 x 256 x 15 x 25 backward: 7 + 7
// us, launch and merge latency.
#include "gn_act.h"
#include "gn_one.h"

namespace {

template <typename T, int V>
__global__ __launch_bounds__(256) void gn_stats(const T* __restrict__ x, GnArgs a, float2* __restrict__ part) {
  extern __shared__ float sh[];
  const GnPos p = gn_pos(a, blockIdx.x, V);
  const T* xi = x + static_cast<size_t>(p.n) * a.S * a.C + static_cast<size_t>(p.on ? p.col : 0) * V;
  float k[V], m[V], q[V];                                     // offset; mean - offset and M2 of the rows so far
#pragma unroll
  for (int i = 0; i < V; ++i) k[i] = m[i] = q[i] = 0.f;
  if (p.on) {
    A8Vec<T, V>::get(A8Vec<T, V>::load(xi + p.r0 * a.C), k);
    float n = 0.f;
    for (long long r = p.r0 + p.rp; r < a.S; r += p.step) {
      typename A8Vec<T, V>::Raw raw[GN_U];
#pragma unroll
      for (int u = 0; u < GN_U; ++u) raw[u] = A8Vec<T, V>::load(xi + min(r + u * a.t.RP, a.S - 1) * a.C);
      float d[GN_U][V];
#pragma unroll
      for (int u = 0; u < GN_U; ++u) {
        A8Vec<T, V>::get(raw[u], d[u]);
#pragma unroll
        for (int i = 0; i < V; ++i) d[u][i] -= k[i];
      }
      const bool full = r + (GN_U - 1) * a.t.RP < a.S;
      const float nb = full ? static_cast<float>(GN_U) : static_cast<float>((a.S - r + a.t.RP - 1) / a.t.RP);
      const float f = nb * __builtin_amdgcn_rcpf(n + nb), nf = n * f;
      const auto batch = [&](bool all, float inv) {           // (two bodies: only an image's last tile has rows to leave out)
#pragma unroll
        for (int i = 0; i < V; ++i) {
          float sum = 0.f, sq = 0.f;
#pragma unroll
          for (int u = 0; u < GN_U; ++u) sum += all || u < nb ? d[u][i] : 0.f;
          const float mb = sum * inv, delta = mb - m[i];
#pragma unroll
          for (int u = 0; u < GN_U; ++u) {
            const float e = d[u][i] - mb;
            sq = all || u < nb ? fmaf(e, e, sq) : sq;
          }
          q[i] += fmaf(delta * delta, nf, sq);
          m[i] = fmaf(delta, f, m[i]);
        }
      };
      if (full) batch(true, 1.f / GN_U);
      else batch(false, __builtin_amdgcn_rcpf(nb));
      n += nb;
    }
  }
  // per channel: the row phases merged the same way, mean and M2 of the chunk's pixels in sh[0 .. CH V), sh[CH V ..)
  const int w = a.t.CH * V, lane = threadIdx.x - p.rp * a.t.CH;
  float *t1 = sh + 2 * w, *t2 = t1 + a.t.RP * w;
  if (p.rp < a.t.RP) {
#pragma unroll
    for (int i = 0; i < V; ++i) {
      t1[p.rp * w + lane * V + i] = m[i];
      t2[p.rp * w + lane * V + i] = q[i];
    }
  }
  __syncthreads();
  const float rows = static_cast<float>(gn_rows(a, p.chunk));
  const T* x0 = x + static_cast<size_t>(p.n) * a.S * a.C + p.r0 * a.C + p.c0;
  const float each = static_cast<float>(gn_phase_rows(a, p.chunk, 0));
  const bool even = p.chunk != a.last;                        // all phases have as many rows
  for (int c = threadIdx.x; c < p.c1 - p.c0; c += blockDim.x) {
    float mean = 0.f, m2 = 0.f;
    if (even) {
#pragma unroll 4
      for (int r = 0; r < a.t.RP; ++r) mean += t1[r * w + c];
      mean /= static_cast<float>(a.t.RP);
#pragma unroll 4
      for (int r = 0; r < a.t.RP; ++r) {
        const float e = t1[r * w + c] - mean;
        m2 += fmaf(each * e, e, t2[r * w + c]);
      }
    } else {
      for (int r = 0; r < a.t.RP; ++r) mean = fmaf(static_cast<float>(gn_phase_rows(a, p.chunk, r)), t1[r * w + c], mean);
      mean /= rows;
      for (int r = 0; r < a.t.RP; ++r) {
        const float e = t1[r * w + c] - mean;
        m2 += fmaf(static_cast<float>(gn_phase_rows(a, p.chunk, r)) * e, e, t2[r * w + c]);
      }
    }
    sh[c] = static_cast<float>(x0[c]) + mean;
    sh[w + c] = m2;
  }
  __syncthreads();
  const int ng = p.g1 - p.g0, lanes = gn_lanes(ng), sub = threadIdx.x % lanes;
  for (int gi = threadIdx.x / lanes; gi < ng; gi += blockDim.x / lanes) {
    const int g = p.g0 + gi, cb = max(p.c0, g * a.cpg) - p.c0, ce = min(p.c1, (g + 1) * a.cpg) - p.c0;
    const float ref = sh[cb];                                 // (sums of offsets would cost digits)
    float m = 0.f;
    for (int c = cb + sub; c < ce; c += lanes) m += sh[c] - ref;
    m = ref + gn_lane_sum(m, lanes) / static_cast<float>(ce - cb);
    float m2 = 0.f;
    for (int c = cb + sub; c < ce; c += lanes) {
      const float d = sh[c] - m;
      m2 += fmaf(rows * d, d, sh[w + c]);
    }
    m2 = gn_lane_sum(m2, lanes);
    if (sub == 0) part[(static_cast<size_t>(p.n) * a.nchunk + p.chunk) * gn_row(a) + g + p.cc] = make_float2(m, m2);
  }
}

// The image's chunk rows of every group that this workgroup touches, added in fp64 into sh[2 gi], sh[2 gi + 1] behind the scratch: neighbouring
// threads take neighbouring groups of a row (coalesced), the chunks are spread over the rest of the workgroup, eight loads in flight.
// STATS: entries (mean, M2) -> (mean, rstd), from sum n m and sum (M2 + n m^2): the cancellation costs (mean / spread)^2 of 2^-53;
// else (A, B) -> (A / D, B / D)
template <bool STATS>
__device__ __forceinline__ float* gn_gather(float* sh, const GnArgs& a, const GnPos& p, int V, const float2* __restrict__ part, float eps) {
  double* scratch = reinterpret_cast<double*>(sh);
  float* out = sh + 4 * blockDim.x;
  const int ng = p.g1 - p.g0, w = a.t.CH * V;
  const int wide = min(ng, static_cast<int>(blockDim.x)), ph = threadIdx.x / wide, np = blockDim.x / wide;
  const float2* image = part + static_cast<size_t>(p.n) * a.nchunk * gn_row(a);
  const double D = static_cast<double>(a.S) * a.cpg;
  for (int first = 0; first < ng; first += wide) {
    const int gi = first + threadIdx.x - ph * wide, g = p.g0 + gi;
    double s0 = 0.0, s1 = 0.0;
    if (ph < np && gi < ng) {
      const int cca = a.t.ncol > 1 ? g * a.cpg / w : 0, ccb = a.t.ncol > 1 ? ((g + 1) * a.cpg - 1) / w + 1 : 1;
      for (int cc = cca; cc < ccb; ++cc) {
        const int width = a.t.ncol > 1 ? min((cc + 1) * w, (g + 1) * a.cpg) - max(cc * w, g * a.cpg) : a.cpg;
#pragma unroll 8
        for (int k = ph; k < a.nchunk; k += np) {
          const float2 e = image[static_cast<size_t>(k) * gn_row(a) + g + cc];
          if (STATS) {
            const double cnt = static_cast<double>(gn_rows(a, k)) * width, m = e.x;
            s0 += cnt * m;
            s1 += e.y + cnt * m * m;
          } else {
            s0 += e.x;
            s1 += e.y;
          }
        }
      }
    }
    scratch[threadIdx.x] = s0;
    scratch[blockDim.x + threadIdx.x] = s1;
    __syncthreads();
    if (ph == 0 && gi < ng) {
      for (int i = 1; i < np; ++i) {
        s0 += scratch[threadIdx.x + i * wide];
        s1 += scratch[blockDim.x + threadIdx.x + i * wide];
      }
      s0 /= D;
      s1 /= D;
      if (STATS) {
        const double var = s1 - s0 * s0;
        s1 = 1.0 / sqrt((var < 0.0 ? 0.0 : var) + static_cast<double>(eps));
      }
      out[2 * gi] = static_cast<float>(s0);
      out[2 * gi + 1] = static_cast<float>(s1);
    }
    __syncthreads();
  }
  return out;
}

template <typename T, int V, int FMT, int ACT, bool NT>
__global__ __launch_bounds__(256) void gn_apply(const T* __restrict__ x, GnArgs a, const float2* __restrict__ part, const float* __restrict__ gamma,
                                                const float* __restrict__ beta, float eps, T* __restrict__ y, float* __restrict__ mean,
                                                float* __restrict__ rstd, uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  extern __shared__ float sh[];
  constexpr int LB = 32 / V;
  const GnPos p = gn_pos(a, gridDim.x - 1 - blockIdx.x, V);
  const float* st = gn_gather<true>(sh, a, p, V, part, eps);
  if (mean != nullptr && p.chunk == 0)
    for (int gi = threadIdx.x; gi < p.g1 - p.g0; gi += blockDim.x)
      if ((p.g0 + gi) * a.cpg >= p.c0) {                      // the column range in which the group begins
        mean[static_cast<size_t>(p.n) * a.G + p.g0 + gi] = st[2 * gi];
        rstd[static_cast<size_t>(p.n) * a.G + p.g0 + gi] = st[2 * gi + 1];
      }
  if (p.rp >= a.t.RP) return;
  float sc[V], bt[V];
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = p.on ? p.col * V + i : 0, gi = p.on ? c / a.cpg - p.g0 : 0;
    sc[i] = st[2 * gi + 1] * (gamma != nullptr ? gamma[c] : 1.f);
    bt[i] = fmaf(-st[2 * gi], sc[i], beta != nullptr ? beta[c] : 0.f);
  }
  const size_t base = static_cast<size_t>(p.n) * a.S;
  for (long long r = p.r0 + p.rp; r < a.S; r += p.step) {
    typename A8Vec<T, V>::Raw raw[GN_U];
#pragma unroll
    for (int u = 0; u < GN_U; ++u) {
      const long long ru = r + u * a.t.RP;
      raw[u] = p.on && ru < a.S ? A8Vec<T, V>::template load<NT>(x + (base + ru) * a.C + static_cast<size_t>(p.col) * V) : A8Vec<T, V>::zero();
    }
#pragma unroll
    for (int u = 0; u < GN_U; ++u) {
      const long long ru = r + u * a.t.RP;
      if (ru >= a.S) break;                                  // all lanes of a block are on the same pixel
      float v[V];
      A8Vec<T, V>::get(raw[u], v);
      const size_t o = (base + ru) * a.C + static_cast<size_t>(p.col) * V;
      if (FMT != DBEV_ACT8_NONE) {
        unsigned m = 0;
#pragma unroll
        for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
        const unsigned b = a8_scale_byte<FMT>(a8_block_max<V>(m));
        if (p.on) {
          *reinterpret_cast<typename A8Bytes<V>::type*>(codes + o) = a8_encode<FMT, V>(v, b);
          if (p.col % LB == 0) scales[(base + ru) * a.nb + p.col / LB] = static_cast<uint8_t>(b);
        }
      }
      if (p.on) {
#pragma unroll
        for (int i = 0; i < V; ++i) v[i] = a8_act<ACT>(fmaf(v[i], sc[i], bt[i]));
        A8Vec<T, V>::template store<NT>(y + o, v);
      }
    }
  }
}

template <typename T, int V, int FMT, int ACT>
__global__ __launch_bounds__(256) void gn_bwd_reduce(const T* __restrict__ gy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                     const uint8_t* __restrict__ scales, GnArgs a, GnCoef k, float2* __restrict__ pc,
                                                     float2* __restrict__ pg) {
  extern __shared__ float sh[];
  const GnPos p = gn_pos(a, blockIdx.x, V);
  float s[V], q[V];
#pragma unroll
  for (int i = 0; i < V; ++i) s[i] = q[i] = 0.f;
  if (p.on) {
    float mu[V], rs[V], sc[V], bt[V];
#pragma unroll
    for (int i = 0; i < V; ++i) {
      const int c = p.col * V + i;
      mu[i] = k.mean[static_cast<size_t>(p.n) * a.G + c / a.cpg];
      rs[i] = k.rstd[static_cast<size_t>(p.n) * a.G + c / a.cpg];
      sc[i] = rs[i] * (k.gamma != nullptr ? k.gamma[c] : 1.f);
      bt[i] = k.beta != nullptr ? k.beta[c] : 0.f;
    }
    const size_t base = static_cast<size_t>(p.n) * a.S;
    for (long long r = p.r0 + p.rp; r < a.S; r += p.step) {
      typename A8Vec<T, V>::Raw draw[GN_U];
      GnX<T, V, FMT> xv[GN_U];
#pragma unroll
      for (int u = 0; u < GN_U; ++u) {
        const long long ru = r + u * a.t.RP;
        if (ru < a.S) {
          draw[u] = A8Vec<T, V>::load(gy + (base + ru) * a.C + static_cast<size_t>(p.col) * V);
          xv[u].load(x, codes, scales, base + ru, a.C, a.nb, p.col);
        }
      }
#pragma unroll
      for (int u = 0; u < GN_U; ++u) {
        if (r + u * a.t.RP >= a.S) break;
        float v[V], d[V];
        xv[u].get(v);
        A8Vec<T, V>::get(draw[u], d);
#pragma unroll
        for (int i = 0; i < V; ++i) {
          const float dev = v[i] - mu[i];
          const float g = a8_act_grad<ACT>(d[i], fmaf(dev, sc[i], bt[i]));
          s[i] += g;
          q[i] = fmaf(g, dev, q[i]);
        }
      }
    }
#pragma unroll
    for (int i = 0; i < V; ++i) q[i] *= rs[i];
  }
  gn_fold<V>(sh, a, p, s, q);
  const int w = a.t.CH * V;
  float2* row = pc + (static_cast<size_t>(p.n) * a.nchunk + p.chunk) * a.C + p.c0;
  for (int c = threadIdx.x; c < p.c1 - p.c0; c += blockDim.x) row[c] = make_float2(sh[c], sh[w + c]);
  const int ng = p.g1 - p.g0, lanes = gn_lanes(ng), sub = threadIdx.x % lanes;
  for (int gi = threadIdx.x / lanes; gi < ng; gi += blockDim.x / lanes) {
    const int g = p.g0 + gi, cb = max(p.c0, g * a.cpg) - p.c0, ce = min(p.c1, (g + 1) * a.cpg) - p.c0;
    float A = 0.f, B = 0.f;
    for (int c = cb + sub; c < ce; c += lanes) {
      const float gm = k.gamma != nullptr ? k.gamma[p.c0 + c] : 1.f;
      A = fmaf(gm, sh[c], A);
      B = fmaf(gm, sh[w + c], B);
    }
    A = gn_lane_sum(A, lanes);
    B = gn_lane_sum(B, lanes);
    if (sub == 0) pg[(static_cast<size_t>(p.n) * a.nchunk + p.chunk) * gn_row(a) + g + p.cc] = make_float2(A, B);
  }
}

constexpr int GN_PC = 8;                                      // channels of a workgroup that adds the parameter gradients up (64-byte pieces of a row)

// dgamma, dbeta: the rows of pc (one chunk's fp32 sums each) added in a fixed order in fp64
__device__ __forceinline__ void gn_param_grads(double* sh, const GnArgs& a, long long rows, int block, const float2* __restrict__ pc,
                                               float* __restrict__ dgamma, float* __restrict__ dbeta) {
  const int c = block * GN_PC + threadIdx.x % GN_PC, ph = threadIdx.x / GN_PC, np = blockDim.x / GN_PC;
  double s = 0.0, q = 0.0;
  if (c < a.C) {
#pragma unroll 8
    for (long long r = ph; r < rows; r += np) {
      const float2 e = pc[r * a.C + c];
      s += e.x;
      q += e.y;
    }
  }
  sh[2 * threadIdx.x] = s;
  sh[2 * threadIdx.x + 1] = q;
  __syncthreads();
  if (ph == 0 && c < a.C) {
    for (int i = 1; i < np; ++i) {
      s += sh[2 * (threadIdx.x + i * GN_PC)];
      q += sh[2 * (threadIdx.x + i * GN_PC) + 1];
    }
    if (dbeta != nullptr) dbeta[c] = static_cast<float>(s);
    if (dgamma != nullptr) dgamma[c] = static_cast<float>(q);
  }
}

template <typename T, int V, int FMT, int ACT, bool NT>
__global__ __launch_bounds__(256) void gn_bwd_dx(const T* __restrict__ gy, const T* __restrict__ x, const uint8_t* __restrict__ codes,
                                                 const uint8_t* __restrict__ scales, GnArgs a, GnCoef k, const float2* __restrict__ pc,
                                                 const float2* __restrict__ pg, int N, int npar, T* __restrict__ dx, float* __restrict__ dgamma, float* __restrict__ dbeta) {
  extern __shared__ float sh[];
  if (static_cast<int>(blockIdx.x) < npar) {
    gn_param_grads(reinterpret_cast<double*>(sh), a, static_cast<long long>(N) * a.nchunk, blockIdx.x, pc, dgamma, dbeta);
    return;
  }
  const GnPos p = gn_pos(a, static_cast<int>(gridDim.x - 1 - blockIdx.x), V);
  const float* ab = gn_gather<false>(sh, a, p, V, pg, 0.f);
  if (!p.on) return;
  float mu[V], sc[V], bt[V], A[V], B[V];                     // dx = sc g - (rstd A) - (x - mean) (rstd^2 B), sc = rstd gamma
#pragma unroll
  for (int i = 0; i < V; ++i) {
    const int c = p.col * V + i, g = c / a.cpg;
    const float rs = k.rstd[static_cast<size_t>(p.n) * a.G + g];
    mu[i] = k.mean[static_cast<size_t>(p.n) * a.G + g];
    sc[i] = rs * (k.gamma != nullptr ? k.gamma[c] : 1.f);
    bt[i] = k.beta != nullptr ? k.beta[c] : 0.f;
    A[i] = rs * ab[2 * (g - p.g0)];
    B[i] = rs * rs * ab[2 * (g - p.g0) + 1];
  }
  const size_t base = static_cast<size_t>(p.n) * a.S;
  for (long long r = p.r0 + p.rp; r < a.S; r += p.step) {
    typename A8Vec<T, V>::Raw draw[GN_U];
    GnX<T, V, FMT> xv[GN_U];
#pragma unroll
    for (int u = 0; u < GN_U; ++u) {
      const long long ru = r + u * a.t.RP;
      if (ru < a.S) {
        draw[u] = A8Vec<T, V>::template load<NT>(gy + (base + ru) * a.C + static_cast<size_t>(p.col) * V);
        xv[u].template load<NT>(x, codes, scales, base + ru, a.C, a.nb, p.col);
      }
    }
#pragma unroll
    for (int u = 0; u < GN_U; ++u) {
      const long long ru = r + u * a.t.RP;
      if (ru >= a.S) break;
      float v[V], d[V];
      xv[u].get(v);
      A8Vec<T, V>::get(draw[u], d);
#pragma unroll
      for (int i = 0; i < V; ++i) {
        const float dev = v[i] - mu[i];
        const float g = a8_act_grad<ACT>(d[i], fmaf(dev, sc[i], bt[i]));
        v[i] = fmaf(sc[i], g, -fmaf(dev, B[i], A[i]));
      }
      A8Vec<T, V>::template store<NT>(dx + (base + ru) * a.C + static_cast<size_t>(p.col) * V, v);
    }
  }
}

// ---- host ---------------------------------------------------------------------------------------------------------------------------
// Chunks per image: enough workgroups for sixteen per CU over the whole batch (twice what fits: 813 -> 776 us at 48 x 256 x 64 x 176 fp32 against
// eight), at least two tiles each, at most 128: every workgroup of the second launch reads its image's chunk rows, 8 G bytes a chunk.  Where
// 128 would leave fewer than four workgroups a CU, as many as make up for it, but no more than keep those rows below the chunk's own bytes.
// With at most 128 / 256 / 512 / 1024 chunks, fp32, SiLU, forward, us: one image of 256 channels, 256 x 256: 102 / 61 / 49 / 54; four: 166 /
// 138 / 136 / 174; one of 128 channels, 1024 x 1024: 994 / 560 / 366 / 292; eight of 128 channels, 128 x 128: 44 with 128, 47 with 181.  Taking
// the batch in slices that fit the 256 MB memory-side cache, so that the second launch would find its data there, was slower at every slice
// size (96 MB: 894 us against 823): a launch's ramp and its merge cost more than the cache gives.  Instead the second launch takes the
// workgroups' shares last to first, the most recently read data first, and tensors that are larger than that cache are read and written past
// it (backward, 48 x 256 x 64 x 176 bf16, SiLU, us: 300; last to first 282; past the cache 264; both 260.  With an operator that writes dy
// and one that reads dx around it: 498, 483, 470, 468)
GnArgs gn_args(int N, long long S, int C, int G, int V, int esize) {
  GnArgs a;
  a.S = S;
  a.C = C;
  a.cv = C / V;
  a.G = G;
  a.cpg = C / G;
  a.nb = (C + 31) / 32;
  a.t = a8_tile(C, V);
  const long long side = static_cast<long long>(N) * a.t.ncol, most = (S + 2 * gn_tile(a) - 1) / (2 * gn_tile(a));
  long long want = (GN_BLOCKS + side - 1) / side;
  long long cap = static_cast<long long>(sqrt(static_cast<double>(S) * C * esize / (8.0 * G)));
  if (cap > (GN_BLOCKS / 4 + side - 1) / side) cap = (GN_BLOCKS / 4 + side - 1) / side;
  if (cap < 128) cap = 128;
  want = want < 1 ? 1 : want > cap ? cap : want;
  a.nchunk = static_cast<int>(want > most ? most : want);
  const long long tiles = (S + gn_tile(a) - 1) / gn_tile(a);
  a.tiles_each = static_cast<int>(tiles / a.nchunk);
  a.extra = static_cast<int>(tiles % a.nchunk);
  a.last = static_cast<int>((tiles - 1) % a.nchunk);
  a.lack = static_cast<int>(tiles * gn_tile(a) - S);
  return a;
}

size_t gn_lds(const GnArgs& a, int V) {
  const size_t fold = static_cast<size_t>(2) * a.t.CH * V * (1 + a.t.RP) * sizeof(float);
  const size_t gather = static_cast<size_t>(2) * a.t.threads * sizeof(double) + static_cast<size_t>(2) * (a.G < a.t.CH * V ? a.G : a.t.CH * V) * sizeof(float);
  return fold > gather ? fold : gather;
}

bool gn_ok(int dtype, int N, long long S, int C, int G) {
  return a8_dtype_ok(dtype) && N >= 0 && S >= 0 && C > 0 && G > 0 && C % G == 0 && C <= 65536 && S <= (1LL << 36) / C && S <= (1LL << 30) &&
         static_cast<long long>(N) <= (1LL << 22) && (N == 0 || S <= (1LL << 40) / C / N);
}

// a launch holds fewer than 2^32 threads
bool gn_grid_ok(int N, const GnArgs& a) { return static_cast<long long>(N) * a.nchunk * a.t.ncol * a.t.threads < (1LL << 32) - (1LL << 26); }

// the chunk rows of whatever element type and vector width a call ends up with (the backward's: C sums, then the groups'); fp32 has at least as
// many chunks as the 16-bit types
size_t gn_ws(int N, long long S, int C, int G) {
  size_t m = gn_one_bytes(N, S, C, G);
  for (int v : {1, 2, 4, 8}) {
    if (C % v != 0) break;
    const GnArgs a = gn_args(N, S, C, G, v, sizeof(float));
    const size_t b = static_cast<size_t>(N) * a.nchunk * (static_cast<size_t>(C) + gn_row(a)) * sizeof(float2);
    m = b > m ? b : m;
  }
  return m;
}

}  // namespace

extern "C" size_t dbev_gn_act_workspace_bytes(int N, long long S, int C, int G) {
  if (!gn_ok(DBEV_DT_F32, N, S, C, G) || N == 0 || S == 0) return 0;
  return gn_ws(N, S, C, G);
}

extern "C" int dbev_gn_act_form(int dtype, int N, long long S, int C, int G, int fmt, int backward) {
  if (!gn_ok(dtype, N, S, C, G) || !(fmt == DBEV_ACT8_NONE || a8_fmt_ok(fmt)) || N == 0 || S == 0) return -1;
  if (!backward && gn_small_takes(dtype, N, S, C, G)) return 1;
  return gn_one_takes(dtype, N, S, C, fmt, backward != 0) ? 2 : 0;
}

extern "C" int dbev_gn_act_forward(const void* x, int dtype, int N, long long S, int C, int G, const float* gamma, const float* beta, float eps,
                                   int act, void* y, float* mean, float* rstd, int fmt, uint8_t* codes, uint8_t* scales, void* workspace,
                                   size_t workspace_bytes, dbevStream_t stream) {
  if (!gn_ok(dtype, N, S, C, G) || !a8_act_ok(act) || !(fmt == DBEV_ACT8_NONE || a8_fmt_ok(fmt))) return DBEV_EINVAL;
  if (N == 0 || S == 0) return 0;
  if (workspace_bytes < gn_ws(N, S, C, G)) return DBEV_EINVAL;
  const int vec = a8_pick_vec(a8_elem_size(dtype), C, C, x, y, nullptr);
  hipStream_t st = dbev_stream(stream);
  if ((fmt == DBEV_ACT8_NONE || reinterpret_cast<uintptr_t>(codes) % 8 == 0) &&
      (gn_small_forward(x, dtype, vec, N, S, C, G, gamma, beta, eps, act, y, mean, rstd, fmt, codes, scales, st) ||
       gn_one_forward(x, dtype, vec, N, S, C, G, gamma, beta, eps, act, y, mean, rstd, fmt, codes, scales, workspace, st))) {
    DBEV_LAUNCH_CHECK();
    return 0;
  }
  float2* part = static_cast<float2*>(workspace);
  A8_TYPE_SWITCH(dtype, vec, {
    const GnArgs a = gn_args(N, S, C, G, V, sizeof(T));
    if ((fmt != DBEV_ACT8_NONE && reinterpret_cast<uintptr_t>(codes) % V != 0) || !gn_grid_ok(N, a)) return DBEV_EINVAL;
    const dim3 grid(static_cast<unsigned>(N) * a.nchunk * a.t.ncol), block(a.t.threads);
    hipLaunchKernelGGL((gn_stats<T, V>), grid, block, gn_lds(a, V), st, static_cast<const T*>(x), a, part);
    DBEV_LAUNCH_CHECK();
    A8_NT_SWITCH(S * C * N * static_cast<long long>(sizeof(T)), A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
      hipLaunchKernelGGL((gn_apply<T, V, FMT, ACT, NT>), grid, block, gn_lds(a, V), st, static_cast<const T*>(x), a, part, gamma, beta, eps,
                         static_cast<T*>(y), mean, rstd, codes, scales);
    })));
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}

extern "C" int dbev_gn_act_backward(const void* gy, int dtype, const void* x, int fmt, const uint8_t* codes, const uint8_t* scales, int N, long long S,
                                    int C, int G, const float* gamma, const float* beta, const float* mean, const float* rstd, int act, void* dx,
                                    float* dgamma, float* dbeta, void* workspace, size_t workspace_bytes, dbevStream_t stream) {
  if (!gn_ok(dtype, N, S, C, G) || !a8_act_ok(act) || !(fmt == DBEV_ACT8_NONE ? x != nullptr : a8_fmt_ok(fmt))) return DBEV_EINVAL;
  if (N == 0 || S == 0) return 0;
  if (workspace_bytes < gn_ws(N, S, C, G)) return DBEV_EINVAL;
  const int vec = a8_pick_vec(a8_elem_size(dtype), C, C, gy, dx, fmt == DBEV_ACT8_NONE ? x : nullptr);
  hipStream_t st = dbev_stream(stream);
  if ((fmt == DBEV_ACT8_NONE || reinterpret_cast<uintptr_t>(codes) % 8 == 0) &&
      gn_one_backward(gy, dtype, vec, x, fmt, codes, scales, N, S, C, G, gamma, beta, mean, rstd, act, dx, dgamma, dbeta, workspace, st)) {
    DBEV_LAUNCH_CHECK();
    return 0;
  }
  const GnCoef k = {gamma, beta, mean, rstd};
  A8_TYPE_SWITCH(dtype, vec, {
    const GnArgs a = gn_args(N, S, C, G, V, sizeof(T));
    if ((fmt != DBEV_ACT8_NONE && reinterpret_cast<uintptr_t>(codes) % V != 0) || !gn_grid_ok(N, a)) return DBEV_EINVAL;
    float2* pc = static_cast<float2*>(workspace);
    float2* pg = pc + static_cast<size_t>(N) * a.nchunk * C;
    const unsigned blocks = static_cast<unsigned>(N) * a.nchunk * a.t.ncol;
    const int npar = (dgamma != nullptr || dbeta != nullptr) ? (C + GN_PC - 1) / GN_PC : 0;
    A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
      hipLaunchKernelGGL((gn_bwd_reduce<T, V, FMT, ACT>), dim3(blocks), dim3(a.t.threads), gn_lds(a, V), st, static_cast<const T*>(gy),
                         static_cast<const T*>(x), codes, scales, a, k, pc, pg);
      A8_NT_SWITCH(S * C * N * static_cast<long long>(sizeof(T)), {
        hipLaunchKernelGGL((gn_bwd_dx<T, V, FMT, ACT, NT>), dim3(blocks + npar), dim3(a.t.threads), gn_lds(a, V), st, static_cast<const T*>(gy),
                           static_cast<const T*>(x), codes, scales, a, k, pc, pg, N, npar, static_cast<T*>(dx), dgamma, dbeta);
      });
    }));
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}
