// Weight and bias gradient of a linear layer (or 1x1 convolution, channels-last) whose saved input is an 8-bit checkpoint (act8.h):
//   gw[Co, Ci] = sum_m gy[m, Co] * x^[m, Ci],   gb[Co] = sum_m gy[m, Co]
// on the bf16 matrix cores.  x^ = code * 2^k has at most 8 significant bits: it is a bf16 number, one operand plane.  gy is split exactly,
// by truncation, into as many bf16 pieces as its type has: three for fp32 (8 + 8 + 8 bits), two for fp16, one for bf16.  Every partial
// product is exact in fp32, the sums are fp32: fp32 accuracy for three matrix instructions where a product of two fp32 operands takes six.
//
// The reduction runs over m, the slow index of both operands, while a matrix instruction wants 8 consecutive m of one channel per lane:
// a thread fetches 8 rows of a few channels (coalesced along the channels), so that a channel's 8 values sit in its registers and go to
// LDS as one 16-byte unit [m / 8][channel]; the unit index is channel ^ ((channel >> 4) & 3), which spreads both the strided writes and
// the reads over all banks.  Workgroup = 4 waves, tile TA output x TB input channels, chunks of 32 rows, two LDS buffers, one barrier per
// chunk; raw values are fetched through buffer descriptors of the share's rows (a row or channel past the end reads as zero).  The rows
// are cut into shares, partial sums [share][Co][Ci] are added in a fixed order by a8_wsum: bit-reproducible, no atomics.
#include "act8.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

constexpr int A8W_KC = 32;                                    // rows a chunk: two reduction steps of 16
constexpr unsigned A8W_OOB = 0x80000000u;                     // offset of a channel past the end: beyond every descriptor (shares stay below 2 GiB)

template <typename T> struct A8Pieces;
template <> struct A8Pieces<float> { static constexpr int n = 3; };
template <> struct A8Pieces<a8_f16> { static constexpr int n = 2; };
template <> struct A8Pieces<a8_bf16> { static constexpr int n = 1; };

__device__ __forceinline__ unsigned long long a8w_uniform(unsigned long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v >> 32));
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t a8w_rsrc(const void* p, long long bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(a8w_uniform(reinterpret_cast<unsigned long long>(p))), 0,
                                           __builtin_amdgcn_readfirstlane(static_cast<int>(bytes < 0 ? 0 : bytes)), 0x00020000);
}

// upper halves of two dwords: (hi(b) << 16) | hi(a)
__device__ __forceinline__ unsigned a8w_hi2(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// (a, b) -> NP dwords of two bf16 each, their sums are a and b exactly: truncation leaves the remainder exact.  INF: the remainder of an
// infinity, inf - inf, is taken as 0, so that the products see inf and not a NaN.
template <int NP, bool INF>
__device__ __forceinline__ void a8w_split(float a, float b, unsigned* p) {
  p[0] = a8w_hi2(__float_as_uint(a), __float_as_uint(b));
#pragma unroll
  for (int i = 1; i < NP; ++i) {
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    a = INF && __builtin_isinf(a) ? 0.f : ra;
    b = INF && __builtin_isinf(b) ? 0.f : rb;
    p[i] = a8w_hi2(__float_as_uint(a), __float_as_uint(b));
  }
}

// raw bits of `n` consecutive elements of `es` bytes, one or several loads (n * es <= 8 bytes; VEC: one access)
template <typename T, int N, bool VEC>
struct A8Raw {
  float v[N];
  __device__ __forceinline__ void load(__amdgpu_buffer_rsrc_t r, const unsigned* off) {
    if (sizeof(T) == 4) {
      if (VEC && N == 2) {
        typedef unsigned u2 __attribute__((ext_vector_type(2)));
        const u2 t = __builtin_bit_cast(u2, __builtin_amdgcn_raw_buffer_load_b64(r, off[0], 0, 0));
        v[0] = __uint_as_float(t[0]);
        v[N - 1] = __uint_as_float(t[1]);
      } else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off[i], 0, 0));
      }
    } else {
      if (VEC && N == 2) v[0] = __uint_as_float(__builtin_amdgcn_raw_buffer_load_b32(r, off[0], 0, 0));
      else {
#pragma unroll
        for (int i = 0; i < N; ++i) v[i] = __uint_as_float(static_cast<unsigned>(static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(r, off[i], 0, 0))));
      }
    }
  }
  __device__ __forceinline__ float get(int i) const {
    if (sizeof(T) == 4) return v[i];
    const unsigned bits = (VEC && N == 2) ? (i ? __float_as_uint(v[0]) >> 16 : __float_as_uint(v[0]) & 0xffffu) : __float_as_uint(v[i]);
    const unsigned short h = static_cast<unsigned short>(bits);
    return static_cast<float>(__builtin_bit_cast(T, h));
  }
};
template <> __device__ __forceinline__ float A8Raw<float, 1, true>::get(int i) const { return v[i]; }
template <> __device__ __forceinline__ float A8Raw<float, 1, false>::get(int i) const { return v[i]; }
template <> __device__ __forceinline__ float A8Raw<float, 2, true>::get(int i) const { return v[i]; }
template <> __device__ __forceinline__ float A8Raw<float, 2, false>::get(int i) const { return v[i]; }

template <typename T, int FMT, int TA, int TB, bool VEC>
__global__ __launch_bounds__(256, 2) void a8_wgrad(const T* __restrict__ gy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
                                                   float* __restrict__ part, float* __restrict__ bpart, long long M, int Co, int Ci, int nb,
                                                   int tiles_n, int tiles, int rows_per, int nsplit) {
  constexpr int NP = A8Pieces<T>::n, CA = TA / 64, CB = TB / 64;
  constexpr int PLA = TA * 64, PLB = TB * 64, BUF = NP * PLA + PLB;
  constexpr int WM = (TA == 64 && TB == 64) ? 2 : TA / 64, WN = 4 / WM, NA = TA / 32 / WM, NB = TB / 32 / WN;
  extern __shared__ __attribute__((aligned(16))) unsigned char smem[];
  const int tid = threadIdx.x, lane = tid & 63, w = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int half = lane >> 5, l31 = lane & 31, wm = w % WM, wn = w / WM;
  const int L = xcd_block(), tile = L % tiles, split = L / tiles;
  if (split >= nsplit) return;
  const int co0 = (tile / tiles_n) * TA, ci0 = (tile % tiles_n) * TB;
  const long long mbeg = static_cast<long long>(split) * rows_per;
  const int nrows = static_cast<int>(min(static_cast<long long>(rows_per), M - mbeg)), nch = (nrows + A8W_KC - 1) / A8W_KC;

  // staging role: rows 8 w .. 8 w + 7 of the chunk, channels CA lane .. of the gradient, CB lane .. of the checkpoint
  const T* gbase = gy + static_cast<size_t>(mbeg) * Co;
  const uint8_t* cbase = codes + static_cast<size_t>(mbeg) * Ci;
  const uint8_t* sbase = scales + static_cast<size_t>(mbeg) * nb;
  unsigned aoff[CA], boff[CB], soff[CB];
#pragma unroll
  for (int i = 0; i < CA; ++i) {
    const int c = co0 + CA * lane + i;
    aoff[i] = c < Co ? static_cast<unsigned>(8 * w * Co + c) * sizeof(T) : A8W_OOB;
  }
#pragma unroll
  for (int i = 0; i < CB; ++i) {
    const int c = ci0 + CB * lane + i;
    boff[i] = c < Ci ? static_cast<unsigned>(8 * w * Ci + c) : A8W_OOB;
    soff[i] = c < Ci ? static_cast<unsigned>(8 * w * nb + c / 32) : A8W_OOB;
  }
  A8Raw<T, CA, VEC> ra[8];
  unsigned rb[8], rs[8];                                      // CB code bytes; their block's scale byte (CB channels never straddle a block)
  const bool bias = bpart != nullptr && ci0 == 0;
  float bsum[CA];
#pragma unroll
  for (int i = 0; i < CA; ++i) bsum[i] = 0.f;

  auto fetch = [&](int ch) {
    const long long r0 = static_cast<long long>(ch) * A8W_KC, left = nrows - r0;
    const __amdgpu_buffer_rsrc_t gr = a8w_rsrc(gbase + r0 * Co, left * Co * static_cast<long long>(sizeof(T)));
    const __amdgpu_buffer_rsrc_t cr = a8w_rsrc(cbase + r0 * Ci, left * Ci);
    const __amdgpu_buffer_rsrc_t sr = a8w_rsrc(sbase + r0 * nb, left * nb);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      unsigned o[CA];
#pragma unroll
      for (int i = 0; i < CA; ++i) o[i] = aoff[i] + static_cast<unsigned>(k * Co) * sizeof(T);
      ra[k].load(gr, o);
    }
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      const unsigned ko = static_cast<unsigned>(k * Ci);
      if (VEC && CB == 4) rb[k] = __builtin_amdgcn_raw_buffer_load_b32(cr, boff[0] + ko, 0, 0);
      else if (VEC && CB == 2) rb[k] = static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(cr, boff[0] + ko, 0, 0));
      else {
        rb[k] = 0;
#pragma unroll
        for (int i = 0; i < CB; ++i) rb[k] |= static_cast<unsigned>(static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(cr, boff[i] + ko, 0, 0))) << (8 * i);
      }
      rs[k] = static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(sr, soff[0] + static_cast<unsigned>(k * nb), 0, 0));
    }
  };

  auto stage = [&](unsigned char* buf) {
    float top = 0.f;                                          // the largest |gy| of this thread: infinities are rare, one test for all
    if (NP > 1) {
#pragma unroll
      for (int k = 0; k < 8; ++k)
#pragma unroll
        for (int c = 0; c < CA; ++c) top = fmaxf(top, fabsf(ra[k].get(c)));
    }
#pragma unroll
    for (int c = 0; c < CA; ++c) {
      unsigned p[4][3];
      if (NP > 1 && __builtin_expect(top == __builtin_inff(), 0)) {
#pragma unroll
        for (int k = 0; k < 4; ++k) a8w_split<NP, true>(ra[2 * k].get(c), ra[2 * k + 1].get(c), p[k]);
      } else {
#pragma unroll
        for (int k = 0; k < 4; ++k) a8w_split<NP, false>(ra[2 * k].get(c), ra[2 * k + 1].get(c), p[k]);
      }
      if (bias) {
#pragma unroll
        for (int k = 0; k < 4; ++k) bsum[c] += ra[2 * k].get(c) + ra[2 * k + 1].get(c);
      }
      const int row = CA * lane + c;
      unsigned char* d = buf + (w * TA + (row ^ ((row >> 4) & 3))) * 16;
#pragma unroll
      for (int i = 0; i < NP; ++i) *reinterpret_cast<uintx4*>(d + i * PLA) = uintx4{p[0][i], p[1][i], p[2][i], p[3][i]};
    }
    float x[8][4];
#pragma unroll
    for (int k = 0; k < 8; ++k) a8_decode4<FMT>(rb[k], a8_scale(rs[k]), x[k]);
#pragma unroll
    for (int c = 0; c < CB; ++c) {
      const int row = CB * lane + c;
      uintx4 u;
#pragma unroll
      for (int k = 0; k < 4; ++k) u[k] = a8w_hi2(__float_as_uint(x[2 * k][c]), __float_as_uint(x[2 * k + 1][c]));     // exact: bf16 numbers
      *reinterpret_cast<uintx4*>(buf + NP * PLA + (w * TB + (row ^ ((row >> 4) & 3))) * 16) = u;
    }
  };

  floatx16 acc[NA][NB];
#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b)
#pragma unroll
      for (int r = 0; r < 16; ++r) acc[a][b][r] = 0.f;
  int aaddr[NA], baddr[NB];
#pragma unroll
  for (int a = 0; a < NA; ++a) {
    const int r = (wm * NA + a) * 32 + l31;
    aaddr[a] = (half * TA + (r ^ ((r >> 4) & 3))) * 16;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int r = (wn * NB + b) * 32 + l31;
    baddr[b] = NP * PLA + (half * TB + (r ^ ((r >> 4) & 3))) * 16;
  }

  fetch(0);
  stage(smem);
  fetch(1);
  __syncthreads();
  for (int ch = 0; ch < nch; ++ch) {
    const unsigned char* rd = smem + (ch & 1) * BUF;
#pragma unroll
    for (int s = 0; s < 2; ++s) {
      bf16x8 af[NA][NP], bf[NB];
#pragma unroll
      for (int b = 0; b < NB; ++b) bf[b] = *reinterpret_cast<const bf16x8*>(rd + baddr[b] + s * 2 * TB * 16);
#pragma unroll
      for (int p = 0; p < NP; ++p)
#pragma unroll
        for (int a = 0; a < NA; ++a) af[a][p] = *reinterpret_cast<const bf16x8*>(rd + p * PLA + aaddr[a] + s * 2 * TA * 16);
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)                       // the smallest pieces first
#pragma unroll
        for (int a = 0; a < NA; ++a)
#pragma unroll
          for (int b = 0; b < NB; ++b) acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[a][p], bf[b], acc[a][b], 0, 0, 0);
    }
    if (ch + 1 < nch) {
      stage(smem + ((ch + 1) & 1) * BUF);
      fetch(ch + 2);                                          // (past the last chunk: empty descriptors, zeros)
    }
    __syncthreads();
  }

#pragma unroll
  for (int a = 0; a < NA; ++a)
#pragma unroll
    for (int b = 0; b < NB; ++b) {
      const int co = co0 + (wm * NA + a) * 32 + 4 * half, ci = ci0 + (wn * NB + b) * 32 + l31;
      float* o = part + (static_cast<size_t>(split) * Co + co) * Ci + ci;
#pragma unroll
      for (int r = 0; r < 16; ++r) {
        const int d = (r & 3) + 8 * (r >> 2);
        if (co + d < Co && ci < Ci) o[static_cast<size_t>(d) * Ci] = acc[a][b][r];
      }
    }
  if (bias) {                                                 // the four waves' rows of every channel, in order (smem is free behind the last barrier)
    float* sb = reinterpret_cast<float*>(smem);
#pragma unroll
    for (int c = 0; c < CA; ++c) sb[w * TA + CA * lane + c] = bsum[c];
    __syncthreads();
    for (int c = tid; c < TA && co0 + c < Co; c += 256)
      bpart[static_cast<size_t>(split) * Co + co0 + c] = (sb[c] + sb[TA + c]) + (sb[2 * TA + c] + sb[3 * TA + c]);
  }
}

// the shares added in a fixed order, rounded once to the output type; elements [0, plane) the weight gradient, [plane, plane + Co) the bias's
template <typename T>
__global__ __launch_bounds__(256) void a8_wsum(const float* __restrict__ part, const float* __restrict__ bpart, int nsplit, long long plane, int Co,
                                               T* __restrict__ gw, T* __restrict__ gb) {
  const long long idx = static_cast<long long>(blockIdx.x) * 256 + threadIdx.x;
  const bool isb = idx >= plane;
  if (idx >= plane + (gb != nullptr ? Co : 0)) return;
  const float* p = isb ? bpart + (idx - plane) : part + idx;
  const long long step = isb ? Co : plane;
  float s0 = 0.f, s1 = 0.f, s2 = 0.f, s3 = 0.f;
  int s = 0;
  for (; s + 4 <= nsplit; s += 4) {
    s0 += p[(s + 0) * step];
    s1 += p[(s + 1) * step];
    s2 += p[(s + 2) * step];
    s3 += p[(s + 3) * step];
  }
  for (; s < nsplit; ++s) s0 += p[s * step];
  (isb ? gb[idx - plane] : gw[idx]) = static_cast<T>((s0 + s1) + (s2 + s3));
}

struct A8WPlan { int ta, tb, tiles_n, tiles, rows_per, nsplit, grid; };

bool a8w_plan(long long M, int Ci, int Co, A8WPlan* p) {
  if (M < 0 || Ci <= 0 || Co <= 0 || Ci > 65536 || Co > 65536 || M > (1LL << 40) / (Ci > Co ? Ci : Co)) return false;
  p->ta = Co > 64 ? 128 : 64;
  p->tb = Ci > 128 ? 256 : Ci > 64 ? 128 : 64;
  p->tiles_n = (Ci + p->tb - 1) / p->tb;
  p->tiles = (Co + p->ta - 1) / p->ta * p->tiles_n;
  long long ns = 512 / p->tiles;                              // two workgroups a CU
  const long long most = (M + 127) / 128;                     // at least four chunks a share
  ns = ns > most ? most : ns;
  ns = ns < 1 ? 1 : ns;
  // a share's rows are addressed with 31 bits of bytes
  const long long cap = ((1LL << 31) - (1 << 20)) / (4LL * (Co > Ci ? Co : Ci)) / A8W_KC * A8W_KC;
  long long rows = (M + ns - 1) / ns;
  rows = (rows + A8W_KC - 1) / A8W_KC * A8W_KC;
  if (rows > cap) rows = cap;
  if (rows < A8W_KC) rows = A8W_KC;
  ns = M > 0 ? (M + rows - 1) / rows : 0;
  if (ns * p->tiles > (1 << 23)) return false;
  p->rows_per = static_cast<int>(rows);
  p->nsplit = static_cast<int>(ns);
  p->grid = dbev_round_xcd(p->nsplit * p->tiles);
  return true;
}

size_t a8w_bytes(const A8WPlan& p, int Ci, int Co) { return static_cast<size_t>(p.nsplit) * Co * (static_cast<size_t>(Ci) + 1) * sizeof(float); }

template <typename T, int FMT, int TA, int TB, bool VEC>
hipError_t a8w_launch(const A8WPlan& p, const void* gy, const uint8_t* codes, const uint8_t* scales, float* part, float* bpart, long long M, int Co, int Ci,
                      hipStream_t st) {
  constexpr int lds = 2 * (A8Pieces<T>::n * TA * 64 + TB * 64);
  auto* fn = a8_wgrad<T, FMT, TA, TB, VEC>;
  if (lds > 64 * 1024) {                                       // idempotent, per device; not a stream operation
    const hipError_t e = hipFuncSetAttribute(reinterpret_cast<const void*>(fn), hipFuncAttributeMaxDynamicSharedMemorySize, lds);
    if (e != hipSuccess) return e;
  }
  hipLaunchKernelGGL(fn, dim3(p.grid), dim3(256), lds, st, static_cast<const T*>(gy), codes, scales, part, bpart, M, Co, Ci, (Ci + 31) / 32, p.tiles_n,
                     p.tiles, p.rows_per, p.nsplit);
  return hipGetLastError();
}

template <typename T, int FMT, bool VEC>
hipError_t a8w_tiles(const A8WPlan& p, const void* gy, const uint8_t* codes, const uint8_t* scales, float* part, float* bpart, long long M, int Co, int Ci,
                     hipStream_t st) {
  if (p.ta == 128) {
    if (p.tb == 256) return a8w_launch<T, FMT, 128, 256, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
    if (p.tb == 128) return a8w_launch<T, FMT, 128, 128, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
    return a8w_launch<T, FMT, 128, 64, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
  }
  if (p.tb == 256) return a8w_launch<T, FMT, 64, 256, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
  if (p.tb == 128) return a8w_launch<T, FMT, 64, 128, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
  return a8w_launch<T, FMT, 64, 64, VEC>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
}

template <typename T>
int a8w_run(const A8WPlan& p, const void* gy, const uint8_t* codes, const uint8_t* scales, int fmt, long long M, int Ci, int Co, void* gw, void* gb,
            void* workspace, hipStream_t st) {
  float* part = static_cast<float*>(workspace);
  float* bpart = gb != nullptr ? part + static_cast<size_t>(p.nsplit) * Co * Ci : nullptr;
  // paired / quadruple accesses: even rows of gy, code rows of a multiple of four, aligned addresses
  const bool vec = Co % 2 == 0 && Ci % 4 == 0 && reinterpret_cast<uintptr_t>(gy) % (2 * sizeof(T)) == 0 && reinterpret_cast<uintptr_t>(codes) % 4 == 0;
  hipError_t e;
  if (p.nsplit > 0) {
    if (fmt == DBEV_ACT8_INT8)
      e = vec ? a8w_tiles<T, DBEV_ACT8_INT8, true>(p, gy, codes, scales, part, bpart, M, Co, Ci, st)
              : a8w_tiles<T, DBEV_ACT8_INT8, false>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
    else
      e = vec ? a8w_tiles<T, DBEV_ACT8_E4M3, true>(p, gy, codes, scales, part, bpart, M, Co, Ci, st)
              : a8w_tiles<T, DBEV_ACT8_E4M3, false>(p, gy, codes, scales, part, bpart, M, Co, Ci, st);
    if (e != hipSuccess) return static_cast<int>(e);
  }
  const long long plane = static_cast<long long>(Co) * Ci, n = plane + (gb != nullptr ? Co : 0);
  hipLaunchKernelGGL((a8_wsum<T>), dim3(static_cast<unsigned>((n + 255) / 256)), dim3(256), 0, st, part, bpart, p.nsplit, plane, Co, static_cast<T*>(gw),
                     static_cast<T*>(gb));
  DBEV_LAUNCH_CHECK();
  return 0;
}

}  // namespace

extern "C" size_t dbev_act8_weight_gradient_workspace_bytes(long long M, int Ci, int Co) {
  A8WPlan p;
  return a8w_plan(M, Ci, Co, &p) ? a8w_bytes(p, Ci, Co) + 16 : 0;
}

extern "C" int dbev_act8_weight_gradient(const void* gy, int dtype, const uint8_t* codes, const uint8_t* scales, int fmt, long long M, int Ci, int Co,
                                         void* gw, void* gb, void* workspace, size_t workspace_bytes, dbevStream_t stream) {
  A8WPlan p;
  if (!a8_dtype_ok(dtype) || !a8_fmt_ok(fmt) || !a8w_plan(M, Ci, Co, &p) || workspace_bytes < a8w_bytes(p, Ci, Co)) return DBEV_EINVAL;
  hipStream_t st = dbev_stream(stream);
  if (dtype == DBEV_DT_F32) return a8w_run<float>(p, gy, codes, scales, fmt, M, Ci, Co, gw, gb, workspace, st);
  if (dtype == DBEV_DT_BF16) return a8w_run<a8_bf16>(p, gy, codes, scales, fmt, M, Ci, Co, gw, gb, workspace, st);
  return a8w_run<a8_f16>(p, gy, codes, scales, fmt, M, Ci, Co, gw, gb, workspace, st);
}
