// Weight and bias gradient of a linear layer (or 1x1 convolution, channels-last) whose saved input is an 8-bit checkpoint (act8.h):
//   gw[Co, Ci] = sum_m gy[m, Co] * x^[m, Ci],   gb[Co] = sum_m gy[m, Co]
// on the bf16 matrix cores.  x^ = code * 2^k has at most 8 significant bits: it is a bf16 number, one operand plane.  gy is split exactly,
// by truncation, into as many bf16 pieces as its type has: three for fp32 (8 + 8 + 8 bits), two for fp16, one for bf16.  Every partial
// product is exact in fp32, the sums are fp32: fp32 accuracy for three matrix instructions where a product of two fp32 operands takes six.
//
// The reduction runs over m, the slow index of both operands, while a matrix instruction wants 8 consecutive m of one channel per lane:
// a thread fetches 8 rows of a few channels (coalesced along the channels), so that a channel's 8 values sit in its registers and go to
// LDS as one 16-byte unit [m / 8][channel]; the unit index is channel ^ ((channel >> 3) & 3), which spreads both the strided writes and
// the reads over all banks.  Raw values come through buffer descriptors of the chunk's rows: a row or channel past the end reads as zero.
//
// Workgroup = 4 waves, tile TA output x TB input channels, chunks of 32 rows, two LDS buffers, one barrier a chunk.  The largest tile, 128 x 256,
// has the register file to itself (one wave a SIMD): one tile of partial sums a CU.  A wave has two chunks of raw values in flight and splits
// the next chunk UNDER the current one's matrix instructions: a chunk is one basic block -- infinities, the last chunk and the bias sums are
// handled without branches -- cut into fenced steps of a few matrix instructions with some seven VALU behind each.  The rows are cut into
// shares, partial sums [share][Co][Ci] are added in a fixed order by a8_wsum: bit-reproducible, no atomics.
//
// Measured, fp32 gy (bf16 gy), both launches, int8: 40000 rows, 256 -> 512: 49 us (35); 33792, 1024 -> 256: 68 us (45); 540672, 64 -> 256: 137 us
// (76, 4.3 TB/s); the fp32 library product alone takes 470 us on the first: 42 + 6.5 us.  Its 20 chunks a share take 0.95 us each (0.64 of
// that matrix instructions at 2.4 GHz), 19 of the 42 us; the rest has not been taken apart: the launch's ramp, three cold fetches before the
// first chunk, and 128 KB a workgroup of partial sums in 4-byte stores, 33 MB that go out and come back.  16-bit gradients have a third or two
// thirds of the matrix work and half the bytes, but the same plan and so the same partial sums, more than their inputs: 35 us in bf16, where
// 51 MB of input take 10.  Two workgroups a CU (64 MB of partial sums): 43 + 12 us; tiles of 128 x 128: 61 us; two teams of waves on
// one tile, or the whole chunk ordered as one block: 44 us; four bytes a row of a lane's codes written with a swizzle by 16 channels: 330
// cycles of LDS conflicts a chunk, by 8: none.
#include "act8.h"

namespace {

typedef float floatx16 __attribute__((ext_vector_type(16)));
typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef unsigned uintx4 __attribute__((ext_vector_type(4)));

#define A8W_SGB(mask_, n_) __builtin_amdgcn_sched_group_barrier((mask_), (n_), 0)
constexpr int A8W_KC = 32;                                    // rows a chunk: two reduction steps of 16
constexpr unsigned A8W_OOB = 0x80000000u;                     // offset of a channel past the end: beyond every descriptor (32 rows of 2^20 values at most)

template <typename T> struct A8Pieces;
template <> struct A8Pieces<float> { static constexpr int n = 3; };
template <> struct A8Pieces<a8_f16> { static constexpr int n = 2; };
template <> struct A8Pieces<a8_bf16> { static constexpr int n = 1; };

__device__ __forceinline__ unsigned long long a8w_uniform(unsigned long long v) {
  const unsigned lo = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v)), hi = __builtin_amdgcn_readfirstlane(static_cast<unsigned>(v >> 32));
  return (static_cast<unsigned long long>(hi) << 32) | lo;
}
__device__ __forceinline__ __amdgpu_buffer_rsrc_t a8w_rsrc(const void* p, int bytes) {
  return __builtin_amdgcn_make_buffer_rsrc(reinterpret_cast<void*>(a8w_uniform(reinterpret_cast<unsigned long long>(p))), 0,
                                           __builtin_amdgcn_readfirstlane(bytes), 0x00020000);
}

// upper halves of two dwords: (hi(b) << 16) | hi(a)
__device__ __forceinline__ unsigned a8w_hi2(unsigned a, unsigned b) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// (a, b) -> NP dwords of two bf16 each, their sums are a and b exactly: truncation leaves the remainder exact.  The remainder of an infinity,
// inf - inf, is taken as 0, so that the products see inf and not a NaN.
template <int NP>
__device__ __forceinline__ void a8w_split(float a, float b, unsigned* p) {
  p[0] = a8w_hi2(__float_as_uint(a), __float_as_uint(b));
#pragma unroll
  for (int i = 1; i < NP; ++i) {
    const float ra = a - __uint_as_float(__float_as_uint(a) & 0xffff0000u), rb = b - __uint_as_float(__float_as_uint(b) & 0xffff0000u);
    a = i == 1 && __builtin_isinf(a) ? 0.f : ra;
    b = i == 1 && __builtin_isinf(b) ? 0.f : rb;
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
__global__ __launch_bounds__(256, TA * TB > 128 * 128 ? 1 : 2) void a8_wgrad(const T* __restrict__ gy, const uint8_t* __restrict__ codes, const uint8_t* __restrict__ scales,
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
  const int nrows = static_cast<int>(min(static_cast<long long>(rows_per), M - mbeg)), nch = (nrows + 2 * A8W_KC - 1) / (2 * A8W_KC) * 2;     // whole turns of the two register sets; rows past the end are zeros

  // staging role: rows 8 w .. 8 w + 7 of the chunk, channels CA lane .. of the gradient, CB lane .. of the checkpoint
  const T* gbase = gy + static_cast<size_t>(mbeg) * Co;
  const uint8_t* cbase = codes + static_cast<size_t>(mbeg) * Ci;
  const uint8_t* sbase = scales + static_cast<size_t>(mbeg) * nb;
  constexpr int EA = VEC ? 1 : CA, EB = VEC ? 1 : CB;         // separately addressed accesses per row
  unsigned aoff[8][EA], boff[8][EB], soff[8];
#pragma unroll
  for (int k = 0; k < 8; ++k) {
#pragma unroll
    for (int i = 0; i < EA; ++i) {
      const int c = co0 + CA * lane + i;
      aoff[k][i] = c < Co ? static_cast<unsigned>((8 * w + k) * Co + c) * sizeof(T) : A8W_OOB;
    }
#pragma unroll
    for (int i = 0; i < EB; ++i) {
      const int c = ci0 + CB * lane + i;
      boff[k][i] = c < Ci ? static_cast<unsigned>((8 * w + k) * Ci + c) : A8W_OOB;
    }
    soff[k] = ci0 + CB * lane < Ci ? static_cast<unsigned>((8 * w + k) * nb + (ci0 + CB * lane) / 32) : A8W_OOB;
  }
  struct Set { A8Raw<T, CA, VEC> a[8]; unsigned b[8], s[8]; };  // raw values of one chunk: CB code bytes and their block's scale byte (CB channels
                                                                // never straddle a block) per row
  Set set0, set1;
  float bsum[CA];
#pragma unroll
  for (int i = 0; i < CA; ++i) bsum[i] = 0.f;

  auto fetch_a = [&](Set& q, int ch) {                        // past the last row: empty descriptors, zeros
    const int r0 = ch * A8W_KC, left = max(0, min(A8W_KC, nrows - r0));
    const __amdgpu_buffer_rsrc_t gr = a8w_rsrc(gbase + static_cast<long long>(r0) * Co, left * Co * static_cast<int>(sizeof(T)));
#pragma unroll
    for (int k = 0; k < 8; ++k) q.a[k].load(gr, aoff[k]);
  };
  auto fetch_b = [&](Set& q, int ch) {
    const int r0 = ch * A8W_KC, left = max(0, min(A8W_KC, nrows - r0));
    const __amdgpu_buffer_rsrc_t cr = a8w_rsrc(cbase + static_cast<long long>(r0) * Ci, left * Ci);
    const __amdgpu_buffer_rsrc_t sr = a8w_rsrc(sbase + static_cast<long long>(r0) * nb, left * nb);
#pragma unroll
    for (int k = 0; k < 8; ++k) {
      if (VEC && CB == 4) q.b[k] = __builtin_amdgcn_raw_buffer_load_b32(cr, boff[k][0], 0, 0);
      else if (VEC && CB == 2) q.b[k] = static_cast<unsigned short>(__builtin_amdgcn_raw_buffer_load_b16(cr, boff[k][0], 0, 0));
      else {
        q.b[k] = 0;
#pragma unroll
        for (int i = 0; i < CB; ++i)
          q.b[k] |= static_cast<unsigned>(static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(cr, boff[k][VEC ? 0 : i], 0, 0))) << (8 * i);
      }
      q.s[k] = static_cast<uint8_t>(__builtin_amdgcn_raw_buffer_load_b8(sr, soff[k], 0, 0));
    }
  };

  // the staging of one chunk in NU pieces: 4 CA pieces split a pair of rows of one gradient channel, 8 decode a row's codes, CB pair a channel's
  // rows up and write them; the gradient channels are written behind their fourth piece
  constexpr int NU = 4 * CA + 8 + CB;
  unsigned pa[4][3];
  float xb[8][4];
  auto piece = [&](int u, const Set& q, unsigned char* buf) {
    if (u < 4 * CA) {
      const int c = u / 4, k = u % 4;
      const float a = q.a[2 * k].get(c), b = q.a[2 * k + 1].get(c);
      a8w_split<NP>(a, b, pa[k]);
      bsum[c] += a + b;
      if (k == 3) {
        const int row = CA * lane + c;
        unsigned char* d = buf + (w * TA + (row ^ ((row >> 3) & 3))) * 16;
#pragma unroll
        for (int i = 0; i < NP; ++i) *reinterpret_cast<uintx4*>(d + i * PLA) = uintx4{pa[0][i], pa[1][i], pa[2][i], pa[3][i]};
      }
    } else if (u < 4 * CA + 8) {
      const int k = u - 4 * CA;
      a8_decode4<FMT>(q.b[k], a8_scale(q.s[k]), xb[k]);
    } else {
      const int c = u - 4 * CA - 8, row = CB * lane + c;
      uintx4 v;
#pragma unroll
      for (int k = 0; k < 4; ++k) v[k] = a8w_hi2(__float_as_uint(xb[2 * k][c]), __float_as_uint(xb[2 * k + 1][c]));     // exact: bf16 numbers
      *reinterpret_cast<uintx4*>(buf + NP * PLA + (w * TB + (row ^ ((row >> 3) & 3))) * 16) = v;
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
    aaddr[a] = (half * TA + (r ^ ((r >> 3) & 3))) * 16;
  }
#pragma unroll
  for (int b = 0; b < NB; ++b) {
    const int r = (wn * NB + b) * 32 + l31;
    baddr[b] = NP * PLA + (half * TB + (r ^ ((r >> 3) & 3))) * 16;
  }

  constexpr int MF = 2 * NP * NA * NB;                        // matrix instructions of a chunk
  // chunk `ch` from buffer `par`; `next` (chunk ch + 1) is staged into the other buffer, a piece between every few matrix
  // instructions, and refilled with chunk ch + 3.  Steps are fenced off and ordered one by one: matrix instruction, some seven VALU (its 32
  // cycles), and so on -- as one block of 48 the scheduler lost the order (MFMA busy 35 %, VALU 30 %, hardly overlapping).
  auto chunk = [&](int ch, int par, Set& next) {
    const unsigned char* rd = smem + par * BUF;
    unsigned char* wr = smem + (par ^ 1) * BUF;
    bf16x8 af[2][NA][NP], bf[2][NB];
    auto operands = [&](int s) {
#pragma unroll
      for (int b = 0; b < NB; ++b) bf[s][b] = *reinterpret_cast<const bf16x8*>(rd + baddr[b] + s * 2 * TB * 16);
#pragma unroll
      for (int p = NP - 1; p >= 0; --p)
#pragma unroll
        for (int a = 0; a < NA; ++a) af[s][a][p] = *reinterpret_cast<const bf16x8*>(rd + p * PLA + aaddr[a] + s * 2 * TA * 16);
    };
    operands(0);
    piece(0, next, wr);
    __builtin_amdgcn_sched_barrier(0);
#pragma unroll
    for (int u = 1; u < NU + 1; ++u) {
      if (u == NU / 4) operands(1);
      const int m0 = (u - 1) * MF / NU, m1 = u * MF / NU;
#pragma unroll
      for (int m = m0; m < m1; ++m) {                         // the smallest pieces first
        const int st = m / (MF / 2), r = m % (MF / 2), p = NP - 1 - r / (NA * NB), a = r % (NA * NB) / NB, b = r % NB;
        acc[a][b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(af[st][a][p], bf[st][b], acc[a][b], 0, 0, 0);
      }
      if (u < NU) piece(u, next, wr);
      if (u == 4 * CA) fetch_a(next, ch + 3);
      if (u == NU) fetch_b(next, ch + 3);
#pragma unroll
      for (int m = m0; m < m1; ++m) {
        A8W_SGB(0x008, 1);
        A8W_SGB(0x002, 7);
      }
      __builtin_amdgcn_sched_barrier(0);
    }
    __syncthreads();
    __builtin_amdgcn_sched_barrier(0);
  };

  fetch_a(set0, 0);
  fetch_b(set0, 0);
  fetch_a(set1, 1);
  fetch_b(set1, 1);
#pragma unroll
  for (int u = 0; u < NU; ++u) piece(u, set0, smem);
  fetch_a(set0, 2);
  fetch_b(set0, 2);
  __syncthreads();
  __builtin_amdgcn_sched_barrier(0);
  // (two bodies: with three sets and two buffers six bodies and a rest were 35 KB of code, and fetching it took longer than the chunks)
  for (int ch = 0; ch < nch; ch += 2) {
    chunk(ch, 0, set1);
    chunk(ch + 1, 1, set0);
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
  if (bpart != nullptr && ci0 == 0) {                         // the four waves' rows of every channel, in order (smem is free behind the last barrier)
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
  float c0 = 0.f, c1 = 0.f, c2 = 0.f, c3 = 0.f;
  for (int s = 0; s < nsplit; s += 16) {                       // sixteen loads in flight, four chains
    float v[16];
#pragma unroll
    for (int i = 0; i < 16; ++i) v[i] = s + i < nsplit ? p[(s + i) * step] : 0.f;
#pragma unroll
    for (int i = 0; i < 16; i += 4) {
      c0 += v[i];
      c1 += v[i + 1];
      c2 += v[i + 2];
      c3 += v[i + 3];
    }
  }
  (isb ? gb[idx - plane] : gw[idx]) = static_cast<T>((c0 + c1) + (c2 + c3));
}

struct A8WPlan { int ta, tb, tiles_n, tiles, rows_per, nsplit, grid; };

bool a8w_plan(long long M, int Ci, int Co, A8WPlan* p) {
  // up to 2^20 channels (a chunk's 32 rows are one descriptor) and 2^31 weights (a launch holds fewer than 2^32 threads)
  if (M < 0 || Ci <= 0 || Co <= 0 || Ci > (1 << 20) || Co > (1 << 20) || static_cast<long long>(Ci) * Co > (1LL << 31) ||
      M > (1LL << 40) / (Ci > Co ? Ci : Co))
    return false;
  p->ta = Co > 64 ? 128 : 64;
  p->tb = Ci > 128 ? 256 : Ci > 64 ? 128 : 64;
  p->tiles_n = (Ci + p->tb - 1) / p->tb;
  p->tiles = (Co + p->ta - 1) / p->ta * p->tiles_n;
  long long ns = (p->ta * p->tb > 128 * 128 ? 256 : 512) / p->tiles;    // one workgroup a CU of the largest tile, two of the others
  const long long most = (M + 127) / 128;                     // at least four chunks a share
  ns = ns > most ? most : ns;
  ns = ns < 1 ? 1 : ns;
  constexpr long long cap = 1LL << 30;                        // rows of a share are counted in 32 bits
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
