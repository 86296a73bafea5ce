// Device helpers shared by the 8-bit activation checkpoints (act8.hip, act8_wgrad.hip) and the group norm (gn_act.hip): typed vector
// access, the block quantiser, the activations and their derivatives.
//
// Checkpoint format: rows x C values, 32 neighbouring channels of a row (fewer in a row's last block) share one power of two 2^k, kept
// as the byte k + 127; a value is one byte, either a signed whole number (int8, -127..127) or an e4m3 float, times 2^k.
//   int8   k = floor(log2 amax) - 6: codes 64..127 at the top of the block, |x - x^| <= 2^(k-1) (2^k where the code is clamped to 127)
//   e4m3   k = floor(log2 amax) - 8, one more when amax > 448 * 2^k: no code saturates, |x - x^| <= 2^-4 |x| down to 2^(k-6).  Rounding up to
//          256 * 2^k can leave the type: fp16 values above 63488 restore as 2^16, an infinity in fp16, fp32's and bf16's above 248 * 2^120 as
//          2^128, an infinity.  (int8 rounds down to 127 * 2^k there)
// Multiplying by 2^-k is exact, so the one rounding (to nearest, ties to even) is the code itself and every correct implementation
// gives the same bytes; the restored value has at most 8 significant bits, i.e. it IS a bf16 number -- the weight gradient feeds it to
// the bf16 matrix cores unsplit.  A block that holds an infinity or a NaN gets the byte 255 and restores as NaN throughout: an overflow
// in the forward pass stays visible in the gradients.
#pragma once
#include "common.h"

typedef __bf16 a8_bf16;
typedef _Float16 a8_f16;

// V values of T as one naturally aligned access (V * sizeof(T) = 2..16 bytes); `Raw` keeps them as loaded (16-bit types: half the registers
// of their float values while other loads are in flight).  float -> T rounds to nearest even
template <typename T, int V>
struct A8Vec {
  typedef T vec __attribute__((ext_vector_type(V)));
  typedef float fvec __attribute__((ext_vector_type(V)));
  typedef vec Raw;
  // NT: without keeping the line in the caches (a8_nt)
  template <bool NT = false>
  static __device__ __forceinline__ Raw load(const T* p) {
    return NT ? __builtin_nontemporal_load(reinterpret_cast<const vec*>(p)) : *reinterpret_cast<const vec*>(p);
  }
  static __device__ __forceinline__ void get(const Raw& t, float* v) {
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = static_cast<float>(t[i]);
  }
  static __device__ __forceinline__ Raw zero() {
    Raw t;
#pragma unroll
    for (int i = 0; i < V; ++i) t[i] = static_cast<T>(0.f);
    return t;
  }
  template <bool NT = false>
  static __device__ __forceinline__ void store(T* p, const float* v) {
    fvec f;
#pragma unroll
    for (int i = 0; i < V; ++i) f[i] = v[i];
    if (NT) __builtin_nontemporal_store(__builtin_convertvector(f, vec), reinterpret_cast<vec*>(p));
    else *reinterpret_cast<vec*>(p) = __builtin_convertvector(f, vec);
  }
};
template <typename T>
struct A8Vec<T, 1> {
  typedef T Raw;
  template <bool NT = false>
  static __device__ __forceinline__ Raw load(const T* p) { return *p; }
  static __device__ __forceinline__ void get(const Raw& t, float* v) { v[0] = static_cast<float>(t); }
  static __device__ __forceinline__ Raw zero() { return static_cast<T>(0.f); }
  template <bool NT = false>
  static __device__ __forceinline__ void store(T* p, const float* v) { *p = static_cast<T>(v[0]); }
};

// V code bytes as one access
template <int V> struct A8Bytes;
template <> struct A8Bytes<1> { typedef uint8_t type; };
template <> struct A8Bytes<2> { typedef uint16_t type; };
template <> struct A8Bytes<4> { typedef uint32_t type; };
template <> struct A8Bytes<8> { typedef unsigned long long type; };

// the largest of `v` over the 32 / V lanes that hold one block (aligned groups of 4, 8, 16 or 32 lanes): DPP moves inside 16 lanes, no LDS
template <int V>
__device__ __forceinline__ unsigned a8_block_max(unsigned v) {
#define A8_DPP(ctrl_) v = max(v, static_cast<unsigned>(__builtin_amdgcn_mov_dpp(static_cast<int>(v), (ctrl_), 0xf, 0xf, true)))
  A8_DPP(0xB1);                                  // quad_perm [1,0,3,2]
  A8_DPP(0x4E);                                  // quad_perm [2,3,0,1]
  if (V <= 4) A8_DPP(0x141);                     // row_half_mirror: the other quad of 8 lanes
  if (V <= 2) A8_DPP(0x140);                     // row_mirror: the other half of 16 lanes
  if (V == 1) v = max(v, static_cast<unsigned>(__shfl_xor(static_cast<int>(v), 16)));
#undef A8_DPP
  return v;
}

// scale byte of a block from the bits of its largest |x| (as unsigned numbers: a NaN is above an infinity is above every finite value)
template <int FMT>
__device__ __forceinline__ unsigned a8_scale_byte(unsigned amax) {
  const unsigned e = amax >> 23;
  unsigned b;
  if (FMT == DBEV_ACT8_INT8) b = e > 6u ? e - 6u : 0u;
  else b = e >= 8u ? e - 8u + ((amax & 0x7fffffu) > 0x600000u ? 1u : 0u) : 0u;       // amax 2^-k > 448 = 1.75 * 2^8
  return e == 255u ? 255u : b;
}

// 2^k of a scale byte; 255 gives infinity, whose product with a zero code is the NaN that such a block restores as
__device__ __forceinline__ float a8_scale(unsigned byte) { return __builtin_ldexpf(1.f, static_cast<int>(byte) - 127); }

// V values of one block -> V codes (byte 255: zero codes)
template <int FMT, int V>
__device__ __forceinline__ typename A8Bytes<V>::type a8_encode(const float* v, unsigned byte) {
  const float inv = __uint_as_float((254u - byte) << 23);       // 2^-k; byte <= 248 for finite blocks
  unsigned long long r = 0;
  if (FMT == DBEV_ACT8_INT8) {
    // adding 1.5 * 2^23 rounds to a whole number (ties to even) and leaves it, two's complement, in the low bits
    constexpr float MAGIC = 12582912.f;
    unsigned q[V];
#pragma unroll
    for (int i = 0; i < V; ++i)
      q[i] = __float_as_uint(__builtin_amdgcn_fmed3f(fmaf(v[i], inv, MAGIC), MAGIC - 127.f, MAGIC + 127.f)) & 0xffu;
#pragma unroll
    for (int i = 0; i < V; ++i) r |= static_cast<unsigned long long>(q[i]) << (8 * i);
  } else {
#pragma unroll
    for (int i = 0; i < V; i += 2) {
      const unsigned p = static_cast<unsigned>(__builtin_amdgcn_cvt_pk_fp8_f32(v[i] * inv, V > 1 ? v[V > 1 ? i + 1 : i] * inv : 0.f, 0, false));
      r |= static_cast<unsigned long long>(p & (V > 1 ? 0xffffu : 0xffu)) << (8 * i);
    }
  }
  return static_cast<typename A8Bytes<V>::type>(byte == 255u ? 0ull : r);
}

// four codes (one dword) -> four values, exact (except that 2^-127 times a small code can be a subnormal, which fp32 holds exactly too)
template <int FMT>
__device__ __forceinline__ void a8_decode4(unsigned c, float s, float* v) {
  if (FMT == DBEV_ACT8_INT8) {
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = static_cast<float>(static_cast<int8_t>(c >> (8 * i))) * s;
  } else {
    typedef float f2 __attribute__((ext_vector_type(2)));
    const f2 lo = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c), false), hi = __builtin_amdgcn_cvt_pk_f32_fp8(static_cast<int>(c), true);
    v[0] = lo[0] * s;
    v[1] = lo[1] * s;
    v[2] = hi[0] * s;
    v[3] = hi[1] * s;
  }
}
template <int FMT, int V>
__device__ __forceinline__ void a8_decode(typename A8Bytes<V>::type c, float s, float* v) {
  if (V >= 4) {
#pragma unroll
    for (int i = 0; i < V; i += 4) a8_decode4<FMT>(static_cast<unsigned>(static_cast<unsigned long long>(c) >> (8 * i)), s, v + i);
  } else {
    float t[4];
    a8_decode4<FMT>(static_cast<unsigned>(c), s, t);
#pragma unroll
    for (int i = 0; i < V; ++i) v[i] = t[i];
  }
}

// ---- activations ------------------------------------------------------------------------------------------------------------------
// exp2 and the reciprocal are the hardware's (1 ulp).
__device__ __forceinline__ float a8_sigmoid(float z) { return __builtin_amdgcn_rcpf(1.f + __builtin_amdgcn_exp2f(-1.4426950408889634f * z)); }

// 1 - Phi(|z|) = exp(-z^2 / 2) * t R(t), t = 1 / (1 + p |z|): the form of Hastings' approximations to the error function, with coefficients of
// its own: R is a least-maximum fit, of degree 8, to erfcx / (2 t) over |z| <= 14.  Relative error 1.46e-7, 4.6e-7 with fp32 evaluation.  The
// same for every type: degree 5 (1.7e-5) for the 16-bit types put 1 % of fp16's results on the neighbouring value for 2 % of time (48 x 256 x
// 64 x 176 group norm, bf16: 161 us, now 165).  Returns t, R(t); e = exp(-z^2 / 2) serves the density of the derivative too.
__device__ __forceinline__ void a8_normal_tail(float z, float* e, float* t, float* r) {
  *t = __builtin_amdgcn_rcpf(fmaf(0.2828427124746192f, fabsf(z), 1.f));
  *e = __builtin_amdgcn_exp2f(z * z * -0.7213475204444817f);
  float p = fmaf(0.02512962929904461f, *t, -0.09144552052021027f);
  p = fmaf(p, *t, 0.08453510701656342f);
  p = fmaf(p, *t, -0.0027980783488601446f);
  p = fmaf(p, *t, 0.07071340829133987f);
  p = fmaf(p, *t, 0.08427148312330246f);
  p = fmaf(p, *t, 0.1039213016629219f);
  p = fmaf(p, *t, 0.11283480376005173f);
  p = fmaf(p, *t, 0.11283793300390244f);
  *r = p;
}

template <int ACT>
__device__ __forceinline__ float a8_act(float z) {
  if (ACT == DBEV_ACT_RELU) return z < 0.f ? 0.f : z;              // a NaN passes
  if (ACT == DBEV_ACT_SILU || ACT == DBEV_ACT_GELU) {
    // |z| (h - q), h = 1 for z > 0 and 0 otherwise, q = 1 - F(|z|) with F the sigmoid or the normal distribution: z F(z) without a difference
    // of like numbers, and where z > 0 the errors of exp2 and the reciprocal count with q / (1 - q) only; 1 - q, one multiply-add, and the
    // product are off by half a step each.  (SiLU as z times the reciprocal of 1 + exp(-z) is off by up to 1.5 2^-23 there, which put bf16's
    // 5.9375 -- 9.5e-8 from a tie -- on the wrong side; it takes three instructions less: 69633 x 1024 bf16 46.6 us, now 49.)  An infinity
    // below gives the NaN that z F(z) gives
    const float h = z > 0.f ? 1.f : 0.f;
    float e, u;                                                // q = e u
    if (ACT == DBEV_ACT_SILU) {
      e = __builtin_amdgcn_exp2f(-1.4426950408889634f * fabsf(z));
      u = __builtin_amdgcn_rcpf(1.f + e);
    } else {
      float t, r;
      a8_normal_tail(z, &e, &t, &r);
      u = t * r;
    }
    return fabsf(z) * fmaf(-e, u, h);
  }
  return z;
}

// g * act'(z); ReLU's derivative at 0 is 0.  GELU: Phi(z) + z phi(z) = h for z <= 0 and 1 - h for z > 0, h = 1 - Phi(|z|) - |z| phi(z).
template <int ACT>
__device__ __forceinline__ float a8_act_grad(float g, float z) {
  if (ACT == DBEV_ACT_RELU) return z > 0.f ? g : (z == z ? 0.f : z);
  if (ACT == DBEV_ACT_SILU) {
    const float s = a8_sigmoid(z);
    return g * (s * fmaf(z, 1.f - s, 1.f));
  }
  if (ACT == DBEV_ACT_GELU) {
    float e, t, r;
    a8_normal_tail(z, &e, &t, &r);
    const float h = e * fmaf(t, r, -0.3989422804014327f * fabsf(z));
    return g * (z > 0.f ? 1.f - h : h);
  }
  return g;
}

// ---- host-side dispatch over element type, vector width, format and activation -----------------------------------------------------
// vector widths: the widest of (16 bytes, 4 elements, 2, 1) that divides the row length and stride and that the base addresses are aligned to
// (40000 x 500 bf16, pack: 4 elements a lane instead of 2 18 -> 13 us)
static inline int a8_pick_vec(int esize, long long c, long long stride, const void* p0, const void* p1, const void* p2) {
  const uintptr_t a = reinterpret_cast<uintptr_t>(p0) | reinterpret_cast<uintptr_t>(p1) | reinterpret_cast<uintptr_t>(p2);
  const int wide = 16 / esize;
  for (int v : {wide, 4, 2})
    if (v <= wide && c % v == 0 && stride % v == 0 && a % (static_cast<uintptr_t>(v) * esize) == 0) return v;
  return 1;
}

// Tensors of more than 192 MB go past the memory-side cache (256 MB), which they would only wash out: with an operator that writes x before and
// one that reads y behind, fp32 SiLU with an int8 checkpoint, us kept / past: 81 MB 76 / 82, 163 MB 160 / 152 (backward 157 / 161), 266 MB
// 291 / 246 (292 / 257), 552 MB 603 / 558 (598 / 566).  16-byte accesses only.
static inline bool a8_nt(long long bytes) { return bytes > (192LL << 20); }
#define A8_NT_SWITCH(bytes_, ...)                                                        \
  if (V * sizeof(T) == 16 && a8_nt(bytes_)) { constexpr bool NT = V * sizeof(T) == 16; __VA_ARGS__; } \
  else { constexpr bool NT = false; __VA_ARGS__; }

#define A8_ACT_SWITCH(act_, ...)                                             \
  switch (act_) {                                                            \
    case DBEV_ACT_NONE: { constexpr int ACT = DBEV_ACT_NONE; __VA_ARGS__; break; } \
    case DBEV_ACT_RELU: { constexpr int ACT = DBEV_ACT_RELU; __VA_ARGS__; break; } \
    case DBEV_ACT_SILU: { constexpr int ACT = DBEV_ACT_SILU; __VA_ARGS__; break; } \
    default: { constexpr int ACT = DBEV_ACT_GELU; __VA_ARGS__; break; }            \
  }

#define A8_FMT_SWITCH(fmt_, ...)                                             \
  switch (fmt_) {                                                            \
    case DBEV_ACT8_INT8: { constexpr int FMT = DBEV_ACT8_INT8; __VA_ARGS__; break; } \
    case DBEV_ACT8_E4M3: { constexpr int FMT = DBEV_ACT8_E4M3; __VA_ARGS__; break; } \
    default: { constexpr int FMT = DBEV_ACT8_NONE; __VA_ARGS__; break; }             \
  }

#define A8_TYPE_SWITCH(dtype_, vec_, ...)                                    \
  switch (dtype_) {                                                          \
    case DBEV_DT_F32:                                                        \
      if ((vec_) == 4) { typedef float T; constexpr int V = 4; __VA_ARGS__; }       \
      else if ((vec_) == 2) { typedef float T; constexpr int V = 2; __VA_ARGS__; }  \
      else { typedef float T; constexpr int V = 1; __VA_ARGS__; }                   \
      break;                                                                 \
    case DBEV_DT_BF16:                                                       \
      if ((vec_) == 8) { typedef a8_bf16 T; constexpr int V = 8; __VA_ARGS__; }     \
      else if ((vec_) == 4) { typedef a8_bf16 T; constexpr int V = 4; __VA_ARGS__; } \
      else if ((vec_) == 2) { typedef a8_bf16 T; constexpr int V = 2; __VA_ARGS__; } \
      else { typedef a8_bf16 T; constexpr int V = 1; __VA_ARGS__; }                 \
      break;                                                                 \
    default:                                                                 \
      if ((vec_) == 8) { typedef a8_f16 T; constexpr int V = 8; __VA_ARGS__; }     \
      else if ((vec_) == 4) { typedef a8_f16 T; constexpr int V = 4; __VA_ARGS__; } \
      else if ((vec_) == 2) { typedef a8_f16 T; constexpr int V = 2; __VA_ARGS__; } \
      else { typedef a8_f16 T; constexpr int V = 1; __VA_ARGS__; }                  \
      break;                                                                 \
  }

static inline int a8_elem_size(int dtype) { return dtype == DBEV_DT_F32 ? 4 : 2; }
static inline bool a8_dtype_ok(int dtype) { return dtype == DBEV_DT_F32 || dtype == DBEV_DT_BF16 || dtype == DBEV_DT_F16; }
static inline bool a8_fmt_ok(int fmt) { return fmt == DBEV_ACT8_INT8 || fmt == DBEV_ACT8_E4M3; }
static inline bool a8_act_ok(int act) { return act >= DBEV_ACT_NONE && act <= DBEV_ACT_GELU; }

// A workgroup's view of a rows x C matrix: CH consecutive vector columns (a whole number of blocks of 32 channels) x RP row phases, a
// thread keeps one column; `ncol` workgroups side by side where the row is longer.
struct A8Tile { int CH, RP, ncol, threads; };
static inline A8Tile a8_tile(int C, int V) {
  const int lb = 32 / V, cv = (C + V - 1) / V;
  A8Tile t;
  t.ncol = (cv + 255) / 256;
  const int per = (cv + t.ncol - 1) / t.ncol;
  t.CH = (per + lb - 1) / lb * lb;
  t.ncol = (cv + t.CH - 1) / t.CH;
  t.RP = t.CH >= 256 ? 1 : 256 / t.CH;
  t.threads = (t.CH * t.RP + 63) / 64 * 64;
  return t;
}
