// 8-bit activation checkpoints: an activation that the backward pass needs is kept as one byte per value + one scale byte per 32
// channels (format and rounding: act8.h) instead of as 2 or 4 bytes per value -- 1.03 / 4 of an fp32 tensor.
//   a8_pack      x -> codes, scales                        reads n * es, writes 1.03 n bytes
//   a8_unpack    codes, scales -> x^                       the reverse
//   a8_act_fwd   y = act(x), and x's checkpoint            reads n * es, writes n * es + 1.03 n: the checkpoint costs no pass of its own
//   a8_act_bwd   dx = dy * act'(x^)                        reads n * es + 1.03 n, writes n * es
// All four are bound by HBM traffic: 5.5 to 7.3 TB/s of the bytes above on 70 to 280 million values, where a copy reaches 5.1 to 5.4 (270000 x 512
// fp32, us: pack 107, unpack 96, SiLU forward 183, backward 185; GELU 184 / 202), but for GELU in 16-bit types, which VALU work holds
// (69633 x 1024 bf16: SiLU 65 / 67, GELU 66 / 79; 540000 x 512: 236 / 222, 242 / 262).
// A lane holds 16 bytes of a row (4, 2 or 1 elements where the row length, the stride or an address is off), the 32 channels of a block are
// 4 (16-bit types) or 8 (fp32) neighbouring lanes and their maximum is taken with DPP moves; a thread keeps its column and handles A8_U
// rows, all loads first.  Dense rows of a multiple of 32 channels are walked as rows of 32: every access of a wave is then one contiguous
// piece whatever C is.
#include "act8.h"

namespace {

constexpr int A8_U = 2;                                        // rows per thread: with 4 the large shapes are 1 to 3 % slower, with 8 5 %

constexpr int A8_GRID_Y = 1 << 16;                             // workgroups along y end here: beyond, the column ranges go along x, the rows along y

struct A8Pos { int col; bool on; long long row0, step; };

// column of this thread, its first row and the distance of its rows
__device__ __forceinline__ A8Pos a8_pos(const A8Tile& t, int cv) {
  A8Pos p;
  const int rp = threadIdx.x / t.CH;
  const unsigned by = t.ncol < A8_GRID_Y ? blockIdx.x : blockIdx.y, bc = t.ncol < A8_GRID_Y ? blockIdx.y : blockIdx.x;
  p.col = static_cast<int>(bc) * t.CH + (threadIdx.x - rp * t.CH);
  p.on = rp < t.RP && p.col < cv;
  p.row0 = rp < t.RP ? static_cast<long long>(by) * (t.RP * A8_U) + rp : (1LL << 62);
  p.step = t.RP;
  return p;
}

template <typename T, int V, int FMT, int ACT, bool WITH_Y, bool NT>
__global__ __launch_bounds__(256) void a8_forward(const T* __restrict__ x, long long xs, long long rows, int cv, int nb, A8Tile t, T* __restrict__ y,
                                                  uint8_t* __restrict__ codes, uint8_t* __restrict__ scales) {
  constexpr int LB = 32 / V;
  const A8Pos p = a8_pos(t, cv);
  typename A8Vec<T, V>::Raw raw[A8_U];
#pragma unroll
  for (int u = 0; u < A8_U; ++u) {
    const long long r = p.row0 + u * p.step;
    raw[u] = p.on && r < rows ? A8Vec<T, V>::template load<NT>(x + r * xs + static_cast<long long>(p.col) * V) : A8Vec<T, V>::zero();
  }
#pragma unroll
  for (int u = 0; u < A8_U; ++u) {
    const long long r = p.row0 + u * p.step;
    if (r >= rows) break;                                      // all lanes of a block are on the same row
    const long long o = (r * cv + p.col) * V;
    float v[V];
    A8Vec<T, V>::get(raw[u], v);
    if (FMT != DBEV_ACT8_NONE) {
      unsigned m = 0;
#pragma unroll
      for (int i = 0; i < V; ++i) m = max(m, __float_as_uint(v[i]) & 0x7fffffffu);
      const unsigned b = a8_scale_byte<FMT>(a8_block_max<V>(m));
      if (p.on) {
        *reinterpret_cast<typename A8Bytes<V>::type*>(codes + o) = a8_encode<FMT, V>(v, b);
        if (p.col % LB == 0) scales[r * nb + p.col / LB] = static_cast<uint8_t>(b);
      }
    }
    if (WITH_Y && p.on) {
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = a8_act<ACT>(v[i]);
      A8Vec<T, V>::template store<NT>(y + o, v);
    }
  }
}

// out = x^ (ACT none, gy null) or gy * act'(x^)
template <typename T, int V, int FMT, int ACT, bool WITH_GY, bool NT>
__global__ __launch_bounds__(256) void a8_backward(const T* __restrict__ gy, long long gs, const uint8_t* __restrict__ codes,
                                                   const uint8_t* __restrict__ scales, long long rows, int cv, int nb, A8Tile t, T* __restrict__ out) {
  constexpr int LB = 32 / V;
  const A8Pos p = a8_pos(t, cv);
  if (!p.on) return;
  typename A8Bytes<V>::type c[A8_U];
  unsigned b[A8_U];
  typename A8Vec<T, V>::Raw graw[A8_U];
#pragma unroll
  for (int u = 0; u < A8_U; ++u) {
    const long long r = p.row0 + u * p.step;
    if (r < rows) {
      c[u] = *reinterpret_cast<const typename A8Bytes<V>::type*>(codes + (r * cv + p.col) * V);
      b[u] = scales[r * nb + p.col / LB];
      if (WITH_GY) graw[u] = A8Vec<T, V>::template load<NT>(gy + r * gs + static_cast<long long>(p.col) * V);
    }
  }
#pragma unroll
  for (int u = 0; u < A8_U; ++u) {
    const long long r = p.row0 + u * p.step;
    if (r >= rows) break;
    float v[V];
    a8_decode<FMT, V>(c[u], a8_scale(b[u]), v);
    if (WITH_GY) {
      float g[V];
      A8Vec<T, V>::get(graw[u], g);
#pragma unroll
      for (int i = 0; i < V; ++i) v[i] = a8_act_grad<ACT>(g[i], v[i]);
    }
    A8Vec<T, V>::template store<NT>(out + (r * cv + p.col) * V, v);
  }
}

struct A8Geo { long long rows, stride; int C, nb; };

// dense rows of whole blocks are rows of 32 channels
A8Geo a8_geo(long long rows, int C, long long stride) {
  if (C % 32 == 0 && stride == C) return A8Geo{rows * (C / 32), 32, 32, 1};
  return A8Geo{rows, stride, C, (C + 31) / 32};
}

bool a8_shape_ok(int dtype, long long rows, int C, long long stride) {
  // (element offsets are 64-bit in the kernels)
  return a8_dtype_ok(dtype) && rows >= 0 && C > 0 && stride >= C && C <= (1 << 30) && rows <= (1LL << 40) / C && stride <= (1LL << 40) / (rows + 1);
}

long long a8_blocks(const A8Geo& g, const A8Tile& t) {
  const long long per = static_cast<long long>(t.RP) * A8_U;
  return (g.rows + per - 1) / per;
}
// a launch holds fewer than 2^32 threads along x (some 2^34 values or more, by vector width)
bool a8_grid_ok(const A8Geo& g, const A8Tile& t) {
  const long long b = a8_blocks(g, t);
  return t.ncol < A8_GRID_Y ? b * t.threads < (1LL << 32) : b < A8_GRID_Y;
}
long long a8_bytes(const A8Geo& g, size_t esize) { return g.rows * g.C * static_cast<long long>(esize); }
dim3 a8_grid(const A8Geo& g, const A8Tile& t) {
  const unsigned b = static_cast<unsigned>(a8_blocks(g, t)), c = static_cast<unsigned>(t.ncol);
  return t.ncol < A8_GRID_Y ? dim3(b, c) : dim3(c, b);
}

}  // namespace

extern "C" int dbev_act8_pack(const void* x, int dtype, long long rows, int C, long long row_stride, int fmt, uint8_t* codes, uint8_t* scales,
                              dbevStream_t stream) {
  if (!a8_shape_ok(dtype, rows, C, row_stride) || !a8_fmt_ok(fmt)) return DBEV_EINVAL;
  if (rows == 0) return 0;
  const A8Geo g = a8_geo(rows, C, row_stride);
  const int vec = a8_pick_vec(a8_elem_size(dtype), g.C, g.stride, x, nullptr, nullptr);
  A8_TYPE_SWITCH(dtype, vec, {
    const A8Tile t = a8_tile(g.C, V);
    if (reinterpret_cast<uintptr_t>(codes) % V != 0 || !a8_grid_ok(g, t)) return DBEV_EINVAL;
    A8_NT_SWITCH(a8_bytes(g, sizeof(T)), {
      if (fmt == DBEV_ACT8_INT8)
        hipLaunchKernelGGL((a8_forward<T, V, DBEV_ACT8_INT8, DBEV_ACT_NONE, false, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           static_cast<const T*>(x), g.stride, g.rows, g.C / V, g.nb, t, nullptr, codes, scales);
      else
        hipLaunchKernelGGL((a8_forward<T, V, DBEV_ACT8_E4M3, DBEV_ACT_NONE, false, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           static_cast<const T*>(x), g.stride, g.rows, g.C / V, g.nb, t, nullptr, codes, scales);
    });
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}

extern "C" int dbev_act8_unpack(const uint8_t* codes, const uint8_t* scales, int fmt, long long rows, int C, void* out, int dtype, dbevStream_t stream) {
  if (!a8_shape_ok(dtype, rows, C, C) || !a8_fmt_ok(fmt)) return DBEV_EINVAL;
  if (rows == 0) return 0;
  const A8Geo g = a8_geo(rows, C, C);
  const int vec = a8_pick_vec(a8_elem_size(dtype), g.C, g.stride, out, nullptr, nullptr);
  A8_TYPE_SWITCH(dtype, vec, {
    const A8Tile t = a8_tile(g.C, V);
    if (reinterpret_cast<uintptr_t>(codes) % V != 0 || !a8_grid_ok(g, t)) return DBEV_EINVAL;
    A8_NT_SWITCH(a8_bytes(g, sizeof(T)), {
      if (fmt == DBEV_ACT8_INT8)
        hipLaunchKernelGGL((a8_backward<T, V, DBEV_ACT8_INT8, DBEV_ACT_NONE, false, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           nullptr, g.stride, codes, scales, g.rows, g.C / V, g.nb, t, static_cast<T*>(out));
      else
        hipLaunchKernelGGL((a8_backward<T, V, DBEV_ACT8_E4M3, DBEV_ACT_NONE, false, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           nullptr, g.stride, codes, scales, g.rows, g.C / V, g.nb, t, static_cast<T*>(out));
    });
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}

extern "C" int dbev_act8_activation_forward(const void* x, int dtype, long long rows, int C, long long row_stride, int act, int fmt, void* y,
                                            uint8_t* codes, uint8_t* scales, dbevStream_t stream) {
  if (!a8_shape_ok(dtype, rows, C, row_stride) || !(fmt == DBEV_ACT8_NONE || a8_fmt_ok(fmt)) || !a8_act_ok(act)) return DBEV_EINVAL;
  if (rows == 0) return 0;
  const A8Geo g = a8_geo(rows, C, row_stride);
  const int vec = a8_pick_vec(a8_elem_size(dtype), g.C, g.stride, x, y, nullptr);
  A8_TYPE_SWITCH(dtype, vec, {
    const A8Tile t = a8_tile(g.C, V);
    if ((fmt != DBEV_ACT8_NONE && reinterpret_cast<uintptr_t>(codes) % V != 0) || !a8_grid_ok(g, t)) return DBEV_EINVAL;
    A8_NT_SWITCH(a8_bytes(g, sizeof(T)), A8_ACT_SWITCH(act, A8_FMT_SWITCH(fmt, {
      hipLaunchKernelGGL((a8_forward<T, V, FMT, ACT, true, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream), static_cast<const T*>(x),
                         g.stride, g.rows, g.C / V, g.nb, t, static_cast<T*>(y), codes, scales);
    })));
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}

extern "C" int dbev_act8_activation_backward(const void* gy, int dtype, long long gy_row_stride, const uint8_t* codes, const uint8_t* scales, int fmt,
                                             long long rows, int C, int act, void* dx, dbevStream_t stream) {
  if (!a8_shape_ok(dtype, rows, C, gy_row_stride) || !a8_fmt_ok(fmt) || !a8_act_ok(act)) return DBEV_EINVAL;
  if (rows == 0) return 0;
  const A8Geo g = a8_geo(rows, C, gy_row_stride);
  const int vec = a8_pick_vec(a8_elem_size(dtype), g.C, g.stride, gy, dx, nullptr);
  A8_TYPE_SWITCH(dtype, vec, {
    const A8Tile t = a8_tile(g.C, V);
    if (reinterpret_cast<uintptr_t>(codes) % V != 0 || !a8_grid_ok(g, t)) return DBEV_EINVAL;
    A8_NT_SWITCH(a8_bytes(g, sizeof(T)), A8_ACT_SWITCH(act, {
      if (fmt == DBEV_ACT8_INT8)
        hipLaunchKernelGGL((a8_backward<T, V, DBEV_ACT8_INT8, ACT, true, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           static_cast<const T*>(gy), g.stride, codes, scales, g.rows, g.C / V, g.nb, t, static_cast<T*>(dx));
      else
        hipLaunchKernelGGL((a8_backward<T, V, DBEV_ACT8_E4M3, ACT, true, NT>), a8_grid(g, t), dim3(t.threads), 0, dbev_stream(stream),
                           static_cast<const T*>(gy), g.stride, codes, scales, g.rows, g.C / V, g.nb, t, static_cast<T*>(dx));
    }));
  });
  DBEV_LAUNCH_CHECK();
  return 0;
}
