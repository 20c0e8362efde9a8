// qk_norm_rope.hip — the norms of queries and keys for each head and the
// position rotation in one pass over the rows, and their gradients.
//
// Bound by HBM: every value is read and written once. A head's row lies
// across 4 to 32 lanes, 8 values (16 bytes of a 16-bit type) each; its sums
// are shuffles inside those lanes, and a rotation by halves takes its other
// value from the lane rot / 16 away. A lane keeps its angles and gammas in
// registers over the heads of a row. All arithmetic is in 32 bits; a result
// is rounded once. Measured: 72,500 rows of 12+12 heads of 64, bf16, 95 us,
// 4.7 TB/s (the card's copy 4.9); 16,384 rows of 16+4 heads of 128, float16,
// forward and gradients 101 us, 4.2 TB/s; 15 rows 3.8 us, the launch.
#include "attend_device.h"
#include "ixh_internal.h"

namespace ixh {
namespace {

constexpr int kThreads = 256;

template <class F>
__device__ __forceinline__ void unpack(const F &f, float *x) {
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] = frag_at(f, e);
}

// v and the value of another lane of the same 16, by a DPP pattern.
template <int CTRL>
__device__ __forceinline__ float add_dpp(float v) {
  const int o = __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), CTRL, 0xf, 0xf, true);
  return v + __builtin_bit_cast(float, o);
}
// The sum over LANES lanes, in each of them: neighbours, pairs, then halves
// and rows of 16 mirrored.
template <int LANES>
__device__ __forceinline__ float lanes_sum(float v) {
  v = add_dpp<0xb1>(v);   // quad_perm 1 0 3 2
  v = add_dpp<0x4e>(v);   // quad_perm 2 3 0 1
  if constexpr (LANES >= 8) v = add_dpp<0x141>(v);   // row_half_mirror
  if constexpr (LANES >= 16) v = add_dpp<0x140>(v);  // row_mirror
  if constexpr (LANES == 32) v += __shfl_xor(v, 16);
  return v;
}

// The lane's 8 columns of one row: whether they are there, and their angles.
template <int LANES>
struct Lane {
  int c;          // first column
  bool in;        // c < dim
  float co[8], si[8];
  int other;      // lane offset to the rotation's other half; 0: none

  __device__ __forceinline__ Lane(const ixh_norm_rope_args &a, int64_t row, int l) {
    c = 8 * l;
    in = c < a.dim;
    const int half = a.rot / 2;
    const int pos = a.pos ? a.pos[row] : (int)row;
    const bool there = pos >= 0 && pos < a.rows;  // else the angle has no row: NaN
    const bool halves = a.pairs == IXH_PAIRS_HALVES;
    other = !halves || c >= a.rot ? 0 : c < half ? half / 8 : -(half / 8);
#pragma unroll
    for (int e = 0; e < 8; e++) co[e] = 1.0f, si[e] = 0.0f;
    if (c < a.rot) {
      const float bad = __builtin_nanf("");
      if (halves) {
        // first half a c - b s, second b c + a s: the sign goes with the sine
        const int at = c < half ? c : c - half;
        const float *ct = a.cos + (int64_t)(there ? pos : 0) * half + at, *st = a.sin + (int64_t)(there ? pos : 0) * half + at;
#pragma unroll
        for (int e = 0; e < 8; e++) {
          co[e] = there ? ct[e] : bad;
          si[e] = c < half ? -st[e] : st[e];
        }
      } else {
        const float *ct = a.cos + (int64_t)(there ? pos : 0) * half, *st = a.sin + (int64_t)(there ? pos : 0) * half;
#pragma unroll
        for (int e = 0; e < 8; e += 2)
          if (c + e < a.rot) {
            const float cs = there ? ct[(c + e) / 2] : bad, sn = st[(c + e) / 2];
            co[e] = co[e + 1] = cs;
            si[e] = -sn;
            si[e + 1] = sn;
          }
      }
    }
  }
  // x rotated, by the opposite angle where sign is -1.
  __device__ __forceinline__ void turn(const ixh_norm_rope_args &a, float *x, float sign) const {
    if (a.rot == 0) return;
    float o[8];
    if (a.pairs == IXH_PAIRS_HALVES) {
      const int from = (int)__lane_id() + other;
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = __shfl(x[e], from);
    } else {
#pragma unroll
      for (int e = 0; e < 8; e++) o[e] = x[e ^ 1];
    }
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = __builtin_fmaf(x[e], co[e], o[e] * (sign * si[e]));
  }
};

__device__ __forceinline__ void load_gamma(const ixh_norm_rope_args &a, const void *p, int c, bool in, float *g) {
#pragma unroll
  for (int e = 0; e < 8; e++) g[e] = 1.0f;
  if (!p || !in) return;
  if (a.gamma_type == IXH_TYPE_F32)
    unpack(*(const v8f *)((const float *)p + c), g);
  else if (a.gamma_type == IXH_TYPE_BF16)
    unpack(*(const v8bf *)((const __bf16 *)p + c), g);
  else
    unpack(*(const v8h *)((const _Float16 *)p + c), g);
}

// x centred and scaled in place; the scale. Columns past dim hold 0 and stay.
template <int LANES, int NORM>
__device__ __forceinline__ float normalise(const ixh_norm_rope_args &a, float *x, bool in) {
  if constexpr (NORM == IXH_HEAD_NORM_NONE) return 1.0f;
  const float inv = 1.0f / (float)a.dim;
  if constexpr (NORM == IXH_HEAD_NORM_LAYER) {
    float s = 0.0f;
#pragma unroll
    for (int e = 0; e < 8; e++) s += x[e];
    const float mean = lanes_sum<LANES>(s) * inv;
#pragma unroll
    for (int e = 0; e < 8; e++) x[e] = in ? x[e] - mean : 0.0f;
  }
  float q = 0.0f;
#pragma unroll
  for (int e = 0; e < 8; e++) q = __builtin_fmaf(x[e], x[e], q);
  const float r = 1.0f / __builtin_sqrtf(__builtin_fmaf(lanes_sum<LANES>(q), inv, (float)a.eps));
#pragma unroll
  for (int e = 0; e < 8; e++) x[e] *= r;
  return r;
}

// A group of LANES lanes has one row and heads_step of its heads, Q's before
// K's. x: the arrays as one list of heads.
template <class T, int LANES, int NORM>
__global__ __launch_bounds__(kThreads) void norm_rope_kernel(NormRopeArgs x) {
  typedef typename Kind<T>::frag Frag;
  const ixh_norm_rope_args &a = x.a;
  const int l = threadIdx.x % LANES;
  const int64_t row0 = (int64_t)blockIdx.x * (kThreads / LANES) + threadIdx.x / LANES;
  const int64_t row = min(row0, (int64_t)a.n - 1);
  const bool mine = row0 < a.n;
  const Lane<LANES> ln(a, row, l);
  const int h0 = blockIdx.y * x.heads_step, h1 = min(h0 + x.heads_step, a.q_heads + a.k_heads);
  auto run = [&](const ixh_heads &from, const ixh_heads &to, const void *gamma, int g0, int g1) {
    if (g0 >= g1) return;
    float g[8];
    load_gamma(a, gamma, ln.c, ln.in, g);
    const T *src = (const T *)from.p + row * from.row + ln.c;
    T *dst = (T *)to.p + row * to.row + ln.c;
    auto one = [&](const Frag &f, int h) {
      float y[8];
      unpack(f, y);
      normalise<LANES, NORM>(a, y, ln.in);
#pragma unroll
      for (int e = 0; e < 8; e++) y[e] *= g[e];
      ln.turn(a, y, 1.0f);
      if (mine && ln.in) *(Frag *)(dst + h * to.head) = pack8<Frag>(y);
    };
    int h = g0;
    for (; h + 4 <= g1; h += 4) {  // four rows' loads in flight
      Frag f[4];
#pragma unroll
      for (int i = 0; i < 4; i++) f[i] = load8(src + (h + i) * from.head, ln.in);
#pragma unroll
      for (int i = 0; i < 4; i++) one(f[i], h + i);
    }
    for (; h < g1; h++) one(load8(src + h * from.head, ln.in), h);
  };
  run(a.q, a.q_out, a.q_gamma, h0, min(h1, a.q_heads));
  run(a.k, a.k_out, a.k_gamma, max(h0 - a.q_heads, 0), h1 - a.q_heads);
}

// The gradients. A lane adds up its columns' gamma gradients over its rows
// and heads; the workgroup's groups meet in LDS, the workgroups in
// norm_rope_gamma_kernel, each in a fixed order. Three waves a SIMD, for
// loads in flight (16,384 rows of 16+4 heads of 128, float16: 55 us).
template <class T, int LANES, int NORM>
__global__ __launch_bounds__(kThreads, sizeof(T) == 2 ? 3 : 2) void norm_rope_backward_kernel(NormRopeArgs x) {
  typedef typename Kind<T>::frag Frag;
  const ixh_norm_rope_args &a = x.a;
  constexpr int GROUPS = kThreads / LANES;
  __shared__ float meet[kThreads * 8];
  const int l = threadIdx.x % LANES, grp = threadIdx.x / LANES;
  const int h0 = blockIdx.y * x.heads_step, h1 = min(h0 + x.heads_step, a.q_heads + a.k_heads);
  const float inv = 1.0f / (float)a.dim;
  float gsum[2][8] = {};
  for (int64_t base = (int64_t)blockIdx.x * GROUPS; base < a.n; base += (int64_t)x.blocks * GROUPS) {
    const int64_t row = min(base + grp, (int64_t)a.n - 1);
    const bool mine = base + grp < a.n;
    const Lane<LANES> ln(a, row, l);
    auto run = [&](const ixh_heads &from, const ixh_heads &grad, const ixh_heads &to, const void *gamma, int g0, int g1,
                   float *gs) {
      if (g0 >= g1) return;
      float g[8];
      load_gamma(a, gamma, ln.c, ln.in, g);
      const T *src = (const T *)from.p + row * from.row + ln.c;
      const T *gsrc = (const T *)grad.p + row * grad.row + ln.c;
      T *dst = (T *)to.p + row * to.row + ln.c;
      auto one = [&](const Frag &f, const Frag &df, int h) {
        float xh[8], d[8];
        unpack(f, xh);
        unpack(df, d);
        const float r = normalise<LANES, NORM>(a, xh, ln.in);
        ln.turn(a, d, -1.0f);
        if constexpr (NORM != IXH_HEAD_NORM_NONE) {
          float dot = 0.0f, s = 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) {
            if (mine) gs[e] = __builtin_fmaf(d[e], xh[e], gs[e]);
            d[e] *= g[e];
            dot = __builtin_fmaf(d[e], xh[e], dot);
            s += d[e];
          }
          dot = lanes_sum<LANES>(dot) * inv;
          s = NORM == IXH_HEAD_NORM_LAYER ? lanes_sum<LANES>(s) * inv : 0.0f;
#pragma unroll
          for (int e = 0; e < 8; e++) d[e] = (__builtin_fmaf(-xh[e], dot, d[e]) - s) * r;
        } else {
#pragma unroll
          for (int e = 0; e < 8; e++) {
            if (mine) gs[e] = __builtin_fmaf(d[e], xh[e], gs[e]);
            d[e] *= g[e];
          }
        }
        if (mine && ln.in) *(Frag *)(dst + h * to.head) = pack8<Frag>(d);
      };
      int h = g0;
      for (; h + 2 <= g1; h += 2) {
        Frag f[2], df[2];
#pragma unroll
        for (int i = 0; i < 2; i++) {
          f[i] = load8(src + (h + i) * from.head, ln.in);
          df[i] = load8(gsrc + (h + i) * grad.head, ln.in);
        }
#pragma unroll
        for (int i = 0; i < 2; i++) one(f[i], df[i], h + i);
      }
      for (; h < g1; h++) one(load8(src + h * from.head, ln.in), load8(gsrc + h * grad.head, ln.in), h);
    };
    run(a.q, x.g.dq_out, x.g.dq, a.q_gamma, h0, min(h1, a.q_heads), gsum[0]);
    run(a.k, x.g.dk_out, x.g.dk, a.k_gamma, max(h0 - a.q_heads, 0), h1 - a.q_heads, gsum[1]);
  }
  if (!x.part) return;
  float *out = x.part + ((int64_t)blockIdx.y * x.blocks + blockIdx.x) * 2 * a.dim;
#pragma unroll
  for (int w = 0; w < 2; w++) {
    __syncthreads();
#pragma unroll
    for (int e = 0; e < 8; e++) meet[grp * (8 * LANES) + 8 * l + e] = gsum[w][e];
    __syncthreads();
    for (int c = threadIdx.x; c < a.dim; c += kThreads) {
      float v = 0.0f;
      for (int i = 0; i < GROUPS; i++) v += meet[i * (8 * LANES) + c];
      out[w * a.dim + c] = v;
    }
  }
}

// A block has 4 columns of one gamma, a thread every 256th part of them.
// Bound by latency (512 workgroups' parts of 128 columns: 5 us).
__global__ __launch_bounds__(256) void norm_rope_gamma_kernel(NormRopeArgs x, int parts) {
  __shared__ f4 strand[4];
  const ixh_norm_rope_args &a = x.a;
  const int c = blockIdx.x * 4;
  void *const to = blockIdx.y ? x.g.dk_gamma : x.g.dq_gamma;
  if (!to) return;
  f4 v{};
#pragma unroll 4
  for (int i = threadIdx.x; i < parts; i += 256) v += *(const f4 *)(x.part + ((int64_t)i * 2 + blockIdx.y) * a.dim + c);
#pragma unroll
  for (int o = 1; o < 64; o <<= 1)
#pragma unroll
    for (int e = 0; e < 4; e++) v[e] += __shfl_xor(v[e], o);
  if (threadIdx.x % 64 == 0) strand[threadIdx.x / 64] = v;
  __syncthreads();
  if (threadIdx.x) return;
  v = (strand[0] + strand[1]) + (strand[2] + strand[3]);
  if (a.gamma_type == IXH_TYPE_F32)
    store4((float *)to + c, v);
  else if (a.gamma_type == IXH_TYPE_BF16)
    store4((__bf16 *)to + c, v);
  else
    store4((_Float16 *)to + c, v);
}

template <class T, int LANES, int NORM>
void launch(const NormRopeArgs &x, bool backward, hipStream_t s) {
  const dim3 grid(x.blocks, (x.a.q_heads + x.a.k_heads + x.heads_step - 1) / x.heads_step);
  if (backward)
    norm_rope_backward_kernel<T, LANES, NORM><<<grid, kThreads, 0, s>>>(x);
  else
    norm_rope_kernel<T, LANES, NORM><<<grid, kThreads, 0, s>>>(x);
}
template <class T, int LANES>
void by_norm(const NormRopeArgs &x, bool backward, hipStream_t s) {
  switch (x.a.norm) {
    case IXH_HEAD_NORM_NONE: return launch<T, LANES, IXH_HEAD_NORM_NONE>(x, backward, s);
    case IXH_HEAD_NORM_RMS: return launch<T, LANES, IXH_HEAD_NORM_RMS>(x, backward, s);
    default: return launch<T, LANES, IXH_HEAD_NORM_LAYER>(x, backward, s);
  }
}
template <class T>
void by_dim(const NormRopeArgs &x, bool backward, hipStream_t s) {
  if (x.a.dim <= 32) return by_norm<T, 4>(x, backward, s);
  if (x.a.dim <= 64) return by_norm<T, 8>(x, backward, s);
  if (x.a.dim <= 128) return by_norm<T, 16>(x, backward, s);
  return by_norm<T, 32>(x, backward, s);
}
void by_type(const NormRopeArgs &x, bool backward, hipStream_t s) {
  switch (x.a.type) {
    case IXH_TYPE_F32: return by_dim<float>(x, backward, s);
    case IXH_TYPE_BF16: return by_dim<__bf16>(x, backward, s);
    default: return by_dim<_Float16>(x, backward, s);
  }
}

}  // namespace

void launch_norm_rope(const NormRopeArgs &x, hipStream_t s) { by_type(x, false, s); }
void launch_norm_rope_backward(const NormRopeArgs &x, hipStream_t s) {
  by_type(x, true, s);
  if (!x.part) return;
  const int steps = (x.a.q_heads + x.a.k_heads + x.heads_step - 1) / x.heads_step;
  norm_rope_gamma_kernel<<<dim3(x.a.dim / 4, 2), 256, 0, s>>>(x, x.blocks * steps);
}

}  // namespace ixh
