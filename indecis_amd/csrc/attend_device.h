// attend_device.h — what the float attention kernels share: fragments of
// the three types, tiles of rows in LDS, the masks' bounds, the scores.
//
// Layout. Every product is taken with a 32x32x16 MFMA (for float32 eight
// 32x32x2 ones over the same fragments): lane l supplies row l % 32 of A
// and column l % 32 of B, eight values each of the 16 of k; which eight is
// free as long as A and B agree. The result's lane l holds column l % 32,
// rows 8 (r / 4) + 4 (l / 32) + r % 4, r = 0..15. So a product whose columns
// are queries leaves in a lane 4 keys of every 8 of one query: taken in that
// order they are the next product's B fragment over k = keys as they stand,
// and its A fragment is read from LDS transposed in the same order
// (ds_read_b64_tr_b16: 4 rows of 16 columns a 16-lane group). No score
// leaves the registers, and a query's softmax is its lane's own.
#pragma once
#include <hip/hip_bf16.h>
#include <hip/hip_fp16.h>

#include <type_traits>

#include "attend.h"

namespace ixh {

typedef float v16f __attribute__((ext_vector_type(16)));
typedef float f4 __attribute__((ext_vector_type(4)));
typedef short v4s __attribute__((ext_vector_type(4)));
typedef __bf16 v8bf __attribute__((ext_vector_type(8)));
typedef _Float16 v8h __attribute__((ext_vector_type(8)));
struct alignas(16) v8f {
  f4 lo, hi;
};
typedef int i4 __attribute__((ext_vector_type(4)));

constexpr float kLog2e = 1.44269504088896340736f;
constexpr float kLn2 = 0.69314718055994530942f;

template <class T>
struct Kind;
template <>
struct Kind<__bf16> {
  typedef v8bf frag;
};
template <>
struct Kind<_Float16> {
  typedef v8h frag;
};
template <>
struct Kind<float> {
  typedef v8f frag;
};

__device__ __forceinline__ v16f mfma16(v8bf a, v8bf b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_bf16(a, b, c, 0, 0, 0);
}
__device__ __forceinline__ v16f mfma16(v8h a, v8h b, v16f c) {
  return __builtin_amdgcn_mfma_f32_32x32x16_f16(a, b, c, 0, 0, 0);
}
// Value e of both halves of the wave together are one 32x32x2 product.
__device__ __forceinline__ v16f mfma16(const v8f &a, const v8f &b, v16f c) {
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.lo[e], b.lo[e], c, 0, 0, 0);
#pragma unroll
  for (int e = 0; e < 4; e++) c = __builtin_amdgcn_mfma_f32_32x32x2f32(a.hi[e], b.hi[e], c, 0, 0, 0);
  return c;
}

template <class F>
__device__ __forceinline__ float frag_at(const F &f, int e) {
  return (float)f[e];
}
__device__ __forceinline__ float frag_at(const v8f &f, int e) { return e < 4 ? f.lo[e] : f.hi[e - 4]; }

// Eight accumulator values as a fragment of the type, rounded to nearest even.
template <class F>
__device__ __forceinline__ F pack8(const float *p) {
  F f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = p[e];
  return f;
}
template <>
__device__ __forceinline__ v8f pack8<v8f>(const float *p) {
  v8f f;
#pragma unroll
  for (int e = 0; e < 4; e++) f.lo[e] = p[e], f.hi[e] = p[e + 4];
  return f;
}
template <>
__device__ __forceinline__ v8bf pack8<v8bf>(const float *p) {
  v8bf f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = (__bf16)p[e];
  return f;
}
template <>
__device__ __forceinline__ v8h pack8<v8h>(const float *p) {
  v8h f;
#pragma unroll
  for (int e = 0; e < 8; e++) f[e] = (_Float16)p[e];
  return f;
}

// Eight values at p; none past `valid` (0 or 8) are read.
template <class T>
__device__ __forceinline__ typename Kind<T>::frag load8(const T *p, bool valid) {
  typename Kind<T>::frag f{};
  if (valid) f = *(const typename Kind<T>::frag *)p;
  return f;
}

// Four consecutive values, rounded once.
__device__ __forceinline__ void store4(float *p, f4 v) { *(f4 *)p = v; }
__device__ __forceinline__ void store4(__bf16 *p, f4 v) {
  typedef __bf16 b4 __attribute__((ext_vector_type(4)));
  b4 o = {(__bf16)v[0], (__bf16)v[1], (__bf16)v[2], (__bf16)v[3]};
  *(b4 *)p = o;
}
__device__ __forceinline__ void store4(_Float16 *p, f4 v) {
  typedef _Float16 h4 __attribute__((ext_vector_type(4)));
  h4 o = {(_Float16)v[0], (_Float16)v[1], (_Float16)v[2], (_Float16)v[3]};
  *(h4 *)p = o;
}

__device__ __forceinline__ float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }

// The other half of the wave's value at the same column.
__device__ __forceinline__ float other_half(float v) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const unsigned u = __builtin_bit_cast(unsigned, v);
  const u2 r = __builtin_amdgcn_permlane32_swap(u, u, false, false);
  return __builtin_bit_cast(float, (__lane_id() & 32) ? r[0] : r[1]);
}
// A fixed order of the two halves, so that both get the same bits.
__device__ __forceinline__ float half_sum(float v) { return v + other_half(v); }
__device__ __forceinline__ float half_max(float v) { return __builtin_fmaxf(v, other_half(v)); }

// The lower half's values of v with 0 in the upper half, and the upper
// half's, brought down.
__device__ __forceinline__ void halves_apart(float v, float *low, float *high) {
  typedef unsigned u2 __attribute__((ext_vector_type(2)));
  const u2 r = __builtin_amdgcn_permlane32_swap(__builtin_bit_cast(unsigned, v), 0u, false, false);
  const unsigned a = r[0], b = r[1];  // a bit cast of r[1] itself reads r[0]
  *low = __builtin_bit_cast(float, a);
  *high = __builtin_bit_cast(float, b);
}
// Every lane's value from the lane below, lane 0's 0 (wave_shr:1).
__device__ __forceinline__ float lane_up(float v) {
  return __builtin_bit_cast(float, __builtin_amdgcn_update_dpp(0, __builtin_bit_cast(int, v), 0x138, 0xf, 0xf, true));
}

// ---- tiles of rows in LDS ---------------------------------------------------
// R rows of DT values in 16-byte pieces; piece c of row r stands at
// c ^ turn(r). A wave's read of rows takes 2 pieces of 32 rows, a transposed
// one 4 pieces side by side of 8 rows. At 256 bytes a row the rows of one
// transposed read are turned by whole groups of 4 pieces (every 16-byte slot
// of the banks' 256 bytes is then asked equally often: a training step of 8
// sequences of 2,048, 16/4 heads of 128, 898 -> 846 us against r & 7); at
// 128 bytes two rows lie in one round of the banks and r & 7 is as good. A
// turn is the same 8 rows on, so that the second half of a transposed read
// is a constant offset.
template <class T, int DT>
__device__ __forceinline__ int turn(int r) {
  if constexpr (sizeof(T) == 2 && DT == 128) return (r & 3) << 2 | (r >> 2 & 1);
  return r & 7;
}
template <class T, int DT, int R, int THREADS>
struct Tile {
  static constexpr int EPC = 16 / (int)sizeof(T);  // values a piece
  static constexpr int CH = DT / EPC;              // pieces a row
  static constexpr int RB = DT * (int)sizeof(T);   // bytes a row
  static constexpr int BYTES = R * RB;
  static constexpr int N = R * CH / THREADS;       // pieces a thread
  static_assert(N * THREADS == R * CH && CH >= 8, "");
  static constexpr int STEP = THREADS / CH;        // rows between a thread's pieces
  static_assert(THREADS % CH == 0, "");
  i4 part[N];
  unsigned off;  // of the thread's first piece, in bytes from the tile's first row

  // A piece past `dim` is read as the row's first and dropped in put().
  __device__ __forceinline__ void init(int64_t stride, int dim, int tid) {
    const int r = tid / CH, c = tid % CH;
    off = (unsigned)(r * stride * sizeof(T)) + (c * EPC < dim ? 16 * c : 0);
  }
  // Starts the loads of the rows at `first`, `left` of which there are: a row
  // past them is read as the last and dropped in put().
  __device__ __forceinline__ void get(const T *first, int64_t stride, int left, int tid) {
    if (left >= R) {
#pragma unroll
      for (int i = 0; i < N; i++) part[i] = *(const i4 *)((const char *)(first + i * STEP * stride) + off);
    } else {
#pragma unroll
      for (int i = 0; i < N; i++) {
        const int past = max(tid / CH + i * STEP - (left - 1), 0);
        part[i] = *(const i4 *)((const char *)(first + (i * STEP - past) * stride) + off);
      }
    }
  }
  // Starts the loads of those rows' tags, by which put() may drop them too.
  struct Tags {
    int v[N];
    __device__ __forceinline__ void get(const int32_t *first, int left, int tid) {
#pragma unroll
      for (int i = 0; i < N; i++) v[i] = first[min(tid / CH + i * STEP, left - 1)];
    }
  };
  // Writes them; what is past `left` rows or `dim` columns, and rows whose
  // tag keep() refuses, as 0. all: nothing is.
  template <class Keep>
  __device__ __forceinline__ void put(char *lds, int left, int dim, int tid, bool all, const Tags &tags, Keep keep) {
#pragma unroll
    for (int i = 0; i < N; i++) {
      const int r = tid / CH + i * STEP, c = tid % CH;
      i4 v = part[i];
      if (!all && !(c * EPC < dim && r < left && keep(tags.v[i]))) v = i4{0, 0, 0, 0};
      *(i4 *)(lds + r * RB + ((c ^ turn<T, DT>(r)) << 4)) = v;
    }
  }

  // A's fragment of rows row0 + l % 32 at k step s (16 values of a row).
  __device__ static __forceinline__ typename Kind<T>::frag rows(const char *lds, int row0, int s, int lane) {
    const int r = row0 + (lane & 31), h = lane >> 5;
    typename Kind<T>::frag f;
    if constexpr (sizeof(T) == 2) {
      f = *(const typename Kind<T>::frag *)(lds + r * RB + (((2 * s + h) ^ turn<T, DT>(r)) << 4));
    } else {
      const int c = 4 * s + 2 * h;
      f.lo = *(const f4 *)(lds + r * RB + ((c ^ turn<T, DT>(r)) << 4));
      f.hi = *(const f4 *)(lds + r * RB + (((c + 1) ^ turn<T, DT>(r)) << 4));
    }
    return f;
  }
  // A's fragment of columns 32 dt + l % 32 over the 16 rows from row0, rows
  // in the order in which a result's registers hold them.
  __device__ static __forceinline__ typename Kind<T>::frag cols(const char *lds, int row0, int dt, int lane) {
    const int h = lane >> 5;
    typename Kind<T>::frag f;
    if constexpr (sizeof(T) == 2) {
      const int a = lane & 15, g = (lane >> 4) & 1;
      const int r = row0 + 4 * h + (a >> 2), c = 4 * dt + 2 * g + ((a >> 1) & 1);
      const char *p = lds + r * RB + ((c ^ turn<T, DT>(r)) << 4) + ((a & 1) << 3);
      typedef __attribute__((address_space(3))) v4s lv4s;
      union {
        v4s q[2];
        typename Kind<T>::frag f;
      } u;
      u.q[0] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *)p);
      u.q[1] = __builtin_amdgcn_ds_read_tr16_b64_v4i16((lv4s *)(p + 8 * RB));
      f = u.f;
    } else {
      const int d = 32 * dt + (lane & 31), c = d >> 2;
#pragma unroll
      for (int j = 0; j < 4; j++) {
        const int r = row0 + 4 * h + j;
        const char *p = lds + r * RB + ((c ^ turn<T, DT>(r)) << 4) + ((d & 3) << 2);
        f.lo[j] = *(const float *)p;
        f.hi[j] = *(const float *)(p + 8 * RB);
      }
    }
    return f;
  }
};

// A wave's 32 result rows (lane l has row l % 32, columns as the registers
// hold them) times f, through 32 rows of its own in LDS to whole rows in
// memory: eight bytes a lane of a row each would cost the address unit a
// cycle a lane (256 sequences of 64-512, 12 heads of 64, window of 64: 162 ->
// 156 us). row_at(i): the address of
// row i, or nullptr. Every wave calls it, the block's tiles no longer needed.
template <class T, int DT, class RowAt>
__device__ __forceinline__ void store_rows(const v16f *acc, float f, char *lds, int dim, int lane, RowAt row_at) {
  constexpr int EPC = 16 / (int)sizeof(T), CH = DT / EPC, RB = DT * (int)sizeof(T);
  const int r = lane & 31, h = lane >> 5;
  __syncthreads();
#pragma unroll
  for (int d = 0; d < DT / 32; d++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int c = 32 * d + 8 * g + 4 * h;
      store4((T *)(lds + r * RB + (((c / EPC) ^ turn<T, DT>(r)) << 4)) + c % EPC,
             f4{acc[d][4 * g] * f, acc[d][4 * g + 1] * f, acc[d][4 * g + 2] * f, acc[d][4 * g + 3] * f});
    }
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 32 * CH / 64; i++) {
    const int at = i * 64 + lane, row = at / CH, c = at % CH;
    T *const to = row_at(row);
    const i4 v = *(const i4 *)(lds + row * RB + ((c ^ turn<T, DT>(row)) << 4));
    if (to && c * EPC < dim) *(i4 *)(to + c * EPC) = v;
  }
}

// Whether a step of the products at this column is taken: a float32 one costs
// 8 slow MFMAs, so those past `dim` are left out; for 16-bit types the branch
// costs more than the MFMA.
template <class T>
__device__ __forceinline__ bool within(int column, int dim) {
  return sizeof(T) == 2 || column < dim;
}

// ---- sequences and masks ----------------------------------------------------

// offs[i] as a row of an array of n rows, whatever it holds.
__device__ __forceinline__ int row_at(const int32_t *offs, int i, int n) { return min(max(offs[i], 0), n); }

// One sequence: its rows in the packed arrays.
struct Seq {
  int q0, nq, k0, nk, shift, prefix;  // shift: a query's place among the keys less its row
};

// The sequence of a slot (attend_slots) of `offs` (a's q_offs or k_offs) and
// its block of rows: a search by the whole wave, 256 sequences a step, each
// lane with four places side by side, and the ends of the sequence found come
// out of the last step's values. n * pack is below 2^31.
__device__ __forceinline__ Seq find_block(const ixh_attend_args &a, bool by_keys, int rows, int pack, int64_t slot,
                                          int64_t *block) {
  const int32_t *const offs = by_keys ? a.k_offs : a.q_offs;
  const int n = by_keys ? a.nk : a.nq, lane = __lane_id();
  int lo = 0, count = a.B, at, v[5];
  for (;;) {
    const int step = (count + 255) / 256;
#pragma unroll
    for (int e = 0; e < 5; e++) v[e] = row_at(offs, min(lo + (4 * lane + e) * step, a.B), n);
    int hits = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
      const int i = (4 * lane + e) * step;
      hits += __popcll(__ballot(i < count && (unsigned)(v[e] * pack) / (unsigned)rows + lo + i <= slot));
    }
    at = __builtin_amdgcn_readfirstlane(max(hits - 1, 0));
    if (step == 1) break;
    lo += at * step;
    count = min(step, count - at * step);
  }
  const int b = lo + at;
  const int from = at & 3;
  const int x = from == 0 ? v[0] : from == 1 ? v[1] : from == 2 ? v[2] : v[3];
  const int y = from == 0 ? v[1] : from == 1 ? v[2] : from == 2 ? v[3] : v[4];
  const int first = __builtin_amdgcn_readlane(x, at >> 2), end = __builtin_amdgcn_readlane(y, at >> 2);
  *block = slot - ((unsigned)(first * pack) / (unsigned)rows + b);
  int first2 = first, end2 = end;
  if (a.q_offs != a.k_offs) {
    const int32_t *const others = by_keys ? a.q_offs : a.k_offs;
    first2 = row_at(others, b, by_keys ? a.nq : a.nk);
    end2 = row_at(others, b + 1, by_keys ? a.nq : a.nk);
  }
  Seq s;
  s.q0 = by_keys ? first2 : first;
  s.k0 = by_keys ? first : first2;
  s.nq = max((by_keys ? end2 : end) - s.q0, 0);
  s.nk = max((by_keys ? end : end2) - s.k0, 0);
  s.shift = s.nk - s.nq;
  s.prefix = a.prefix ? a.prefix[b] : 0;
  return s;
}

// The keys lo..hi that the query at place p sees (documents apart); empty
// where hi < lo. Both ends grow with p.
__device__ __forceinline__ void key_bounds(const ixh_attend_args &a, const Seq &s, int p, int *lo, int *hi) {
  int h = s.nk - 1, l = 0;
  if (a.causal) h = min(h, max(p, s.prefix - 1));
  if (a.window >= 0) {
    h = min((int64_t)h, (int64_t)p + a.window);
    l = max((int64_t)l, (int64_t)p - a.window);
  }
  *lo = l;
  *hi = h;
}
// The places lo..hi of the queries that see key j.
__device__ __forceinline__ void query_bounds(const ixh_attend_args &a, const Seq &s, int j, int *lo, int *hi) {
  int l = s.shift, h = s.nk - 1;
  if (a.causal && j >= s.prefix) l = max(l, j);
  if (a.window >= 0) {
    l = max((int64_t)l, (int64_t)j - a.window);
    h = min((int64_t)h, (int64_t)j + a.window);
  }
  *lo = l;
  *hi = h;
}

// ---- documents --------------------------------------------------------------

constexpr int kDocWords = 64;  // of 64 steps; later steps are taken as live

// Which of the steps t0..t1 - 1 (STEP rows each, of the n in `theirs`) may
// hold a row of a document that a row first..last of `mine` has. Every wave
// calls it; a barrier before the words are read.
template <int STEP, int WAVES>
__device__ __forceinline__ void doc_steps(const int32_t *mine, int first, int last, const int32_t *theirs, int n, int t0,
                                          int t1, uint64_t *live, int wave, int lane) {
  int mn = INT32_MAX, mx = -1;
  for (int i = first + lane; i <= last; i += 64) {
    const int d = mine[i];
    mn = min(mn, d < 0 ? INT32_MAX : d);
    mx = max(mx, d);
  }
#pragma unroll
  for (int o = 32; o; o >>= 1) {
    mn = min(mn, __shfl_xor(mn, o));
    mx = max(mx, __shfl_xor(mx, o));
  }
  // A wave takes the 64 steps of a word, 16 at a time: 4 lanes a step, each
  // with every 4th row of it, whose loads are launched together.
  for (int w = wave; w < kDocWords && t0 + 64 * w < t1; w += WAVES) {
    uint64_t word = 0;
    for (int part = 0; part < 4 && t0 + 64 * w + 16 * part < t1; part++) {
      const int t = t0 + 64 * w + 16 * part + (lane >> 2);
      int d[STEP / 4];
#pragma unroll
      for (int i = 0; i < STEP / 4; i++) d[i] = theirs[min(t * STEP + 4 * i + (lane & 3), n - 1)];
#pragma unroll
      for (int i = 0; i < STEP / 4; i++) asm volatile("" : "+v"(d[i]));  // none is used before all are on their way
      int tmn = INT32_MAX, tmx = -1;
#pragma unroll
      for (int i = 0; i < STEP / 4; i++) {
        tmn = min(tmn, d[i] < 0 ? INT32_MAX : d[i]);
        tmx = max(tmx, d[i]);
      }
#pragma unroll
      for (int o = 1; o < 4; o <<= 1) {
        tmn = min(tmn, __shfl_xor(tmn, o));
        tmx = max(tmx, __shfl_xor(tmx, o));
      }
      uint64_t hit = __ballot(t < t1 && tmx >= 0 && mx >= 0 && tmn <= mx && tmx >= mn);
      // every 4th lane's bit, side by side
      hit &= 0x1111111111111111ull;
      hit = (hit | hit >> 3) & 0x0303030303030303ull;
      hit = (hit | hit >> 6) & 0x000f000f000f000full;
      hit = (hit | hit >> 12) & 0x000000ff000000ffull;
      hit = (hit | hit >> 24) & 0xffffull;
      word |= hit << (16 * part);
    }
    if (lane == 0) live[w] = word;
  }
}
// Every load so far has come in: a loop's own loads need no wait for those
// of values that it only reads.
__device__ __forceinline__ void loads_done() { __builtin_amdgcn_s_waitcnt(0x0f70); }

// The first live step from t on, t1 if none.
__device__ __forceinline__ int next_live(const uint64_t *live, int t, int t0, int t1) {
  while (t < t1) {
    const int i = t - t0;
    if (i >= 64 * kDocWords) return t;
    const uint64_t w = live[i >> 6] >> (i & 63);
    const int skip = __builtin_amdgcn_readfirstlane(w ? __builtin_ctzll(w) : 64 - (i & 63));
    const bool hit = __builtin_amdgcn_readfirstlane(w != 0);
    t += skip;
    if (hit) return min(t, t1);
  }
  return t1;
}

// The documents of a wave's 32 columns.
struct ColumnDocs {
  int doc;   // the lane's: -1 for padding
  int all;   // that of all of them,
  bool one;  // if they have one
  __device__ __forceinline__ explicit ColumnDocs(int d) {
    doc = max(d, -1);
    all = __builtin_amdgcn_readfirstlane(doc);
    one = __ballot(doc == all) == ~0ull;
  }
  // Takes the lane's bits of the 32 rows whose documents stand at `rows` in
  // LDS (padding: -2) that are of other documents out of `bits` (row_bits'
  // order); whether any row is left to any lane. Where the columns or the
  // rows have one document alone, that takes no comparison a score.
  __device__ __forceinline__ bool tile(const int *rows, int lane, unsigned *bits) const {
    const int h = lane >> 5, theirs = rows[lane & 31];
    if (one) {
      const unsigned hit = (unsigned)__ballot(theirs == all);
      *bits &= hit >> (4 * h);
      return hit != 0;
    }
    const int first = __builtin_amdgcn_readfirstlane(theirs);
    if (__ballot(theirs == first) == ~0ull) {
      if (doc != first) *bits = 0;
      return __ballot(doc == first) != 0;
    }
    unsigned hit = 0;
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const i4 d = *(const i4 *)(rows + 8 * g + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; e++) hit |= d[e] == doc ? 1u << (8 * g + e) : 0u;
    }
    *bits &= hit;
    return true;
  }
};

// ---- scores -----------------------------------------------------------------
// FEAT: 1 a tanh cap, 2 a bias by distance.
enum { kCap = 1, kBias = 2 };

// A call's scores in base 2: z = gain * q.k, or, capped, gain * tanh(c1 q.k);
// the softmax is 2^(z - maximum).
struct Score {
  float c1, gain;
  __device__ __forceinline__ explicit Score(const ixh_attend_args &a, bool cap) {
    c1 = cap ? a.scale / a.cap : 1.0f;
    gain = (cap ? a.cap : a.scale) * kLog2e;
  }
};

// tanh(c1 z) of a tile's 16 scores a lane. Where every score of the wave is
// within half the cap, as most are, an odd polynomial: tanh(x) / x over x^2
// in 0..1/4 (interpolated at Chebyshev's nodes, 2.7e-8 off), 2 * 2^-24 of
// tanh with its roundings and no dearer than an exponential and a
// reciprocal. Else 1 - 2 / (1 + e^2x) by those, off by up to 2^-21 of 1, next
// to a 16-bit result nothing, and for float32 the library's tanh.
template <class T>
__device__ __forceinline__ void tanh_tile(v16f &z, const Score &sc) {
  float most = 0.0f;
#pragma unroll
  for (int r = 0; r < 16; r++) {
    z[r] *= sc.c1;
    most = __builtin_fmaxf(most, __builtin_fabsf(z[r]));
  }
  if (__ballot(!(most <= 0.5f)) == 0) {
#pragma unroll
    for (int r = 0; r < 16; r++) {
      const float x = z[r], y = x * x;
      float p = __builtin_fmaf(y, 0.017141319811344147f, -0.05298924073576927f);
      p = __builtin_fmaf(p, y, 0.13324828445911407f);
      p = __builtin_fmaf(p, y, -0.3333307206630707f);
      z[r] = __builtin_fmaf(p * y, x, x);
    }
  } else {
#pragma unroll
    for (int r = 0; r < 16; r++) {
      if constexpr (sizeof(T) == 4)
        z[r] = tanhf(z[r]);
      else
        z[r] = __builtin_fmaf(-2.0f, __builtin_amdgcn_rcpf(1.0f + exp2_fast(z[r] * (2 * kLog2e))), 1.0f);
    }
  }
}

// The bias starts the first product's sum, in units of q.k (bias / scale), so
// that it costs no operation of its own; under a cap it is added to z, in
// base 2.
__device__ __forceinline__ float bias_unit(const ixh_attend_args &a, bool cap) { return cap ? kLog2e : 1.0f / a.scale; }

// One head's bias table by distance, copied to LDS with its ends drawn out
// by kBiasPad.
template <class T>
__device__ __forceinline__ void load_bias(const ixh_attend_args &a, int head, float unit, float *lds, int tid,
                                          int threads) {
  const int len = attend_bias_len(a.reach);
  for (int i = tid; i < len; i += threads) {
    const int d = min(max(i - a.reach - kBiasPad, -a.reach), a.reach);
    const int b = a.buckets[d + a.reach];
    lds[i] = b >= 0 && b < a.n_buckets ? (float)((const T *)a.table)[(int64_t)b * a.heads + head] * unit : 0.0f;
  }
}

// One head's bias of a lane's 16 scores of a 32x32 tile. d0: the distance at
// register 0, which grows by `sign` a row; near..far: the tile's distances.
struct Bias {
  const float *tab;  // nullptr: no table
  float slope;       // 0: none
  int reach;
  template <int SIGN>
  __device__ __forceinline__ v16f at(int d0, int near, int far) const {
    v16f z{};
    if (tab) {
      if (near >= reach || far <= -reach) {
        const float c = tab[near >= reach ? 2 * (reach + kBiasPad) : 0];
#pragma unroll
        for (int r = 0; r < 16; r++) z[r] = c;
      } else {
        const float *p = tab + d0 + reach + kBiasPad;
#pragma unroll
        for (int r = 0; r < 16; r++) z[r] = p[SIGN * (8 * (r >> 2) + (r & 3))];
      }
    }
    if (slope != 0.0f) {
      const float f = (float)d0;
#pragma unroll
      for (int r = 0; r < 16; r++)
        z[r] = __builtin_fmaf(slope, __builtin_fabsf(f + (float)(SIGN * (8 * (r >> 2) + (r & 3)))), z[r]);
    }
    return z;
  }
};

// ---- masks ------------------------------------------------------------------
// The lane's rows of a 32-row tile from j0 on that lie in lo..hi, a bit each,
// bit 8 (r / 4) + r % 4 its register r's.
__device__ __forceinline__ unsigned row_bits(int j0, int lo, int hi, int h) {
  const int l = min(max(lo - j0, 0), 32), u = min(max(hi + 1 - j0, 0), 32);
  const unsigned below = (unsigned)((1ull << l) - 1), upto = (unsigned)((1ull << u) - 1);
  return (upto & ~below) >> (4 * h);
}
// All ones where the bit of register r is set, else 0: one instruction, which
// the compiler would make a test, a comparison and a select of.
__device__ __forceinline__ unsigned bit_mask(unsigned bits, int r) {
  unsigned m;
  asm("v_bfe_i32 %0, %1, %2, 1" : "=v"(m) : "v"(bits), "n"(8 * (r >> 2) + (r & 3)));
  return m;
}
// v where the bit of register r is set, else -inf.
__device__ __forceinline__ float or_minus_inf(unsigned bits, int r, float v) {
  const unsigned m = bit_mask(bits, r);
  return __builtin_bit_cast(float, (__builtin_bit_cast(unsigned, v) & m) | (0xff800000u & ~m));
}
// v where the bit of register r is set, else 0.
__device__ __forceinline__ float if_bit(unsigned bits, int r, float v) {
  return __builtin_bit_cast(float, __builtin_bit_cast(unsigned, v) & bit_mask(bits, r));
}


}  // namespace ixh
