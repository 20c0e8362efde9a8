// attend_fwd.hip — attention of float rows with shaped scores: one pass over
// the keys with a running maximum and sum a query.
//
// A workgroup of 4 waves has 128 query rows of a sequence and head, 32 a
// wave (one wave and 32 rows where sequences are short). K and V come through
// LDS, 64 keys a step in two buffers, loaded into registers a step ahead.
// The scores are taken transposed (keys x queries, attend_device.h): a lane
// has one query, so maximum, sum and rescaling are its own, and the
// probabilities go into the second product from the registers they are in.
//
// What bounds it, by the shape (bf16, heads of 64 unless said otherwise; the
// card's copy 4.9 TB/s, a large product 1,060 TFLOP/s):
//  - long sequences: the issue of matrix and vector instructions together (4
//    sequences of 8,192, 12 heads, causal with prefix: 570 us, 742 TFLOP/s);
//  - many short blocks: a block's start, its few steps in series, and the
//    vector work of cap and masks (256 sequences of 64-512, 12 heads, cap and
//    window of 64: 146 us, 3.1 TB/s; learned bias, no window: 205 us, 369
//    TFLOP/s);
//  - one token over long keys: the reading of K and V (32 sequences of
//    512-8,192, 16/4 heads of 128, float16: 67 us and the join's 9, 2.8 TB/s
//    of the whole call);
//  - one short sequence: its block's steps in series (15 tokens, 4 heads,
//    float32: 9 us).
#include "attend_device.h"
#include "ixh_internal.h"

namespace ixh {
namespace {

template <class T, int DT, int WAVES>
struct FwdShape {
  static constexpr int THREADS = 64 * WAVES, ROWS = 32 * WAVES;
  static constexpr int BK = attend_keys(sizeof(T), WAVES == 1);
  typedef Tile<T, DT, BK, THREADS> KV;
  static_assert(4 * KV::BYTES >= WAVES * 32 * DT * (int)sizeof(T), "the result's rows");
  // LDS: K and V twice, the key documents twice, the live steps of documents,
  // then the bias
  static constexpr int DOCS = 4 * KV::BYTES, LIVE = DOCS + 2 * 4 * BK, BIAS = LIVE + 8 * kDocWords;
};

template <class T, int DT, int WAVES, int FEAT>
__global__ __launch_bounds__(64 * WAVES, sizeof(T) * DT == 128 ? 3 : sizeof(T) * DT == 512 && WAVES == 1 ? 1 : 2)
void attend_fwd_kernel(AttendArgs x) {
  typedef FwdShape<T, DT, WAVES> Sh;
  typedef typename Sh::KV KV;
  typedef typename Kind<T>::frag Frag;
  constexpr int THREADS = Sh::THREADS, ROWS = Sh::ROWS, BK = Sh::BK, KS = DT / 16, ND = DT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const ixh_attend_args &a = x.a;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  int *const kdocs = (int *)(smem + Sh::DOCS);
  uint64_t *const live = (uint64_t *)(smem + Sh::LIVE);
  float *const bias = (float *)(smem + Sh::BIAS);

  // last blocks first: under a causal mask they have the most keys
  const int pack = x.pack, nh = pack > 1 ? a.kv_heads : a.heads;
  const int hb = blockIdx.x % nh;
  int64_t blk;
  const Seq s = find_block(a, false, ROWS, pack, x.slots - 1 - blockIdx.x / nh, &blk);
  const int rows = s.nq * pack;
  if (blk < 0 || blk * ROWS >= rows) return;  // below 0: offsets that do not ascend
  const int row0 = (int)blk * ROWS, row1 = min(row0 + ROWS, rows);
  const int kvh = pack > 1 ? hb : hb / x.group;

  // the lane's query: its row, head and place; rows past the last repeat it
  auto token = [&](int r) { return pack > 1 ? r / pack : r; };
  const int r = min(row0 + wave * 32 + (lane & 31), rows - 1), tok = token(r), sub = r - tok * pack;
  const bool mine = row0 + wave * 32 + (lane & 31) < rows;
  const int head = pack > 1 ? hb * pack + sub : hb;
  const int p = tok + s.shift;
  int lo, hi;
  key_bounds(a, s, p, &lo, &hi);
  const int p_lo = __builtin_amdgcn_readlane(p, 0), p_hi = __builtin_amdgcn_readlane(p, 31);
  const int lo_min = __builtin_amdgcn_readlane(lo, 0), lo_max = __builtin_amdgcn_readlane(lo, 31);
  const int hi_min = __builtin_amdgcn_readlane(hi, 0);
  // a wave past the last row has nothing to see
  const int hi_max = row0 + wave * 32 < rows ? __builtin_amdgcn_readlane(hi, 31) : -1;

  // the workgroup's steps of keys
  int t_begin, t_end;
  {
    int l, u, unused;
    key_bounds(a, s, token(row0) + s.shift, &l, &unused);
    key_bounds(a, s, token(row1 - 1) + s.shift, &unused, &u);
    t_begin = l / BK;
    t_end = u >= l ? u / BK + 1 : t_begin;
    if (x.splits > 1) {
      const int per = (t_end - t_begin + x.splits - 1) / x.splits;
      t_begin = min(t_begin + per * (int)blockIdx.y, t_end);
      t_end = min(t_begin + per, t_end);
    }
  }

  // Q's fragments, columns past dim 0
  Frag q[KS];
  {
    const T *qr = (const T *)a.q.p + (s.q0 + tok) * a.q.row + head * a.q.head;
#pragma unroll
    for (int i = 0; i < KS; i++) q[i] = load8(qr + 16 * i + 8 * h, 16 * i + 8 * h < a.dim);
  }
  const T *const kb = (const T *)a.k.p + s.k0 * a.k.row + kvh * a.k.head;
  const T *const vb = (const T *)a.v.p + s.k0 * a.v.row + kvh * a.v.head;
  KV kt, vt;
  typename KV::Tags tags;
  kt.init(a.k.row, a.dim, tid);
  vt.init(a.v.row, a.dim, tid);
  int kdoc = 0;
  auto fetch = [&](int t) {
    const int left = s.nk - t * BK;
    kt.get(kb + (int64_t)(t * BK) * a.k.row, a.k.row, left, tid);
    vt.get(vb + (int64_t)(t * BK) * a.v.row, a.v.row, left, tid);
    if (a.q_docs) {
      tags.get(a.k_docs + s.k0 + t * BK, left, tid);
      if (tid < BK) kdoc = a.k_docs[s.k0 + t * BK + min(tid, left - 1)];
    }
  };

  const ColumnDocs docs(a.q_docs ? a.q_docs[s.q0 + tok] : 0);
  if (a.q_docs)
    doc_steps<BK, WAVES>(a.q_docs + s.q0, token(row0), token(row1 - 1), a.k_docs + s.k0, s.nk, t_begin, t_end, live, wave,
                         lane);
  if constexpr (FEAT & kBias) {
    if (a.table)
      for (int i = 0; i < pack; i++)
        load_bias<T>(a, pack > 1 ? hb * pack + i : hb, bias_unit(a, FEAT & kCap), bias + i * attend_bias_len(a.reach), tid, THREADS);
  }
  if (a.q_docs || (FEAT & kBias)) __syncthreads();

  auto next = [&](int t) { return a.q_docs ? next_live(live, t, t_begin, t_end) : t; };

  const Score sc(a, FEAT & kCap);
  const Bias by{(FEAT & kBias) && a.table ? bias + sub * attend_bias_len(a.reach) : nullptr,
                (FEAT & kBias) && a.slopes ? -a.slopes[head] * bias_unit(a, FEAT & kCap) : 0.0f, a.reach};

  v16f acc[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = v16f{};
  // the maximum so far; what scores are taken against
  float m = -INFINITY, ref = 0.0f, sum = 0.0f;

  // The 32 keys from key j0 of the sequence, row r0 of the step in LDS:
  // scores, running maximum and sum, and their part of the output.
  auto tile = [&](int j0, int r0, const char *kl, const char *vl, const int *kd) {
    const bool masked = kd || j0 < lo_max || j0 + 31 > hi_min;
    unsigned bits = ~0u;
    if (masked) {
      bits = row_bits(j0, lo, hi, h);
      if (kd && !docs.tile(kd + r0, lane, &bits)) return;
    }
    const int d0 = j0 + 4 * h - p, near = j0 - p_hi, far = j0 + 31 - p_lo;
    v16f z{};  // a score is z * gain in base 2
    float gain = sc.gain;
    if constexpr (FEAT == kBias) z = by.template at<1>(d0, near, far);
#pragma unroll
    for (int i = 0; i < KS; i++)
      if (within<T>(16 * i, a.dim)) z = mfma16(KV::rows(kl, r0, i, lane), q[i], z);
    if constexpr (FEAT & kCap) {
      tanh_tile<T>(z, sc);
      if constexpr (FEAT & kBias) {
        const v16f b = by.template at<1>(d0, near, far);
#pragma unroll
        for (int r = 0; r < 16; r++) z[r] = __builtin_fmaf(z[r], gain, b[r]);
        gain = 1.0f;
      }
    }
    // The probabilities are taken against an old maximum until they add up
    // to over 2^8: far inside every type's range, so few tiles after a
    // query's first need their own maximum or rescale the sums.
    float part, pr[16];
    auto probabilities = [&] {
      part = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; r++) pr[r] = exp2_fast(__builtin_fmaf(z[r], gain, -ref));
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; r++) pr[r] = if_bit(bits, r, pr[r]);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) part += pr[r];
      return __ballot(!(part <= 256.0f)) != 0;
    };
    bool again = __ballot(bits != 0 && m == -INFINITY) != 0;
    if (!again) again = probabilities();
    if (again) {
      float top = -INFINITY, y[16];
#pragma unroll
      for (int r = 0; r < 16; r++) y[r] = z[r] * gain;
      if (masked) {
#pragma unroll
        for (int r = 0; r < 16; r++) y[r] = or_minus_inf(bits, r, y[r]);
      }
#pragma unroll
      for (int r = 0; r < 16; r++) top = __builtin_fmaxf(top, y[r]);
      top = half_max(top);
      const float next_m = __builtin_fmaxf(m, top);
      const float f = m == -INFINITY ? 0.0f : exp2_fast(m - next_m);
      m = next_m;
      ref = m == -INFINITY ? 0.0f : m;
      sum *= f;
#pragma unroll
      for (int d = 0; d < ND; d++)
#pragma unroll
        for (int r = 0; r < 16; r++) acc[d][r] *= f;
      probabilities();
    }
    sum += part;
    // the probabilities are rounded to the rows' type here, as V is: the
    // product's sum stays in 32 bits
#pragma unroll
    for (int v = 0; v < 2; v++) {
      const Frag pf = pack8<Frag>(pr + 8 * v);
#pragma unroll
      for (int d = 0; d < ND; d++)
        if (within<T>(32 * d, a.dim)) acc[d] = mfma16(KV::cols(vl, r0 + 16 * v, d, lane), pf, acc[d]);
    }
  };

  int buf = 0;
  int t = next(t_begin);
  if (t < t_end) fetch(t);
  while (t < t_end) {
    char *const kl = smem + buf * 2 * KV::BYTES, *const vl = kl + KV::BYTES;
    {
      // padding that no query sees may hold anything: its rows are cleared
      const bool all = a.dim == DT && t * BK + BK <= s.nk && !a.q_docs;
      auto keep = [&](int d) { return !a.q_docs || d >= 0; };
      if (a.q_docs && tid < BK) kdocs[buf * BK + tid] = kdoc < 0 ? -2 : kdoc;
      kt.put(kl, s.nk - t * BK, a.dim, tid, all, tags, keep);
      vt.put(vl, s.nk - t * BK, a.dim, tid, all, tags, keep);
    }
    __syncthreads();
    const int tn = next(t + 1);
    if (tn < t_end) fetch(tn);

    const int j0 = t * BK;
    const int *const kd = a.q_docs ? kdocs + buf * BK : nullptr;
    // a tile at a time: two tiles' scores cost a wave of every SIMD
#pragma unroll 1
    for (int u = 0; u < BK; u += 32)
      if (j0 + u <= hi_max && j0 + u + 31 >= lo_min) tile(j0 + u, u, kl, vl, kd);
    buf ^= 1;
    t = tn;
  }

  sum = half_sum(sum);
  const int64_t row = s.q0 + tok;
  if (x.splits > 1) {
    if (!mine) return;
    const int64_t at = ((int64_t)blockIdx.y * a.nq + row) * a.heads + head;
    float *o = x.part_o + at * a.dim;
#pragma unroll
    for (int d = 0; d < ND; d++)
#pragma unroll
      for (int g = 0; g < 4; g++) {
        const int c = 32 * d + 8 * g + 4 * h;
        if (c < a.dim) *(f4 *)(o + c) = f4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
      }
    if (h == 0) x.part_ml[2 * at] = m, x.part_ml[2 * at + 1] = sum;
    return;
  }
  if (a.lse && mine && h == 0) a.lse[(int64_t)head * a.nq + row] = (ref + __builtin_amdgcn_logf(sum)) * kLn2;
  store_rows<T, DT>(acc, sum > 0.0f ? 1.0f / sum : 0.0f, smem + wave * (32 * DT * (int)sizeof(T)), a.dim, lane, [&](int i) {
    const int r = row0 + wave * 32 + i, tok = token(r);
    if (r >= rows) return (T *)nullptr;
    return (T *)a.o.p + (s.q0 + tok) * a.o.row + (pack > 1 ? hb * pack + r - tok * pack : hb) * a.o.head;
  });
}

// The parts of the keys joined: a thread has four columns of a query's head,
// which it adds up over the parts in their order. Bound by latency: the parts'
// maxima, then their rows (32 x 16 heads of 128, 8.9 us).
template <class T>
__global__ __launch_bounds__(64) void attend_join_kernel(AttendArgs x) {
  const ixh_attend_args &a = x.a;
  const int quads = a.dim / 4;
  const int64_t at = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int64_t rh = at / quads;
  const int c = (int)(at - rh * quads) * 4;
  const int64_t row = rh / a.heads;
  const int head = (int)(rh - row * a.heads);
  if (row >= row_at(a.q_offs, a.B, a.nq) || row < row_at(a.q_offs, 0, a.nq)) return;
  float m = -INFINITY;
  const int64_t step = (int64_t)a.nq * a.heads;
#pragma unroll 8
  for (int i = 0; i < x.splits; i++) m = __builtin_fmaxf(m, x.part_ml[2 * (i * step + rh)]);
  const float ref = m == -INFINITY ? 0.0f : m;
  f4 o{};
  float sum = 0.0f;
#pragma unroll 8
  for (int i = 0; i < x.splits; i++) {
    const float f = exp2_fast(x.part_ml[2 * (i * step + rh)] - ref);
    sum = __builtin_fmaf(f, x.part_ml[2 * (i * step + rh) + 1], sum);
    const f4 v = *(const f4 *)(x.part_o + (i * step + rh) * a.dim + c);
#pragma unroll
    for (int e = 0; e < 4; e++) o[e] = __builtin_fmaf(f, v[e], o[e]);
  }
  const float inv = sum > 0.0f ? 1.0f / sum : 0.0f;
  store4((T *)a.o.p + row * a.o.row + head * a.o.head + c, o * inv);
  if (a.lse && c == 0) a.lse[(int64_t)head * a.nq + row] = (ref + __builtin_amdgcn_logf(sum)) * kLn2;
}

template <class T, int DT, int WAVES, int FEAT>
bool launch(const AttendArgs &x, hipStream_t s) {
  typedef FwdShape<T, DT, WAVES> Sh;
  const int shm = Sh::BIAS + ((FEAT & kBias) && x.a.table ? 4 * x.pack * attend_bias_len(x.a.reach) : 0);
  static PerDevice lds;
  if (!lds_granted(lds, (const void *)attend_fwd_kernel<T, DT, WAVES, FEAT>, 160 << 10)) return false;
  const dim3 grid((unsigned)(x.slots * (x.pack > 1 ? x.a.kv_heads : x.a.heads)), x.splits);
  attend_fwd_kernel<T, DT, WAVES, FEAT><<<grid, Sh::THREADS, shm, s>>>(x);
  return true;
}

template <class T, int DT, int WAVES>
bool by_feat(const AttendArgs &x, hipStream_t s) {
  const bool cap = x.a.cap > 0, bias = x.a.slopes || x.a.table;
  if (cap) return bias ? launch<T, DT, WAVES, 3>(x, s) : launch<T, DT, WAVES, 1>(x, s);
  return bias ? launch<T, DT, WAVES, 2>(x, s) : launch<T, DT, WAVES, 0>(x, s);
}
template <class T>
bool by_dim(const AttendArgs &x, bool few, hipStream_t s) {
  if (x.a.dim <= 64) return few ? by_feat<T, 64, 1>(x, s) : by_feat<T, 64, 4>(x, s);
  return few ? by_feat<T, 128, 1>(x, s) : by_feat<T, 128, 4>(x, s);
}

}  // namespace

bool launch_attend_fwd(const AttendArgs &x, bool few, hipStream_t s) {
  switch (x.a.type) {
    case IXH_TYPE_F32: return by_dim<float>(x, few, s);
    case IXH_TYPE_BF16: return by_dim<__bf16>(x, few, s);
    default: return by_dim<_Float16>(x, few, s);
  }
}

void launch_attend_join(const AttendArgs &x, hipStream_t s) {
  const int64_t n = (int64_t)x.a.nq * x.a.heads * (x.a.dim / 4);
  const unsigned grid = (unsigned)((n + 63) / 64);
  switch (x.a.type) {
    case IXH_TYPE_F32: attend_join_kernel<float><<<grid, 64, 0, s>>>(x); break;
    case IXH_TYPE_BF16: attend_join_kernel<__bf16><<<grid, 64, 0, s>>>(x); break;
    default: attend_join_kernel<_Float16><<<grid, 64, 0, s>>>(x); break;
  }
}

}  // namespace ixh
