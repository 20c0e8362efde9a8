// attend_bwd.hip — the gradients of attend_fwd.hip, from the rows, the
// output and the logarithms of the sums that the forward left.
//
// With P = 2^(z - lse) taken again, dP = dO V^T and delta = dO . o:
//   dZ = P (dP - delta), dS = dZ z'(s),
//   dQ = scale dS K, dK = scale dS^T Q, dV = P^T dO.
// Two kernels, so that no sum crosses workgroups and no result depends on
// an order of atomics: one has a block of queries and runs over the keys
// (dQ), one has a block of keys and runs over the queries of every head that
// shares them (dK, dV and the bias' sums). Both take S and dP again: 7
// products for the 5 of one kernel with atomics.
//
// Precision of 16-bit rows. delta from the rounded o is off by the rounding
// times |dO|, which every dZ of the row inherits. The first kernel's sum of
// a row's dZ is minus that error (the exact ones add up to 0), so it passes
// the second a delta that is right to 32 bits. dQ itself is taken from dS in
// two pieces, rounded and what that took off: an eighth product, in place of
// an error as large as the result's own rounding.
#include "attend_device.h"
#include "ixh_internal.h"

namespace ixh {
namespace {

// 16 products to scores: z * the returned gain in base 2. Under a cap slope_of
// gets their derivative by the product, in units of scale.
template <class T, int FEAT>
__device__ __forceinline__ float shape_scores(v16f &z, float *slope_of, const Score &sc, const v16f &bias) {
  if constexpr (!(FEAT & kCap)) return sc.gain;
  tanh_tile<T>(z, sc);
#pragma unroll
  for (int r = 0; r < 16; r++) {
    slope_of[r] = __builtin_fmaf(-z[r], z[r], 1.0f);
    if constexpr (FEAT & kBias) z[r] = __builtin_fmaf(z[r], sc.gain, bias[r]);
  }
  return FEAT & kBias ? 1.0f : sc.gain;
}

// A block's share of its steps, where they are in parts (blockIdx.y).
__device__ __forceinline__ void part_of(int splits, int *t_begin, int *t_end) {
  if (splits == 1) return;
  const int per = (*t_end - *t_begin + splits - 1) / splits;
  *t_begin = min(*t_begin + per * (int)blockIdx.y, *t_end);
  *t_end = min(*t_begin + per, *t_end);
}

// A lane's columns of one row of a part's sums.
template <int ND>
__device__ __forceinline__ void store_part(const v16f *acc, float *to, int dim, int h) {
#pragma unroll
  for (int d = 0; d < ND; d++)
#pragma unroll
    for (int g = 0; g < 4; g++) {
      const int c = 32 * d + 8 * g + 4 * h;
      if (c < dim) *(f4 *)(to + c) = f4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
    }
}

// ---- dQ ---------------------------------------------------------------------

// As the forward: a lane has a query (row), K and V come through LDS, 32 keys
// a step. S^T, dP^T and dQ (twice, for dS in two pieces) are its products.
// Bound by the issue of vector and matrix instructions (8 sequences of 2,048,
// 16/4 heads of 128, bf16, documents, causal, cap: 245-260 us; 48 sequences of
// 64-512, 12 heads of 64, learned bias: 78 us).

template <class T, int DT>
struct DqShape {
  static constexpr int WAVES = 4, THREADS = 256, ROWS = 128;
  static constexpr int BK = 32;
  typedef Tile<T, DT, BK, THREADS> KV;
  static_assert(4 * KV::BYTES >= WAVES * 32 * DT * (int)sizeof(T), "the result's rows");
  static constexpr int DOCS = 4 * KV::BYTES, LIVE = DOCS + 2 * 4 * BK, BIAS = LIVE + 8 * kDocWords;
};

template <class T, int DT, int FEAT>
__global__ __launch_bounds__(256, sizeof(T) == 4 ? 1 : DT == 64 ? 3 : 2) void attend_dq_kernel(AttendArgs x) {
  typedef DqShape<T, DT> Sh;
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
  const int pack = x.pack, nh = pack > 1 ? a.kv_heads : a.heads;
  const int hb = blockIdx.x % nh, kvh = pack > 1 ? hb : hb / x.group;
  int64_t blk;
  const Seq s = find_block(a, false, ROWS, pack, x.slots - 1 - blockIdx.x / nh, &blk);
  const int rows = s.nq * pack;
  if (blk < 0 || blk * ROWS >= rows) return;  // below 0: offsets that do not ascend
  const int row0 = (int)blk * ROWS, row1 = min(row0 + ROWS, rows);
  auto token = [&](int r) { return pack > 1 ? r / pack : r; };
  const int r = min(row0 + wave * 32 + (lane & 31), rows - 1), tok = token(r), sub = r - tok * pack;
  const int head = pack > 1 ? hb * pack + sub : hb;
  const bool mine = row0 + wave * 32 + (lane & 31) < rows;
  const int p = tok + s.shift;
  int lo, hi;
  key_bounds(a, s, p, &lo, &hi);
  const int p_lo = __builtin_amdgcn_readlane(p, 0), p_hi = __builtin_amdgcn_readlane(p, 31);
  const int lo_min = __builtin_amdgcn_readlane(lo, 0), lo_max = __builtin_amdgcn_readlane(lo, 31);
  const int hi_min = __builtin_amdgcn_readlane(hi, 0);
  const int hi_max = row0 + wave * 32 < rows ? __builtin_amdgcn_readlane(hi, 31) : -1;
  int t_begin, t_end;
  {
    int l, u, unused;
    key_bounds(a, s, token(row0) + s.shift, &l, &unused);
    key_bounds(a, s, token(row1 - 1) + s.shift, &unused, &u);
    t_begin = l / BK;
    t_end = u >= l ? u / BK + 1 : t_begin;
  }
  const bool one_step = t_end - t_begin == 1;
  part_of(x.splits, &t_begin, &t_end);
  const int64_t row = s.q0 + tok;
  const ColumnDocs docs(a.q_docs ? a.q_docs[row] : 0);

  // a row that sees nothing has lse -inf: its dO and o are not read
  const float lse = a.lse[(int64_t)head * a.nq + row];
  const bool alive = lse > -INFINITY;
  const bool dead_rows = __ballot(!alive) != 0;
  const float lse2 = alive ? lse * kLog2e : 0.0f;
  Frag q[KS], dO[KS];
  float delta = 0.0f;
  {
    const T *qr = (const T *)a.q.p + row * a.q.row + head * a.q.head;
    const T *gr = (const T *)x.g.d_out.p + row * x.g.d_out.row + head * x.g.d_out.head;
    const T *orow = (const T *)a.o.p + row * a.o.row + head * a.o.head;
#pragma unroll
    for (int i = 0; i < KS; i++) {
      const bool in = 16 * i + 8 * h < a.dim && alive;
      q[i] = load8(qr + 16 * i + 8 * h, in);
      dO[i] = load8(gr + 16 * i + 8 * h, in);
      const Frag o = load8(orow + 16 * i + 8 * h, in);
#pragma unroll
      for (int e = 0; e < 8; e++) delta = __builtin_fmaf(frag_at(dO[i], e), frag_at(o, e), delta);
    }
    delta = half_sum(delta);
  }
  const T *const kb = (const T *)a.k.p + s.k0 * a.k.row + kvh * a.k.head;
  const T *const vb = (const T *)a.v.p + s.k0 * a.v.row + kvh * a.v.head;
  const Score sc(a, FEAT & kCap);
  const float unit = bias_unit(a, FEAT & kCap);
  const Bias by{(FEAT & kBias) && a.table ? bias + sub * attend_bias_len(a.reach) : nullptr,
                (FEAT & kBias) && a.slopes ? -a.slopes[head] * unit : 0.0f, a.reach};
  if constexpr (FEAT & kBias) {
    if (a.table)
      for (int i = 0; i < pack; i++)
        load_bias<T>(a, pack > 1 ? hb * pack + i : hb, unit, bias + i * attend_bias_len(a.reach), tid, THREADS);
  }
  if (a.q_docs)
    doc_steps<BK, Sh::WAVES>(a.q_docs + s.q0, token(row0), token(row1 - 1), a.k_docs + s.k0, s.nk, t_begin, t_end, live,
                             wave, lane);
  if (a.q_docs || (FEAT & kBias)) __syncthreads();
  auto next = [&](int t) { return a.q_docs ? next_live(live, t, t_begin, t_end) : t; };
  float row_sum = 0.0f;  // of dZ

  v16f acc[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) acc[d] = v16f{};

  KV kt, vt;
  typename KV::Tags tags;
  int kdoc = 0;
  kt.init(a.k.row, a.dim, tid);
  vt.init(a.v.row, a.dim, tid);
  auto fetch = [&](int t) {
    const int left = s.nk - t * BK;
    kt.get(kb + (int64_t)(t * BK) * a.k.row, a.k.row, left, tid);
    vt.get(vb + (int64_t)(t * BK) * a.v.row, a.v.row, left, tid);
    if (a.q_docs) {
      tags.get(a.k_docs + s.k0 + t * BK, left, tid);
      if (tid < BK) kdoc = a.k_docs[s.k0 + t * BK + min(tid, left - 1)];
    }
  };
  int buf = 0, t = next(t_begin);
  if (t < t_end) fetch(t);
  for (int tn; t < t_end; t = tn, buf ^= 1) {
    char *const kl = smem + buf * 2 * KV::BYTES, *const vl = kl + KV::BYTES;
    {
      const bool all = a.dim == DT && t * BK + BK <= s.nk && !a.q_docs;
      auto keep = [&](int d) { return !a.q_docs || d >= 0; };
      if (a.q_docs && tid < BK) kdocs[buf * BK + tid] = kdoc < 0 ? -2 : kdoc;
      kt.put(kl, s.nk - t * BK, a.dim, tid, all, tags, keep);
      vt.put(vl, s.nk - t * BK, a.dim, tid, all, tags, keep);
    }
    __syncthreads();
    tn = next(t + 1);
    if (tn < t_end) fetch(tn);
    const int j0 = t * BK;
    if (j0 > hi_max || j0 + BK <= lo_min) continue;
    const bool masked = a.q_docs || j0 < lo_max || j0 + BK - 1 > hi_min || dead_rows;
    unsigned bits = ~0u;
    if (masked) {
      bits = alive ? row_bits(j0, lo, hi, h) : 0;
      if (a.q_docs && !docs.tile(kdocs + buf * BK, lane, &bits)) continue;
    }

    const int d0 = j0 + 4 * h - p;
    const int near = j0 - p_hi, far = j0 + 31 - p_lo;
    const bool flat = near >= a.reach || far <= -a.reach;
    v16f z = v16f{}, dp = v16f{}, bz = v16f{};
    if constexpr (FEAT & kBias) bz = by.template at<1>(d0, near, far);
    if constexpr (FEAT == kBias) z = bz;
#pragma unroll
    for (int i = 0; i < KS; i++)
      if (within<T>(16 * i, a.dim)) {
        z = mfma16(KV::rows(kl, 0, i, lane), q[i], z);
        dp = mfma16(KV::rows(vl, 0, i, lane), dO[i], dp);
      }
    float by_cap[16];
    const float gain = shape_scores<T, FEAT>(z, by_cap, sc, bz);
    float dz[16];
#pragma unroll
    for (int r = 0; r < 16; r++) dz[r] = exp2_fast(__builtin_fmaf(z[r], gain, -lse2));
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; r++) dz[r] = if_bit(bits, r, dz[r]);
    }
    if (one_step) {
      // all of a row's keys are here: delta without o's rounding
      delta = 0.0f;
#pragma unroll
      for (int r = 0; r < 16; r++) delta = __builtin_fmaf(dz[r], dp[r], delta);
      delta = half_sum(delta);
    }
#pragma unroll
    for (int r = 0; r < 16; r++) dz[r] *= dp[r] - delta;
#pragma unroll
    for (int r = 0; r < 16; r++) row_sum += dz[r];
    if constexpr (FEAT & kCap) {
#pragma unroll
      for (int r = 0; r < 16; r++) dz[r] *= by_cap[r];
    }
    // dS in the rows' type, as K is, and what that rounding took off; scale
    // comes after the sum
#pragma unroll
    for (int v = 0; v < 2; v++) {
      const Frag f = pack8<Frag>(dz + 8 * v);
      Frag rest{};
      if constexpr (sizeof(T) == 2) {
        float off[8];
#pragma unroll
        for (int e = 0; e < 8; e++) off[e] = dz[8 * v + e] - frag_at(f, e);
        rest = pack8<Frag>(off);
      }
#pragma unroll
      for (int d = 0; d < ND; d++)
        if (within<T>(32 * d, a.dim)) {
          const Frag k = KV::cols(kl, 16 * v, d, lane);
          acc[d] = mfma16(k, f, acc[d]);
          if constexpr (sizeof(T) == 2) acc[d] = mfma16(k, rest, acc[d]);
        }
    }
  }

  row_sum = half_sum(row_sum);
  if (x.splits > 1) {
    if (!mine) return;
    store_part<ND>(acc, x.part_o + (((int64_t)blockIdx.y * a.nq + row) * a.heads + head) * a.dim, a.dim, h);
    // one step is the first part's, with the delta that it found
    if (h == 0)
      x.part_delta[((int64_t)blockIdx.y * a.heads + head) * a.nq + row] = (blockIdx.y == 0 ? delta : 0.0f) + row_sum;
    return;
  }
  if (mine && h == 0) x.delta[(int64_t)head * a.nq + row] = delta + row_sum;
  store_rows<T, DT>(acc, a.scale, smem + wave * (32 * DT * (int)sizeof(T)), a.dim, lane, [&](int i) {
    const int r = row0 + wave * 32 + i, tok = token(r);
    if (r >= rows) return (T *)nullptr;
    return (T *)x.g.dq.p + (int64_t)(s.q0 + tok) * x.g.dq.row + (pack > 1 ? hb * pack + r - tok * pack : hb) * x.g.dq.head;
  });
}

// ---- dK, dV -----------------------------------------------------------------

// Four waves have 128 keys, 32 each, and 32 queries a step. A block of keys
// that many queries see holds up a launch of few blocks: there two waves
// share 32 keys (SHARE 2), each with every other 32 queries of a step of 64,
// and add their sums up at the end. attend_api.cpp says when.
// A lane has a key, whose dK and dV stay in registers; K and V are fragments
// in registers, Q and dO come through LDS for both uses, by rows for S and dP,
// transposed for dK and dV. At heads over 64 the sums take a SIMD's registers,
// so that one wave's products, vector work and LDS reads follow one another
// (about 2.7 us a step of 64 queries): that, not a rate, is what bounds it (8
// sequences of 2,048, 16/4 heads of 128, bf16, documents, causal, cap: 410-430
// us; 48 sequences of 64-512, 12 heads of 64, learned bias with its gradient:
// 122 us; 24 of 33-300, 6 heads of 48, float32: 69).
template <class T, int DT, int SHARE>
struct DkvShape {
  static constexpr int WAVES = 4, THREADS = 256, KEYS = 128 / SHARE;
  static constexpr int BQ = 32 * SHARE;
  typedef Tile<T, DT, BQ, THREADS> QO;
  static_assert(4 * QO::BYTES >= WAVES * 32 * DT * (int)sizeof(T), "the result's rows");
  // Q and dO twice, then lse, delta and the documents of the rows twice
  static constexpr int STAT = 4 * QO::BYTES, DOCS = STAT + 4 * 4 * BQ, LIVE = DOCS + 2 * 4 * BQ,
                       BIAS = LIVE + 8 * kDocWords;
};

template <class T, int DT, int FEAT, int SHARE>
__global__ __launch_bounds__(256, sizeof(T) == 4 || DT == 128 ? 1 : 2) void attend_dkv_kernel(AttendArgs x) {
  typedef DkvShape<T, DT, SHARE> Sh;
  typedef typename Sh::QO QO;
  typedef typename Kind<T>::frag Frag;
  constexpr int THREADS = Sh::THREADS, KEYS = Sh::KEYS, BQ = Sh::BQ, KS = DT / 16, ND = DT / 32;
  extern __shared__ __attribute__((aligned(16))) char smem[];
  const ixh_attend_args &a = x.a;
  const int tid = threadIdx.x, lane = tid & 63, h = lane >> 5;
  const int wave = __builtin_amdgcn_readfirstlane(tid >> 6);
  const int kw = wave / SHARE, qw = wave % SHARE;  // the wave's keys, its queries of a step
  float *const stat = (float *)(smem + Sh::STAT);
  int *const qdocs = (int *)(smem + Sh::DOCS);
  uint64_t *const live = (uint64_t *)(smem + Sh::LIVE);
  // the bias of two heads in turn; the sums of dZ by distance, an array each
  // wave, with the bias' ends
  float *const bias = (float *)(smem + Sh::BIAS);
  const int span = 2 * a.reach + 1, len = attend_bias_len(a.reach);
  float *const dist = bias + 2 * len, *const my_dist = dist + wave * len;
  const bool grad_table = (FEAT & kBias) && x.dist;

  const int kvh = blockIdx.x % a.kv_heads;
  int64_t blk;
  const Seq s = find_block(a, true, KEYS, 1, blockIdx.x / a.kv_heads, &blk);
  const int64_t slot = blockIdx.x / a.kv_heads * x.splits + blockIdx.y;
  if (blk < 0 || blk * KEYS >= s.nk) {
    if (grad_table)
      for (int g = 0; g < x.group; g++)
        for (int i = tid; i < span; i += THREADS) x.dist[(slot * a.heads + kvh * x.group + g) * span + i] = 0.0f;
    return;
  }
  const int first = (int)(blk * KEYS);
  const int key = min(first + kw * 32 + (lane & 31), s.nk - 1);
  int lo, hi;  // places of the queries that see the key
  query_bounds(a, s, key, &lo, &hi);
  const int k_lo = __builtin_amdgcn_readlane(key, 0), k_hi = __builtin_amdgcn_readlane(key, 31);
  const int lo_min = __builtin_amdgcn_readlane(lo, 0), lo_max = __builtin_amdgcn_readlane(lo, 31);
  const int hi_min = __builtin_amdgcn_readlane(hi, 0);
  const bool mine = first + kw * 32 + (lane & 31) < s.nk;
  const int hi_max = first + kw * 32 < s.nk ? __builtin_amdgcn_readlane(hi, 31) : INT32_MIN;
  int t_begin, t_end;  // steps of BQ queries
  {
    int l, u, unused;
    query_bounds(a, s, first, &l, &unused);
    query_bounds(a, s, min(first + KEYS, s.nk) - 1, &unused, &u);
    l -= s.shift, u -= s.shift;
    t_begin = max(l, 0) / BQ;
    t_end = u >= max(l, 0) ? min(u, s.nq - 1) / BQ + 1 : t_begin;
    if (t_end < t_begin) t_end = t_begin;
    part_of(x.splits, &t_begin, &t_end);
  }
  const int64_t row = s.k0 + key;
  const ColumnDocs docs(a.k_docs ? a.k_docs[row] : 0);
  const bool alive = docs.doc >= 0;

  Frag k[KS], v[KS];
  {
    const T *kr = (const T *)a.k.p + row * a.k.row + kvh * a.k.head;
    const T *vr = (const T *)a.v.p + row * a.v.row + kvh * a.v.head;
#pragma unroll
    for (int i = 0; i < KS; i++) {
      const bool in = 16 * i + 8 * h < a.dim && alive;
      k[i] = load8(kr + 16 * i + 8 * h, in);
      v[i] = load8(vr + 16 * i + 8 * h, in);
    }
  }
  if (a.q_docs) {
    doc_steps<BQ, Sh::WAVES>(a.k_docs + s.k0, first, min(first + KEYS, s.nk) - 1, a.q_docs + s.q0, s.nq, t_begin, t_end,
                             live, wave, lane);
    __syncthreads();
  }
  auto next = [&](int t) { return a.q_docs ? next_live(live, t, t_begin, t_end) : t; };
  const int t_first = next(t_begin);
  const Score sc(a, FEAT & kCap);
  v16f dk[ND], dv[ND];
#pragma unroll
  for (int d = 0; d < ND; d++) dk[d] = v16f{}, dv[d] = v16f{};

  // A step's rows on their way: in registers while the step before it is
  // computed.
  struct {
    QO q, g;
    typename QO::Tags tags;
    float lse, delta;
    int doc;
  } e;
  auto fetch = [&](int g, int t) {
    const int head = kvh * x.group + g, left = s.nq - t * BQ;
    const int64_t row = s.q0 + t * BQ;
    e.q.get((const T *)a.q.p + row * a.q.row + head * a.q.head, a.q.row, left, tid);
    e.g.get((const T *)x.g.d_out.p + row * x.g.d_out.row + head * x.g.d_out.head, x.g.d_out.row, left, tid);
    const int64_t at = (int64_t)head * a.nq + row;
    // a row that sees nothing has lse -inf
    e.tags.get((const int32_t *)a.lse + at, left, tid);
    const int r = min(tid, left - 1);
    e.lse = a.lse[at + r];
    e.delta = x.delta[at + r];
    e.doc = (a.q_docs ? a.q_docs + row : (const int32_t *)a.lse + at)[r];
  };
  auto put = [&](int t, int buf) {
    // such rows, and those past the last, are cleared: P is 0 at -inf
    char *const ql = smem + buf * 2 * QO::BYTES;
    const int left = s.nq - t * BQ;
    if (tid < BQ) {
      float *const st = stat + buf * 2 * BQ;
      const bool there = e.lse > -INFINITY && tid < left;
      st[tid] = there ? e.lse * -kLog2e : -INFINITY;
      st[BQ + tid] = there ? e.delta : 0.0f;
      if (a.q_docs) qdocs[buf * BQ + tid] = e.doc < 0 ? -2 : e.doc;
    }
    auto keep = [&](int l) { return __builtin_bit_cast(float, l) > -INFINITY; };
    e.q.put(ql, left, a.dim, tid, false, e.tags, keep);
    e.g.put(ql + QO::BYTES, left, a.dim, tid, false, e.tags, keep);
  };
  e.q.init(a.q.row, a.dim, tid);
  e.g.init(x.g.d_out.row, a.dim, tid);

  float below = 0.0f, above = 0.0f;  // dZ at distances of -reach and less, reach and more
  auto clear_dist = [&] {
    for (int i = lane; i < len; i += 64) my_dist[i] = 0.0f;
    below = above = 0.0f;
  };
  // A head's sums: the ends' lanes in a fixed order, the waves' arrays, and
  // what lies past the reach, which is the ends' too.
  auto write_dist = [&](int g) {
#pragma unroll
    for (int o = 1; o < 64; o <<= 1) {
      above += __shfl_xor(above, o);
      below += __shfl_xor(below, o);
    }
    if (lane == 0) my_dist[0] += below, my_dist[len - 1] += above;
    __syncthreads();
    for (int i = tid; i < len; i += THREADS) {
      float v = 0.0f;
#pragma unroll
      for (int w = 0; w < Sh::WAVES; w++) v += dist[w * len + i];
      dist[i] = v;
    }
    __syncthreads();
    float *const out = x.dist + (slot * a.heads + kvh * x.group + g) * span;
    for (int i = tid; i < span; i += THREADS) {
      float v = dist[i + kBiasPad];
      if (i == 0)
        for (int e = 0; e < kBiasPad; e++) v += dist[e];
      if (i == span - 1)
        for (int e = 1; e <= kBiasPad; e++) v += dist[i + kBiasPad + e];
      out[i] = v;
    }
    __syncthreads();
  };
  auto compute = [&](int g, int t, int buf) {
    const int r0 = 32 * qw, p0 = t * BQ + r0 + s.shift;  // the wave's first row, its place
    if (p0 > hi_max || p0 + 32 <= lo_min) return;
    const bool masked = a.q_docs || p0 < lo_max || p0 + 31 > hi_min;
    unsigned bits = ~0u;
    if (masked) {
      bits = row_bits(p0, lo, hi, h);
      if (a.q_docs && !docs.tile(qdocs + buf * BQ + r0, lane, &bits)) return;
    }
    const char *const ql = smem + buf * 2 * QO::BYTES, *const gl = ql + QO::BYTES;
    const float *const st = stat + buf * 2 * BQ + r0;
    v16f z = v16f{}, dp = v16f{}, bz = v16f{};
    if constexpr (FEAT & kBias) {
      const Bias by{a.table ? bias + (g & 1) * len : nullptr,
                    a.slopes ? -a.slopes[kvh * x.group + g] * bias_unit(a, FEAT & kCap) : 0.0f, a.reach};
      bz = by.template at<-1>(key - p0 - 4 * h, k_lo - p0 - 31, k_hi - p0);
    }
    if constexpr (FEAT == kBias) z = bz;
#pragma unroll
    for (int i = 0; i < KS; i++)
      if (within<T>(16 * i, a.dim)) {
        z = mfma16(QO::rows(ql, r0, i, lane), k[i], z);
        dp = mfma16(QO::rows(gl, r0, i, lane), v[i], dp);
      }
    float by_cap[16], pr[16], ds[16];
    const float gain = shape_scores<T, FEAT>(z, by_cap, sc, bz);
#pragma unroll
    for (int g4 = 0; g4 < 4; g4++) {
      const f4 less = *(const f4 *)(st + 8 * g4 + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; e++) pr[4 * g4 + e] = exp2_fast(__builtin_fmaf(z[4 * g4 + e], gain, less[e]));
    }
    if (masked) {
#pragma unroll
      for (int r = 0; r < 16; r++) pr[r] = if_bit(bits, r, pr[r]);
    }
#pragma unroll
    for (int g4 = 0; g4 < 4; g4++) {
      const f4 dl = *(const f4 *)(st + BQ + 8 * g4 + 4 * h);
#pragma unroll
      for (int e = 0; e < 4; e++) {
        const int r = 4 * g4 + e;
        ds[r] = pr[r] * (dp[r] - dl[e]);
      }
    }
    if constexpr (FEAT & kBias) {
      if (grad_table) {
        float dz[16];
#pragma unroll
        for (int r = 0; r < 16; r++) dz[r] = mine ? ds[r] : 0.0f;
        const int near = k_lo - p0 - 31, far = k_hi - p0;
        if (near >= a.reach || far <= -a.reach) {
          float part = 0.0f;
#pragma unroll
          for (int r = 0; r < 16; r++) part += dz[r];
          if (near >= a.reach)
            above += part;
          else
            below += part;
        } else {
          // Along the tile's diagonals: a row of 64 lanes moves one lane up
          // for each query and takes up that query's 32 values, so that
          // lane l ends with the sum at distance k_lo - p0 - 31 + l. A swap
          // with zeros gives both halves' queries as such rows. Two chains
          // of 16 queries, for the adds' latency; the first, 16 lanes low,
          // is brought up at the end. (LDS adds by distance took 128 cycles
          // an instruction: 302 -> 86 us over 48 sequences of 64-512.)
          float row[2] = {};
#pragma unroll
          for (int g = 0; g < 2; g++) {
            float up[2][4], dn[2][4];
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
              for (int c = 0; c < 2; c++) halves_apart(dz[4 * (2 * c + g) + e], &up[c][e], &dn[c][e]);
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
              for (int c = 0; c < 2; c++) row[c] = lane_up(row[c]) + up[c][e];
#pragma unroll
            for (int e = 0; e < 4; e++)
#pragma unroll
              for (int c = 0; c < 2; c++) row[c] = lane_up(row[c]) + dn[c][e];
          }
          const float low = __shfl(row[0], lane - 16);
          my_dist[near + lane + a.reach + kBiasPad] += (lane >= 16 ? low : 0.0f) + row[1];
        }
      }
    }
    if constexpr (FEAT & kCap) {
#pragma unroll
      for (int r = 0; r < 16; r++) ds[r] *= by_cap[r];
    }
    // P and dS are rounded to the rows' type, as dO and Q are
#pragma unroll
    for (int w = 0; w < 2; w++) {
      const Frag pf = pack8<Frag>(pr + 8 * w), sf = pack8<Frag>(ds + 8 * w);
#pragma unroll
      for (int d = 0; d < ND; d++) {
        if (!within<T>(32 * d, a.dim)) continue;
        dv[d] = mfma16(QO::cols(gl, r0 + 16 * w, d, lane), pf, dv[d]);
        dk[d] = mfma16(QO::cols(ql, r0 + 16 * w, d, lane), sf, dk[d]);
      }
    }
  };

  // The steps of every head that shares the keys, one after another.
  auto bias_of = [&](int g) {
    if constexpr (FEAT & kBias)
      if (a.table)
        load_bias<T>(a, kvh * x.group + g, bias_unit(a, FEAT & kCap), bias + (g & 1) * len, tid,
                     THREADS);
  };
  const bool any = t_first < t_end;
  if constexpr (FEAT & kBias)
    if (grad_table) {
      clear_dist();
      if (!any)
        for (int g = 0; g < x.group; g++) write_dist(g);
    }
  if (any) {
    fetch(0, t_first);
    bias_of(0);
    put(t_first, 0);
  }
  for (int g = 0, t = t_first, buf = 0; any && g < x.group; buf ^= 1) {
    int then_g = g, then = next(t + 1);
    if (then >= t_end) then_g++, then = t_first;
    const bool more = then_g < x.group;
    __syncthreads();
    if (more) fetch(then_g, then);
    compute(g, t, buf);
    if constexpr (FEAT & kBias)
      if (grad_table && then_g != g) {
        write_dist(g);
        clear_dist();
      }
    if (more) {
      if (then_g != g) bias_of(then_g);
      put(then, buf ^ 1);
    }
    g = then_g, t = then;
  }
  if constexpr (SHARE == 2) {
    // the second wave's sums, through LDS to the first: dK's, then dV's
    static_assert(4 * QO::BYTES >= 2 * 64 * 16 * ND * 4, "");
    f4 *const sums = (f4 *)smem + kw * 64 * 4 * ND + lane;
    auto meet = [&](v16f *acc) {
      __syncthreads();
      if (qw == 1)
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int g = 0; g < 4; g++)
            sums[64 * (4 * d + g)] = f4{acc[d][4 * g], acc[d][4 * g + 1], acc[d][4 * g + 2], acc[d][4 * g + 3]};
      __syncthreads();
      if (qw == 0)
#pragma unroll
        for (int d = 0; d < ND; d++)
#pragma unroll
          for (int g = 0; g < 4; g++) {
            const f4 v = sums[64 * (4 * d + g)];
#pragma unroll
            for (int e = 0; e < 4; e++) acc[d][4 * g + e] += v[e];
          }
    };
    meet(dk);
    meet(dv);
  }
  if (x.splits > 1) {
    int r = first + kw * 32 + (lane & 31);
    asm volatile("" : "+v"(r));
    if (qw != 0 || r >= s.nk) return;
    float *const part = x.part_o + (((int64_t)blockIdx.y * 2 * a.nk + s.k0 + r) * a.kv_heads + kvh) * a.dim;
    store_part<ND>(dk, part, a.dim, h);
    store_part<ND>(dv, part + (int64_t)a.nk * a.kv_heads * a.dim, a.dim, h);
    return;
  }
  auto to = [&](const ixh_heads &t) {
    return [&, t](int i) {
      const int r = first + kw * 32 + i;
      return qw == 0 && r < s.nk ? (T *)t.p + (int64_t)(s.k0 + r) * t.row + kvh * t.head : (T *)nullptr;
    };
  };
  char *const mine_lds = smem + wave * (32 * DT * (int)sizeof(T));
  store_rows<T, DT>(dk, a.scale, mine_lds, a.dim, lane, to(x.g.dk));
  store_rows<T, DT>(dv, 1.0f, mine_lds, a.dim, lane, to(x.g.dv));
}

// The parts of dQ (and of delta), or of dK and dV (blockIdx.y), in their
// order: a thread has four columns of a head's row.
template <class T>
__global__ __launch_bounds__(64) void attend_sum_kernel(AttendArgs x, bool keys) {
  const ixh_attend_args &a = x.a;
  const int quads = a.dim / 4, heads = keys ? a.kv_heads : a.heads, n = keys ? a.nk : a.nq;
  const int64_t at = (int64_t)blockIdx.x * 64 + threadIdx.x;
  const int64_t rh = at / quads;
  const int c = (int)(at - rh * quads) * 4;
  const int64_t row = rh / heads;
  const int head = (int)(rh - row * heads);
  const int *const offs = keys ? a.k_offs : a.q_offs;
  if (row >= row_at(offs, a.B, n) || row < row_at(offs, 0, n)) return;
  const int64_t step = (int64_t)n * heads * a.dim;
  const float *const p = x.part_o + blockIdx.y * step + rh * a.dim + c;
  f4 v{};
#pragma unroll 8
  for (int i = 0; i < x.splits; i++) v += *(const f4 *)(p + i * step * (keys ? 2 : 1));
  const ixh_heads &to = !keys ? x.g.dq : blockIdx.y ? x.g.dv : x.g.dk;
  store4((T *)to.p + row * to.row + head * to.head + c, v * (blockIdx.y ? 1.0f : a.scale));
  if (!keys && c == 0) {
    float delta = 0.0f;
    for (int i = 0; i < x.splits; i++) delta += x.part_delta[((int64_t)i * heads + head) * n + row];
    x.delta[(int64_t)head * n + row] = delta;
  }
}

// ---- the table's gradient ----------------------------------------------------

// Sums of dZ by distance over the workgroups of attend_dkv_kernel: a part of
// them each block, four strands a distance. Bound by latency (12 heads, reach
// 128, 160 workgroups a head: 4.8 us).
__global__ __launch_bounds__(256) void attend_dist_kernel(AttendArgs x) {
  __shared__ float strand[4][64];
  const int span = 2 * x.a.reach + 1, head = blockIdx.y, part = blockIdx.z;
  const int i = blockIdx.x * 64 + (threadIdx.x & 63), w = threadIdx.x >> 6;
  const int64_t per = (x.slots + x.dist_parts - 1) / x.dist_parts;
  const int64_t end = min(x.slots, (part + 1) * per);
  float v = 0.0f;
  if (i < span)
#pragma unroll 8
    for (int64_t slot = part * per + w; slot < end; slot += 4) v += x.dist[(slot * x.a.heads + head) * span + i];
  strand[w][threadIdx.x & 63] = v;
  __syncthreads();
  if (w == 0 && i < span)
    x.dist_sum[((int64_t)part * x.a.heads + head) * span + i] =
        (strand[0][threadIdx.x] + strand[1][threadIdx.x]) + (strand[2][threadIdx.x] + strand[3][threadIdx.x]);
}

// The distances of each bucket: a block a head, 256 / n_buckets strands a
// bucket (at least one), each of its distances in ascending order. Bound by
// the latency of its steps, loads and adds eight at a time (12 heads, reach
// 128, 32 buckets: 6 us, 10 one by one).
template <class T>
__global__ __launch_bounds__(256) void attend_dtable_kernel(AttendArgs x) {
  extern __shared__ __attribute__((aligned(16))) char smem[];
  __shared__ float strand[256];
  const int span = 2 * x.a.reach + 1, head = blockIdx.x, nb = x.a.n_buckets;
  float *const sum = (float *)smem;
  int *const of = (int *)(sum + span);
  for (int i = threadIdx.x; i < span; i += 256) {
    float v = 0.0f;
#pragma unroll 8
    for (int part = 0; part < x.dist_parts; part++) v += x.dist_sum[((int64_t)part * x.a.heads + head) * span + i];
    sum[i] = v;
    of[i] = x.a.buckets[i];
  }
  __syncthreads();
  const int strands = max(256 / nb, 1), per = (span + strands - 1) / strands;
  const int w = nb < 256 ? threadIdx.x / nb : 0;
  for (int b0 = 0; b0 < nb; b0 += 256) {
    const int b = b0 + (nb < 256 ? threadIdx.x % nb : threadIdx.x);
    float v = 0.0f;
    if (b < nb && w < strands)
#pragma unroll 8
      for (int i = w * per; i < min(span, (w + 1) * per); i++) v += of[i] == b ? sum[i] : 0.0f;
    strand[threadIdx.x] = v;
    __syncthreads();
    if (w == 0 && b < nb) {
      for (int i = 1; i < strands; i++) v += strand[i * nb + b];
      ((T *)x.g.dtable)[(int64_t)b * x.a.heads + head] = (T)v;
    }
    __syncthreads();
  }
}

template <class T, int DT, int FEAT>
bool run_dq(const AttendArgs &x, hipStream_t s) {
  typedef DqShape<T, DT> Sh;
  const int len = (FEAT & kBias) && x.a.table ? attend_bias_len(x.a.reach) : 0;
  const int shm = Sh::BIAS + 4 * x.pack * len;
  static PerDevice lds;
  if (!lds_granted(lds, (const void *)attend_dq_kernel<T, DT, FEAT>, 160 << 10)) return false;
  const dim3 grid((unsigned)(x.slots * (x.pack > 1 ? x.a.kv_heads : x.a.heads)), x.splits);
  attend_dq_kernel<T, DT, FEAT><<<grid, Sh::THREADS, shm, s>>>(x);
  return true;
}
template <class T, int DT, int FEAT, int SHARE>
bool run_dkv_shared(const AttendArgs &x, hipStream_t s) {
  typedef DkvShape<T, DT, SHARE> Sh;
  const int len = (FEAT & kBias) && x.a.table ? attend_bias_len(x.a.reach) : 0;
  const int shm = Sh::BIAS + 4 * len * (2 + Sh::WAVES);
  static PerDevice lds;
  if (!lds_granted(lds, (const void *)attend_dkv_kernel<T, DT, FEAT, SHARE>, 160 << 10)) return false;
  attend_dkv_kernel<T, DT, FEAT, SHARE><<<dim3((unsigned)(x.slots * x.a.kv_heads), x.splits), Sh::THREADS, shm, s>>>(x);
  return true;
}
template <class T, int DT, int FEAT>
bool run_dkv(const AttendArgs &x, hipStream_t s) {
  if constexpr (sizeof(T) == 4 && DT == 128)
    return run_dkv_shared<T, DT, FEAT, 1>(x, s);
  else if constexpr (sizeof(T) == 2 && DT == 64)
    return x.share == 1 ? run_dkv_shared<T, DT, FEAT, 1>(x, s) : run_dkv_shared<T, DT, FEAT, 2>(x, s);
  else
    return run_dkv_shared<T, DT, FEAT, 2>(x, s);
}

template <class T, int DT>
bool by_feat(const AttendArgs &x, bool dq, hipStream_t s) {
  const bool cap = x.a.cap > 0, bias = x.a.slopes || x.a.table;
  if (dq) {
    if (cap) return bias ? run_dq<T, DT, 3>(x, s) : run_dq<T, DT, 1>(x, s);
    return bias ? run_dq<T, DT, 2>(x, s) : run_dq<T, DT, 0>(x, s);
  }
  if (cap) return bias ? run_dkv<T, DT, 3>(x, s) : run_dkv<T, DT, 1>(x, s);
  return bias ? run_dkv<T, DT, 2>(x, s) : run_dkv<T, DT, 0>(x, s);
}
bool by_type(const AttendArgs &x, bool dq, hipStream_t s) {
  const bool small = x.a.dim <= 64;
  switch (x.a.type) {
    case IXH_TYPE_F32: return small ? by_feat<float, 64>(x, dq, s) : by_feat<float, 128>(x, dq, s);
    case IXH_TYPE_BF16: return small ? by_feat<__bf16, 64>(x, dq, s) : by_feat<__bf16, 128>(x, dq, s);
    default: return small ? by_feat<_Float16, 64>(x, dq, s) : by_feat<_Float16, 128>(x, dq, s);
  }
}

}  // namespace

bool launch_attend_dq(const AttendArgs &x, hipStream_t s) { return by_type(x, true, s); }
bool launch_attend_dkv(const AttendArgs &x, hipStream_t s) { return by_type(x, false, s); }

void launch_attend_sum(const AttendArgs &x, bool keys, hipStream_t s) {
  const int64_t n = (int64_t)(keys ? x.a.nk : x.a.nq) * (keys ? x.a.kv_heads : x.a.heads) * (x.a.dim / 4);
  const dim3 grid((unsigned)((n + 63) / 64), keys ? 2 : 1);
  switch (x.a.type) {
    case IXH_TYPE_F32: attend_sum_kernel<float><<<grid, 64, 0, s>>>(x, keys); break;
    case IXH_TYPE_BF16: attend_sum_kernel<__bf16><<<grid, 64, 0, s>>>(x, keys); break;
    default: attend_sum_kernel<_Float16><<<grid, 64, 0, s>>>(x, keys); break;
  }
}

void launch_attend_dtable(const AttendArgs &x, hipStream_t s) {
  const int span = 2 * x.a.reach + 1;
  if (x.dist_sum != x.dist) attend_dist_kernel<<<dim3((span + 63) / 64, x.a.heads, x.dist_parts), 256, 0, s>>>(x);
  const int shm = 8 * span;
  switch (x.a.type) {
    case IXH_TYPE_F32: attend_dtable_kernel<float><<<x.a.heads, 256, shm, s>>>(x); break;
    case IXH_TYPE_BF16: attend_dtable_kernel<__bf16><<<x.a.heads, 256, shm, s>>>(x); break;
    default: attend_dtable_kernel<_Float16><<<x.a.heads, 256, shm, s>>>(x); break;
  }
}

}  // namespace ixh
