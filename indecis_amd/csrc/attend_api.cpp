// attend_api.cpp — the entry points of the float attention operators: the
// arguments' checks, the choice of kernels, the workspaces.
#include <hip/hip_runtime.h>

#include <algorithm>
#include <cmath>
#include <cstdarg>
#include <cstdio>
#include <exception>
#include <vector>

#include "attend.h"
#include "ixh_internal.h"

using namespace ixh;

namespace {

int fail(int code, const char *fmt, ...) {
  char buf[512];
  va_list ap;
  va_start(ap, fmt);
  vsnprintf(buf, sizeof buf, fmt, ap);
  va_end(ap);
  return set_error(code, buf);
}

// A failed call also leaves its error as the thread's last error, which a
// later check would report as its own: it is taken back here.
int hip_fail(hipError_t e, const char *what) {
  (void)hipGetLastError();
  return fail(IXH_EHIP, "linalg: hip: %s (%s)", hipGetErrorString(e), what);
}
int launched(const char *what) {
  const hipError_t e = hipGetLastError();
  return e == hipSuccess ? IXH_OK : fail(IXH_EHIP, "linalg: hip: %s (launch %s)", hipGetErrorString(e), what);
}

struct OnDevice {
  int prev = -1;
  hipError_t err;
  explicit OnDevice(int dev) {
    if (hipGetDevice(&prev) != hipSuccess) prev = -1;
    err = prev == dev ? hipSuccess : hipSetDevice(dev);
    if (prev == dev) prev = -1;
  }
  ~OnDevice() {
    if (prev >= 0) (void)hipSetDevice(prev);
  }
};

int type_size(int type) { return type == IXH_TYPE_F32 ? 4 : 2; }
bool type_ok(int type) { return type == IXH_TYPE_F32 || type == IXH_TYPE_BF16 || type == IXH_TYPE_F16; }
bool aligned(const void *p) { return ((uintptr_t)p & 15) == 0; }
int64_t up(int64_t n) { return (n + 255) / 256 * 256; }

int check_heads(const char *op, const char *name, const ixh_heads &t, int type) {
  const int v = 16 / type_size(type);
  if (!t.p) return fail(IXH_EINVAL, "linalg: %s: %s is missing", op, name);
  // a thread's place in a tile of rows is a 32-bit offset: 32 rows
  if (!aligned(t.p) || t.row % v || t.head % v || t.row < 0 || t.head < 0 || t.row >= (1LL << 27) / type_size(type))
    return fail(IXH_EINVAL,
                "linalg: %s: %s needs a pointer and strides that are multiples of 16 bytes, rows less than 2^27 bytes "
                "apart (strides %lld, %lld values of %d bytes)",
                op, name, (long long)t.row, (long long)t.head, type_size(type));
  return IXH_OK;
}

// ---- attention --------------------------------------------------------------

// Reach 1024 is 8 KB of table a head in LDS and 64 KB of sums in the dQ
// kernel, beside 32 to 64 KB of keys.
constexpr int kMaxReach = 1024, kMaxBuckets = 65536, kMaxRows = 1 << 30;
constexpr int64_t kMaxGrid = (1LL << 24) - 1;  // workgroups: a launch has fewer than 2^32 threads along x
constexpr int kCus = 256;
constexpr int kMaxSplits = 64;
constexpr int kMaxDistParts = 16;

// The sizes, apart from pointers.
int check_sizes(const ixh_attend_args *a) {
  if (!a) return fail(IXH_EINVAL, "linalg: Attend: no arguments");
  if (!type_ok(a->type)) return fail(IXH_EINVAL, "linalg: Attend: type %d", a->type);
  if (a->B < 0 || a->nq < 0 || a->nk < 0 || a->nq > kMaxRows || a->nk > kMaxRows || a->B > kMaxRows)
    return fail(IXH_EINVAL, "linalg: Attend: %d sequences of %d queries and %d keys (0 to 2^30 each)", a->B, a->nq, a->nk);
  if (a->dim < 8 || a->dim > 128 || a->dim % 8)
    return fail(IXH_EINVAL, "linalg: Attend: head dimension %d not supported (a multiple of 8 up to 128)", a->dim);
  if (a->kv_heads < 1 || a->heads < 1 || a->heads > 65535 || a->heads % a->kv_heads)
    return fail(IXH_EINVAL, "linalg: Attend: %d heads over %d key heads", a->heads, a->kv_heads);
  if (a->table && (a->reach < 1 || a->reach > kMaxReach || a->n_buckets < 1 || a->n_buckets > kMaxBuckets))
    return fail(IXH_EINVAL, "linalg: Attend: a table of %d buckets, reach %d (1 to %d, 1 to %d)", a->n_buckets, a->reach,
                kMaxBuckets, kMaxReach);
  return IXH_OK;
}

int check_attend(const ixh_attend_args *a) {
  if (int rc = check_sizes(a)) return rc;
  // a bias is taken in units of 1 / scale, a capped score in units of cap
  const bool scale_ok = a->scale >= 1e-10f && a->scale <= 1e10f, cap_ok = a->cap == 0 || (a->cap >= 1e-10f && a->cap <= 1e10f);
  if (!scale_ok || !cap_ok)
    return fail(IXH_EINVAL, "linalg: Attend: scale %g (1e-10 to 1e10), cap %g (the same, or 0)", (double)a->scale,
                (double)a->cap);
  if (a->prefix && !a->causal) return fail(IXH_EINVAL, "linalg: Attend: a prefix needs causal");
  if (a->B == 0) return IXH_OK;
  if (!a->q_offs) return fail(IXH_EINVAL, "linalg: Attend: q_offs is missing");
  if (!a->k_offs && a->nk != a->nq)
    return fail(IXH_EINVAL, "linalg: Attend: %d keys for %d queries need k_offs", a->nk, a->nq);
  if (a->k_docs && !a->q_docs) return fail(IXH_EINVAL, "linalg: Attend: k_docs without q_docs");
  if (a->q_docs && !a->k_docs && a->nk != a->nq)
    return fail(IXH_EINVAL, "linalg: Attend: %d keys for %d queries need k_docs", a->nk, a->nq);
  if (a->table && !a->buckets) return fail(IXH_EINVAL, "linalg: Attend: a table needs buckets");
  int rc;
  if (a->nq > 0 && ((rc = check_heads("Attend", "q", a->q, a->type)) || (rc = check_heads("Attend", "o", a->o, a->type))))
    return rc;
  if (a->nk > 0 && ((rc = check_heads("Attend", "k", a->k, a->type)) || (rc = check_heads("Attend", "v", a->v, a->type))))
    return rc;
  return IXH_OK;
}

struct Plan {
  bool few;
  int64_t work;  // bytes of workspace
};

// Whether the heads that share a key head become rows of one block: it then
// takes fewer tokens, so that short sequences fill it and masks cut it finer
// (16/4 heads of 128, 64 sequences, 512 keys, bf16: 1 token 50 -> 22 us, 16
// tokens 61 -> 33, 32 tokens 68 -> 31). Each head's bias is in LDS.
int pack_of(const ixh_attend_args &a) {
  const int group = a.heads / a.kv_heads;
  const bool fits = !a.table || 4LL * group * attend_bias_len(a.reach) <= 32 << 10;
  return fits && (int64_t)a.nq * group <= INT32_MAX ? group : 1;
}

// The forward's kernels. Everything goes by the mean length: the lengths
// themselves are on the device.
Plan plan_forward(AttendArgs &x) {
  ixh_attend_args &a = x.a;
  Plan p{};
  x.group = a.heads / a.kv_heads;
  x.pack = pack_of(a);
  const int64_t B = std::max(a.B, 1);
  // blocks of one wave where most would have one or two waves' rows (bf16, 12
  // heads of 64, 256 sequences: 8 tokens 12 against 22 us with four waves, 32
  // 15 / 25, 64 27 / 29, 96 45 / 37; 16 heads of 128, 64 sequences: 24 tokens
  // 13 / 16, 48 22 / 20)
  p.few = (int64_t)a.nq * x.pack <= (a.dim <= 64 ? 64 : 32) * B;
  const int rows = p.few ? kAttendRowsFew : kAttendRowsMany;
  x.slots = attend_slots(a.nq, a.B, rows, x.pack);
  const int64_t groups = x.slots * (x.pack > 1 ? a.kv_heads : a.heads);
  const int64_t steps = a.nk / B / attend_keys(type_size(a.type), p.few);
  x.splits = 1;
  // few blocks: their keys in parts, until the chip is full (bf16, 12 heads of
  // 64: 1 query on 512 keys 19 -> 11 us, on 4,096 126 -> 19; 128 queries on
  // 2,048 48 -> 16, 512 on 4,096 93 -> 29)
  const int64_t want = (p.few ? 8 : 2) * kCus;
  if (groups < want && steps >= 8)
    x.splits = (int)std::min<int64_t>(std::min<int64_t>((want + groups - 1) / std::max<int64_t>(groups, 1), steps / 4),
                                      kMaxSplits);
  x.splits = std::max(x.splits, 1);
  if (x.splits > 1) p.work = up(4LL * x.splits * a.nq * a.heads * a.dim) + up(8LL * x.splits * a.nq * a.heads);
  return p;
}

// Waves that share 32 keys in the dK, dV kernel. Two, for more blocks, where
// one workgroup's sums take a CU (over 64 columns of 16 bits: 8 sequences of
// 2,048, 16/4 heads of 128, documents, forward and backward 1,015 -> 817 us; 8
// heads, 64 sequences of 512, 652 -> 690; float32 to 64 columns: 24 sequences
// of 33-300, 6 heads, 185 -> 172, 8 of 2,048, 8 heads, 2,950 -> 3,070).
// float32 past 64 columns has no LDS for it. 16 bits to 64 columns leave two
// workgroups a CU: two waves share where there are no more than that, or,
// with a key head a query head and so shorter blocks, half as many (bf16,
// heads of 64: 8 of 2,048, 8/2 heads, 597 -> 469; 64 of 512, 8/2, 311 -> 290,
// 64 of 2,048 3,390 -> 3,545; 2 of 2,048, 8/8, 220 -> 192, 4 of 1,024, 12/12,
// 132 -> 135).
int share_of(const ixh_attend_args &a) {
  if (type_size(a.type) == 4) return a.dim > 64 ? 1 : 2;
  if (a.dim > 64) return 2;
  return (int64_t)a.nk * a.kv_heads <= 128LL * kCus * (a.heads > a.kv_heads ? 2 : 1) ? 2 : 1;
}

// The backward's parts for `groups` workgroups of `steps` steps, each `heads`
// heads long: of at least four steps in float32 and eight in 16 bits until
// there are `want` workgroups a CU, and of at least 16 until there are twice
// as many; not where they save a workgroup less than 3 (12) steps, as the
// parts' sums go through memory and a launch of their own. Forward and
// backward, heads of 64: 1 sequence of 2,048, 2 heads, float32, 460 -> 135
// us; 1 of 2,048, 4 heads, bf16, 130 -> 86; 1 of 8,192, 2 heads, float16, 455 ->
// 246; 2 of 4,096, 12 heads, float16, 448 -> 462; 8 of 512, 6 heads, bf16, in
// parts of eight steps 67, without 63.
int splits_of(const ixh_attend_args &a, int64_t groups, int64_t steps, int heads, int64_t want) {
  const bool wide = type_size(a.type) == 4;
  auto parts = [&](int64_t workgroups, int least) -> int64_t {
    if (groups >= workgroups) return 1;
    least = std::max(least / heads, 2);
    const int64_t n = std::min<int64_t>({(workgroups + groups - 1) / std::max<int64_t>(groups, 1), steps / least, kMaxSplits});
    return n > 1 && steps * heads * (n - 1) >= n * (wide ? 3 : 12) ? n : 1;
  };
  return (int)std::max(parts(want * kCus, wide ? 4 : 8), parts(2 * want * kCus, 16));
}

// The backward's launches: x the dQ kernel's, y the dK, dV kernel's. Returns
// the bytes of workspace, the pointers into it set from x.a.workspace.
int64_t plan_backward(AttendArgs &x, AttendArgs &y) {
  const ixh_attend_args &a = x.a;
  const int64_t B = std::max(a.B, 1);
  x.group = a.heads / a.kv_heads;
  x.pack = pack_of(a);
  x.share = share_of(a);
  x.slots = attend_slots(a.nq, a.B, 128, x.pack);
  x.dist_parts = 0;
  y = x;
  y.slots = attend_slots(a.nk, a.B, 128 / x.share, 1);
  x.splits = splits_of(a, x.slots * (x.pack > 1 ? a.kv_heads : a.heads), a.nk / B / 32, 1, type_size(a.type) == 4 ? 1 : 2);
  y.splits = splits_of(a, y.slots * a.kv_heads, a.nq / B / (32 * x.share), x.group, 1);

  char *const w = (char *)a.workspace;
  int64_t bytes = 0;
  auto take = [&](int64_t n) {
    const int64_t at = bytes;
    bytes += up(4 * n);
    return w ? (float *)(w + at) : nullptr;
  };
  x.delta = y.delta = take((int64_t)a.heads * a.nq);
  if (a.table) {
    const int64_t span = 2LL * a.reach + 1;
    y.dist_parts = kMaxDistParts;
    y.dist = take(y.slots * y.splits * a.heads * span);
    y.dist_sum = take(y.dist_parts * a.heads * span);
    if (y.slots * y.splits <= kMaxDistParts) {  // few enough for the last kernel alone
      y.dist_sum = y.dist;
      y.dist_parts = (int)(y.slots * y.splits);
    }
  }
  if (x.splits > 1) x.part_delta = take((int64_t)x.splits * a.heads * a.nq);
  // dQ's parts are added up before dK's and dV's come into the same place
  const int64_t of_q = x.splits > 1 ? (int64_t)x.splits * a.nq * a.heads * a.dim : 0;
  const int64_t of_k = y.splits > 1 ? 2LL * y.splits * a.nk * a.kv_heads * a.dim : 0;
  x.part_o = y.part_o = take(std::max(of_q, of_k));
  return bytes;
}

int check_workspace(const char *op, const void *p, int64_t have, int64_t need) {
  if (need > 0 && (!p || have < need || !aligned(p)))
    return fail(IXH_EINVAL, "linalg: %s: needs %lld bytes of workspace, 16-byte aligned (%lld given)", op,
                (long long)need, (long long)have);
  return IXH_OK;
}

void fill_in(ixh_attend_args &a) {
  if (!a.k_offs) a.k_offs = a.q_offs;
  if (a.q_docs && !a.k_docs) a.k_docs = a.q_docs;
  if (!a.table) a.reach = a.n_buckets = 0;
}

}  // namespace

extern "C" {

int ixh_attend_workspace(const ixh_attend_args *a, int backward, int64_t *bytes) {
  if (int rc = check_sizes(a)) return rc;
  if (!bytes) return fail(IXH_EINVAL, "linalg: Attend: bad arguments");
  AttendArgs x{};
  x.a = *a;
  fill_in(x.a);
  AttendArgs y;
  *bytes = backward ? plan_backward(x, y) : plan_forward(x).work;
  return IXH_OK;
}

int ixh_attend(int device, const ixh_attend_args *a, void *stream) {
  if (int rc = check_attend(a)) return rc;
  if (a->B == 0 || a->nq == 0) return IXH_OK;
  AttendArgs x{};
  x.a = *a;
  fill_in(x.a);
  const Plan p = plan_forward(x);
  if (x.slots * a->heads > kMaxGrid) return fail(IXH_EINVAL, "linalg: Attend: too many rows and heads for one launch");
  if (int rc = check_workspace("Attend", a->workspace, a->workspace_bytes, p.work)) return rc;
  x.part_o = (float *)a->workspace;
  x.part_ml = (float *)((char *)a->workspace + up(4LL * x.splits * a->nq * a->heads * a->dim));
  OnDevice on(device);
  if (on.err != hipSuccess) return hip_fail(on.err, "hipSetDevice");
  hipStream_t const st = (hipStream_t)stream;
  if (!launch_attend_fwd(x, p.few, st)) return fail(IXH_EHIP, "linalg: hip: Attend: LDS refused");
  if (int rc = launched("attend_fwd")) return rc;
  if (x.splits > 1) {
    launch_attend_join(x, st);
    return launched("attend_join");
  }
  return IXH_OK;
}

int ixh_attend_backward(int device, const ixh_attend_args *a, const ixh_attend_grads *g, void *stream) {
  if (int rc = check_attend(a)) return rc;
  if (!g) return fail(IXH_EINVAL, "linalg: AttendBackward: no gradients");
  if (g->dtable && !a->table) return fail(IXH_EINVAL, "linalg: AttendBackward: dtable without a table");
  AttendArgs x{};
  x.a = *a;
  x.g = *g;
  fill_in(x.a);
  int rc;
  if (a->B > 0 && a->nq > 0) {
    if (!a->lse) return fail(IXH_EINVAL, "linalg: AttendBackward: lse is missing");
    if ((rc = check_heads("AttendBackward", "d_out", g->d_out, a->type)) ||
        (rc = check_heads("AttendBackward", "dq", g->dq, a->type)))
      return rc;
  }
  if (a->B > 0 && a->nk > 0) {
    if ((rc = check_heads("AttendBackward", "dk", g->dk, a->type)) ||
        (rc = check_heads("AttendBackward", "dv", g->dv, a->type)))
      return rc;
  }
  AttendArgs y;
  const int64_t need = plan_backward(x, y);
  if (x.slots * a->heads > kMaxGrid || y.slots * a->kv_heads > kMaxGrid)
    return fail(IXH_EINVAL, "linalg: AttendBackward: too many rows and heads for one launch");
  if ((rc = check_workspace("AttendBackward", a->workspace, a->workspace_bytes, need))) return rc;
  OnDevice on(device);
  if (on.err != hipSuccess) return hip_fail(on.err, "hipSetDevice");
  hipStream_t const st = (hipStream_t)stream;
  if (!g->dtable) y.dist = nullptr;
  if (a->B > 0) {
    if (!launch_attend_dq(x, st)) return fail(IXH_EHIP, "linalg: hip: AttendBackward: LDS refused");
    if ((rc = launched("attend_dq"))) return rc;
    if (x.splits > 1) {
      launch_attend_sum(x, false, st);
      if ((rc = launched("attend_sum"))) return rc;
    }
    if (!launch_attend_dkv(y, st)) return fail(IXH_EHIP, "linalg: hip: AttendBackward: LDS refused");
    if ((rc = launched("attend_dkv"))) return rc;
    if (y.splits > 1) {
      launch_attend_sum(y, true, st);
      if ((rc = launched("attend_sum"))) return rc;
    }
  } else {
    y.slots = y.dist_parts = 0;
  }
  y.slots *= y.splits;
  if (g->dtable) {
    launch_attend_dtable(y, st);
    return launched("attend_dtable");
  }
  return IXH_OK;
}

int ixh_rel_buckets(int buckets, int max_distance, int bidirectional, int32_t *map) {
  const int half = bidirectional ? buckets / 2 : buckets, near = half / 2, steps = half - near;
  if (!map || buckets < (bidirectional ? 4 : 2) || buckets > 1024 || (bidirectional && buckets % 2) ||
      max_distance <= near || max_distance > kMaxReach)
    return fail(IXH_EINVAL, "linalg: RelBuckets: %d buckets up to distance %d", buckets, max_distance);
  try {
    // Bucket near + t starts at the least whole a with
    // a / near >= (max_distance / near)^(t / steps), that is
    // a^steps >= near^(steps - t) * max_distance^t, in whole numbers of any
    // length (32-bit digits, the lowest first).
    typedef std::vector<uint32_t> Big;
    auto times = [](Big &x, uint32_t f) {
      uint64_t carry = 0;
      for (uint32_t &d : x) {
        carry += (uint64_t)d * f;
        d = (uint32_t)carry;
        carry >>= 32;
      }
      if (carry) x.push_back((uint32_t)carry);
    };
    auto power = [&](int base, int e) {
      Big x{1};
      for (int i = 0; i < e; i++) times(x, (uint32_t)base);
      return x;
    };
    auto at_least = [](const Big &x, const Big &y) {
      if (x.size() != y.size()) return x.size() > y.size();
      for (size_t i = x.size(); i-- > 0;)
        if (x[i] != y[i]) return x[i] > y[i];
      return true;
    };
    std::vector<int> starts;  // of buckets near + 1 .. half - 1
    for (int t = 1, a = near; t < steps; t++) {
      Big border = power(near, steps - t);
      for (int i = 0; i < t; i++) times(border, (uint32_t)max_distance);
      while (!at_least(power(a, steps), border)) a++;
      starts.push_back(a);
    }
    for (int d = -max_distance; d <= max_distance; d++) {
      const int a = bidirectional ? std::abs(d) : std::max(-d, 0);
      const int b = a < near ? a : near + (int)(std::upper_bound(starts.begin(), starts.end(), a) - starts.begin());
      map[d + max_distance] = b + (bidirectional && d > 0 ? half : 0);
    }
  } catch (const std::exception &e) {
    return fail(IXH_ENOMEM, "linalg: RelBuckets: %s", e.what());
  }
  return IXH_OK;
}

}  // extern "C"

// ---- norms and rotation -----------------------------------------------------

namespace {

// Lanes of a row of this dimension.
int row_lanes(int dim) { return dim <= 32 ? 4 : dim <= 64 ? 8 : dim <= 128 ? 16 : 32; }

int check_norm_rope(const ixh_norm_rope_args *a) {
  if (!a) return fail(IXH_EINVAL, "linalg: QKNormRope: no arguments");
  if (!type_ok(a->type)) return fail(IXH_EINVAL, "linalg: QKNormRope: type %d", a->type);
  if (a->n < 0 || a->n > kMaxRows || a->q_heads < 0 || a->k_heads < 0 || a->q_heads > 32767 || a->k_heads > 32767)
    return fail(IXH_EINVAL, "linalg: QKNormRope: %d rows of %d and %d heads", a->n, a->q_heads, a->k_heads);
  if (a->dim < 8 || a->dim > 256 || a->dim % 8)
    return fail(IXH_EINVAL, "linalg: QKNormRope: head dimension %d not supported (a multiple of 8 up to 256)", a->dim);
  if (a->norm != IXH_HEAD_NORM_NONE && a->norm != IXH_HEAD_NORM_RMS && a->norm != IXH_HEAD_NORM_LAYER)
    return fail(IXH_EINVAL, "linalg: QKNormRope: norm %d", a->norm);
  if (!(a->eps >= 0) || !std::isfinite(a->eps)) return fail(IXH_EINVAL, "linalg: QKNormRope: eps %g", a->eps);
  if (a->gamma_type != IXH_TYPE_F32 && a->gamma_type != a->type)
    return fail(IXH_EINVAL, "linalg: QKNormRope: gammas of type %d with rows of type %d (the rows' or float32)",
                a->gamma_type, a->type);
  if (!aligned(a->q_gamma) || !aligned(a->k_gamma))
    return fail(IXH_EINVAL, "linalg: QKNormRope: gammas need a pointer that is a multiple of 16 bytes");
  const bool halves = a->pairs == IXH_PAIRS_HALVES;
  if (!halves && a->pairs != IXH_PAIRS_NEIGHBOURS) return fail(IXH_EINVAL, "linalg: QKNormRope: pairs %d", a->pairs);
  if (a->rot < 0 || a->rot > a->dim || a->rot % (halves ? 16 : 2))
    return fail(IXH_EINVAL, "linalg: QKNormRope: %d rotated columns of %d (a multiple of %d)", a->rot, a->dim,
                halves ? 16 : 2);
  if (a->rot > 0 && a->n > 0 && (!a->cos || !a->sin || a->rows < 1))
    return fail(IXH_EINVAL, "linalg: QKNormRope: a rotation needs cos and sin");
  if (a->n == 0) return IXH_OK;
  if (a->n / (256 / row_lanes(a->dim)) >= kMaxGrid)
    return fail(IXH_EINVAL, "linalg: QKNormRope: too many rows for one launch (%d of %d columns)", a->n, a->dim);
  int rc;
  if (a->q_heads > 0 && (rc = check_heads("QKNormRope", "q", a->q, a->type))) return rc;
  if (a->k_heads > 0 && (rc = check_heads("QKNormRope", "k", a->k, a->type))) return rc;
  return IXH_OK;
}

// Every row's heads to one group of lanes where there are rows enough to
// give a CU two workgroups (it keeps its angles and gammas), else fewer heads
// each (16,384 rows of 16+4 heads of 128, float16, forward and gradients: one
// workgroup a CU 101 us, two 101, eight 104, sixteen 113; 13,900 rows of 12+12
// heads of 64, bf16, with the attention: 317, 317, 326, 340).
void plan_norm_rope(NormRopeArgs &x, bool backward) {
  const int heads = std::max(x.a.q_heads + x.a.k_heads, 1);
  const int64_t groups = 256 / row_lanes(x.a.dim);
  const int64_t blocks = std::max<int64_t>((x.a.n + groups - 1) / groups, 1);
  const int64_t want = 4 * kCus;  // workgroups
  x.heads_step = (int)std::min<int64_t>(heads, std::max<int64_t>(1, blocks * heads / want));
  x.blocks = (int)(backward ? std::min<int64_t>(blocks, kNormRopeBlocks) : blocks);
}
int64_t norm_rope_parts(const NormRopeArgs &x) {
  const int heads = std::max(x.a.q_heads + x.a.k_heads, 1);
  return (int64_t)x.blocks * ((heads + x.heads_step - 1) / x.heads_step);
}

}  // namespace

extern "C" {

int ixh_qk_norm_rope(int device, const ixh_norm_rope_args *a, void *stream) {
  if (int rc = check_norm_rope(a)) return rc;
  if (a->n == 0 || a->q_heads + a->k_heads == 0) return IXH_OK;
  int rc;
  if (a->q_heads > 0 && (rc = check_heads("QKNormRope", "q_out", a->q_out, a->type))) return rc;
  if (a->k_heads > 0 && (rc = check_heads("QKNormRope", "k_out", a->k_out, a->type))) return rc;
  OnDevice on(device);
  if (on.err != hipSuccess) return hip_fail(on.err, "hipSetDevice");
  NormRopeArgs x{};
  x.a = *a;
  plan_norm_rope(x, false);
  launch_norm_rope(x, (hipStream_t)stream);
  return launched("norm_rope");
}

int ixh_qk_norm_rope_workspace(const ixh_norm_rope_args *a, int64_t *bytes) {
  if (!a || !bytes || a->dim < 8 || a->dim > 256 || a->n < 0 || a->q_heads < 0 || a->k_heads < 0)
    return fail(IXH_EINVAL, "linalg: QKNormRope: bad arguments");
  NormRopeArgs x{};
  x.a = *a;
  plan_norm_rope(x, true);
  *bytes = up(norm_rope_parts(x) * 2 * a->dim * 4);
  return IXH_OK;
}

int ixh_qk_norm_rope_backward(int device, const ixh_norm_rope_args *a, const ixh_norm_rope_grads *g, void *stream) {
  if (int rc = check_norm_rope(a)) return rc;
  if (!g) return fail(IXH_EINVAL, "linalg: QKNormRopeBackward: no gradients");
  int rc;
  NormRopeArgs x{};
  x.a = *a;
  x.g = *g;
  const bool want = g->dq_gamma || g->dk_gamma;
  if (a->n > 0) {
    if (a->q_heads > 0 && ((rc = check_heads("QKNormRopeBackward", "dq_out", g->dq_out, a->type)) ||
                           (rc = check_heads("QKNormRopeBackward", "dq", g->dq, a->type))))
      return rc;
    if (a->k_heads > 0 && ((rc = check_heads("QKNormRopeBackward", "dk_out", g->dk_out, a->type)) ||
                           (rc = check_heads("QKNormRopeBackward", "dk", g->dk, a->type))))
      return rc;
  }
  plan_norm_rope(x, true);
  if (want) {
    if ((rc = check_workspace("QKNormRopeBackward", a->workspace, a->workspace_bytes,
                              up(norm_rope_parts(x) * 2 * a->dim * 4))))
      return rc;
    x.part = (float *)a->workspace;
  }
  if ((a->n == 0 || a->q_heads + a->k_heads == 0) && !want) return IXH_OK;
  OnDevice on(device);
  if (on.err != hipSuccess) return hip_fail(on.err, "hipSetDevice");
  launch_norm_rope_backward(x, (hipStream_t)stream);
  return launched("norm_rope_backward");
}

}  // extern "C"
