// attend.h — arguments and launchers of the float attention operators
// (attend_fwd.hip, attend_bwd.hip, qk_norm_rope.hip), checked and filled in
// by attend_api.cpp.
#pragma once
#include <hip/hip_runtime.h>
#include <stdint.h>

#include "../../include/indecis_hip.h"

namespace ixh {

// One (sequence, block of rows) each: sequence b's blocks of `rows` rows
// (times `pack` heads a row) have the slots from offs[b] * pack / rows + b
// on, so that a workgroup finds its block from offs alone. Some slots stay
// empty.
constexpr int64_t attend_slots(int64_t n, int64_t B, int64_t rows, int64_t pack) { return n * pack / rows + B; }

struct AttendArgs {
  ixh_attend_args a;   // as the caller gave them, k_offs and k_docs filled in
  ixh_attend_grads g;  // backward only
  int group;           // heads / kv_heads
  int share;           // waves that have the same 32 keys in the dK, dV kernel: 1 or 2
  int pack;            // heads of a token that are rows of a block (forward, dQ): 1 or group
  int64_t slots;       // of the launch's row blocks
  int splits;          // parts of the keys (forward, dQ), of the queries (dK, dV)
  float *part_o;       // [splits][nq][heads][dim], unnormalised; the backward's
                       // too, and [splits][2][nk][kv_heads][dim] for dK and dV
  float *part_ml;      // [splits][nq][heads][2]: maximum (base 2) and sum
  float *delta;        // [heads][nq]: sum of dO * o (backward)
  float *part_delta;   // [splits][heads][nq]
  float *dist;         // [slots * splits][heads][2 reach + 1]: sums of dZ by distance (backward)
  float *dist_sum;     // [parts][heads][2 reach + 1]
  int dist_parts;
};

// Forward kernels' rows a workgroup.
constexpr int kAttendRowsFew = 32, kAttendRowsMany = 128;
// Keys a step of the forward and dQ kernels, by type size and variant.
constexpr int attend_keys(int size, bool few) { return size == 4 || few ? 32 : 64; }
// Distances past the bias' reach that a step's scores can touch, so that a
// row of the table's copy in LDS needs no clamped index.
constexpr int kBiasPad = 96;
constexpr int attend_bias_len(int reach) { return 2 * (reach + kBiasPad) + 1; }

bool launch_attend_fwd(const AttendArgs &x, bool few, hipStream_t s);
void launch_attend_join(const AttendArgs &x, hipStream_t s);
bool launch_attend_dq(const AttendArgs &x, hipStream_t s);
bool launch_attend_dkv(const AttendArgs &x, hipStream_t s);
// The parts of dQ and delta, or of dK and dV, added up.
void launch_attend_sum(const AttendArgs &x, bool keys, hipStream_t s);
void launch_attend_dtable(const AttendArgs &x, hipStream_t s);

struct NormRopeArgs {
  ixh_norm_rope_args a;
  ixh_norm_rope_grads g;
  int heads_step;   // heads a workgroup takes of each of its rows
  int blocks;       // workgroups over the rows
  float *part;      // [blocks * head steps][2][dim] (backward)
};
constexpr int kNormRopeBlocks = 1024;
void launch_norm_rope(const NormRopeArgs &x, hipStream_t s);
void launch_norm_rope_backward(const NormRopeArgs &x, hipStream_t s);

}  // namespace ixh
