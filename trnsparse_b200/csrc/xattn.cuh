// What the dense attention kernels (cross attention, shared-prefix attention)
// share: how rows and keys are addressed, which keys a row may see, and the
// host-side view of the C-ABI arguments.
//
// A "side" is one set of keys with the query rows that read it. The rows of
// one item (bi, kv head h) are packed: all G query heads of the kv head, all T
// tokens and, where the keys are shared by the batch, all n2 sequences, so a
// K / V tile is read once for every row that needs it:
//   r -> token r % T, group head (r / T) % G, sequence r / (T G).
#pragma once

#include <cuda_bf16.h>
#include <stdint.h>

#include "common.cuh"

namespace tsb {

struct XSide {
  const void *q, *k, *v;
  int64_t q_bi, q_b2, q_h, q_t;  // element strides; q_h: per query head
  int64_t o_bi, o_b2, o_h, o_t;
  int64_t k_b, k_h, k_t, v_b, v_h, v_t;
  const int* lengths;   // kept keys of item bi (nullable: klen)
  const uint8_t* mask;  // byte per key, 0 = hidden (nullable)
  int64_t mask_stride;
  int nb, hkv, G, T, n2, klen;
  int causal;  // row's token t sees keys < length - T + 1 + t
};

__host__ __device__ inline int64_t side_rows(const XSide& s) { return static_cast<int64_t>(s.n2) * s.G * s.T; }

__device__ __forceinline__ int side_len(const XSide& s, int bi) {
  if (s.lengths == nullptr) return s.klen;
  return max(0, min(s.lengths[bi], s.klen));
}

struct XRow {
  int t, g, b2;
};
__device__ __forceinline__ XRow side_row(const XSide& s, int64_t r) {
  XRow x;
  // packed rows stay below 2^31 (checked by the entry points)
  const unsigned rr = static_cast<unsigned>(r), T = s.T, G = s.G;
  x.t = static_cast<int>(rr % T);
  const unsigned u = rr / T;
  x.g = static_cast<int>(u % G);
  x.b2 = static_cast<int>(u / G);
  return x;
}
// One past the last key row x may see.
__device__ __forceinline__ int row_limit(const XSide& s, const XRow& x, int len) {
  return s.causal ? max(0, min(len, len - s.T + 1 + x.t)) : len;
}
__device__ __forceinline__ int64_t q_offset(const XSide& s, int bi, int h, const XRow& x) {
  return bi * s.q_bi + x.b2 * s.q_b2 + (static_cast<int64_t>(h) * s.G + x.g) * s.q_h + x.t * s.q_t;
}
__device__ __forceinline__ int64_t o_offset(const XSide& s, int bi, int h, const XRow& x) {
  return bi * s.o_bi + x.b2 * s.o_b2 + (static_cast<int64_t>(h) * s.G + x.g) * s.o_h + x.t * s.o_t;
}
// Row of the (batch, query head, token) order that statistics and partial results use.
__device__ __forceinline__ int64_t flat_row(const XSide& s, int bi, int h, const XRow& x) {
  return ((static_cast<int64_t>(bi + x.b2) * s.hkv + h) * s.G + x.g) * s.T + x.t;
}

// Sides of a call: cross attention has one; shared-prefix attention has the prefix (n2 = batch) and the
// sequences' own keys. Either may have no keys.
int make_sides(const trnsparse_attention_args* a, bool prefix, XSide (&s)[2], int* n);
int check_attention(const trnsparse_attention_args* a, const char* what);

// Joins `pieces` partial results per row: O = sum 2^(lse_i - max) O_i / sum 2^(lse_i - max), a row of which
// every piece is empty (-inf) is zero. part_o [pieces][rows][D], part_lse [pieces][rows] (base 2).
int combine_pieces(const float* part_o, const float* part_lse, int pieces, const trnsparse_attention_args* a,
                   cudaStream_t st);

// Steps of a walk that one of `ctas` CTAs takes when the walks are cut into at most `most` parts to fill `sms` SMs,
// `resident` CTAs each. The time is counted in steps of a CTA that has an SM for itself: a step beside r - 1 others
// takes (1 + r) / 2, a CTA starts and ends in two, the join takes two, and each part `part_cost` and the traffic of its
// CTAs' 128 rows.
inline int64_t walk_steps(int64_t ctas, int64_t steps, int64_t sms, int resident, int64_t most,
                          double part_cost) {
  const int64_t slots = sms * resident;
  int64_t best = steps > 0 ? steps : 1;
  double least = 1e300;
  for (int64_t n = 1; n <= most && n <= steps; ++n) {
    const int64_t per = (steps + n - 1) / n, parts = (steps + per - 1) / per, all = ctas * parts;
    const int64_t waves = all / slots, rest = (all - waves * slots + sms - 1) / sms;
    const double time = 0.5 * static_cast<double>(waves * (1 + resident) + (rest ? 1 + rest : 0));
    const double join = 2.0 + static_cast<double>(parts) * (part_cost + static_cast<double>(ctas) / 128.0);
    const double cost = time * static_cast<double>(per + 2) + (parts > 1 ? join : 0.0);
    if (cost < least) {
      least = cost;
      best = per;
    }
  }
  return best;
}

// Tensor-core forms (bf16, head_dim a multiple of 8 up to 128, 16-byte rows).
bool xattn_tc_ok(const trnsparse_attention_args* a, bool prefix);
size_t xattn_tc_workspace(const trnsparse_attention_args* a, bool prefix);
int xattn_tc_forward(const trnsparse_attention_args* a, bool prefix, void* ws, cudaStream_t st);
bool xattn_bwd_tc_ok(const trnsparse_attention_args* a);
size_t xattn_bwd_tc_workspace(const trnsparse_attention_args* a);
int xattn_bwd_tc(const trnsparse_attention_args* a, void* ws, cudaStream_t st);

}  // namespace tsb
