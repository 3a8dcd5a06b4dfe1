// The work of the tensor-core attention forwards: items (a block of packed rows against the keys of one batch
// entry and key head), how they are cut into equal runs of key tiles over the CTAs, and where the pieces of an item
// that several CTAs share are kept until they are joined.
#pragma once

#include "xattn_tc.cuh"

namespace tsb {

// A run of key tiles of one item; side < 0 ends the list. Made by one warp, read by all roles from a ring in
// shared memory: the walk's state and divisions stay out of the other warps' registers.
struct FwSeg {
  int side, item, bi, h, rt, k0, k1, n, len;
};
constexpr int kFwSegs = 4;

// Division by a run-time constant: n / d for 0 <= n < 2^31 is the high word of n * mul, shifted by s, with
// 2^s < d <= 2^(s + 1) and mul = 2^(32 + s) / d rounded up (below 2^32): the rounding adds less than d n to n 2^(32 +
// s), so less than one part in n to the quotient.
struct FastDiv {
  uint32_t d, mul, shift;
};
inline FastDiv fast_div(int d) {
  FastDiv f = {static_cast<uint32_t>(d), 0u, 0u};
  while ((2u << f.shift) < static_cast<uint32_t>(d)) ++f.shift;
  if (d > 1) f.mul = static_cast<uint32_t>(((1ull << (32 + f.shift)) + d - 1) / d);
  return f;
}
__device__ __forceinline__ int fdiv(const FastDiv& f, int n) {
  return f.d == 1 ? n : static_cast<int>(__umulhi(static_cast<uint32_t>(n), f.mul) >> f.shift);
}

struct FwSide {
  XSide s;
  int row_tiles, items, tile_rows, key_shift;  // rows of an item, log2 of a key tile
  FastDiv by_T, by_G;
  int mul_kh, mul_kb, mul_vh, mul_vb;
  // Slots of (O / l, log-sum-exp) as [D / 4][rows][4], so that a warp's rows write whole lines: two per CTA of the
  // launch and, where a call has two sides, one per item that a single CTA finished.
  float *slots, *slot_lse, *item_slots, *item_lse;
  int slot_rows, item_rows;
  int2* pieces;  // first and last CTA of the side's items from `first` on
  int first;     // items before it were taken whole
};

struct FwArgs {
  FwSide side[2];
  int sides, D, whole;  // whole: items per CTA taken whole (one side only)
  int item_cost;        // see fw_cost
  int keep;             // the call has two sides: finished items go to their slots
  uint64_t seg_ns;      // limit of the waits that last as long as a segment of another role
  float* flush;         // per CTA of the 256-row form, [HD / 4][256][4]: see kFwFlushTiles
  __nv_bfloat16* out;
  float* lse;
  float scale_log2;  // |scale| log2(e)
  uint32_t q_flip;   // sign bits of a negative scale, applied to Q
};

namespace {

__device__ __forceinline__ int fw_tiles_of(const FwSide& sd, int len) {
  return (len + (1 << sd.key_shift) - 1) >> sd.key_shift;
}
__device__ __forceinline__ int fw_tiles(const FwSide& sd, int bi) { return fw_tiles_of(sd, side_len(sd.s, bi)); }
// Cost of an item in key tiles: its tiles and, unless it has none, item_cost for its Q, drain and output.
__device__ __forceinline__ int fw_cost(const FwArgs& A, int tiles) { return tiles > 0 ? tiles + A.item_cost : 0; }

__device__ __forceinline__ XRow fw_row(const FwSide& sd, int64_t r) {
  const int n = static_cast<int>(r), u = fdiv(sd.by_T, n), b2 = fdiv(sd.by_G, u);
  XRow x;
  x.t = n - u * sd.s.T;
  x.g = u - b2 * sd.s.G;
  x.b2 = b2;
  return x;
}

// Walks a CTA's items: whole ones first (also those without keys), then its run [begin, begin + left) of the
// split part's cost.
struct FwCursor {
  const FwArgs& A;
  long long begin, left;
  long long at;  // where the last item begins
  int w, side, item, k;
  __device__ void decode(FwSeg& g) const {
    const FwSide& sd = A.side[g.side];
    const int per = sd.s.hkv * sd.row_tiles;
    g.bi = g.item / per;
    const int r = g.item - g.bi * per;
    g.h = r / sd.row_tiles;
    g.rt = r - g.h * sd.row_tiles;
    g.len = side_len(sd.s, g.bi);
    g.n = fw_tiles_of(sd, g.len);
  }
  __device__ bool next(FwSeg& g) {
    if (w < A.whole) {
      g.side = 0;
      g.item = w * gridDim.x + blockIdx.x;
      ++w;
      decode(g);
      g.k0 = 0;
      g.k1 = g.n;
      return true;
    }
    while (left > 0) {
      if (item >= A.side[side].items) {
        ++side;
        item = 0;
      }
      g.side = side;
      g.item = item++;
      decode(g);
      const int k0 = k;
      k = 0;
      if (g.n == 0) continue;
      at = begin - k0;
      const long long take = min(static_cast<long long>(fw_cost(A, g.n) - k0), left);
      g.k0 = k0;
      g.k1 = static_cast<int>(min(static_cast<long long>(g.n), k0 + take));
      begin += take;
      left -= take;
      if (g.k0 < g.k1) return true;
    }
    return false;
  }
};

// Sums of the items' costs, and position lookups, by one warp.
// Lane l holds 8 consecutive entries of every 256.
struct FwScan {
  // Cost of the items before item `i`.
  static __device__ long long before(const FwArgs& A, const FwSide& sd, int i, int lane) {
    const int per = sd.s.hkv * sd.row_tiles, b0 = i / per;
    long long t = 0;
    if (sd.s.lengths == nullptr) {
      t = static_cast<long long>(b0) * fw_cost(A, fw_tiles(sd, 0));
    } else {
      for (int base = 0; base < b0; base += 256)
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const int b = base + lane * 8 + e;
          if (b < b0) t += fw_cost(A, fw_tiles(sd, b));
        }
#pragma unroll
      for (int o = 16; o > 0; o >>= 1) t += __shfl_xor_sync(0xffffffffu, t, o);
    }
    t *= per;
    const int r = i - b0 * per;
    return r == 0 ? t : t + static_cast<long long>(r) * fw_cost(A, fw_tiles(sd, b0));
  }
  // Item and place within it at position x of the side (x below its total).
  static __device__ void locate(const FwArgs& A, const FwSide& sd, long long x, int lane, int& item, int& k) {
    const int per = sd.s.hkv * sd.row_tiles;
    if (sd.s.lengths == nullptr) {
      const int n = fw_cost(A, fw_tiles(sd, 0));
      item = static_cast<int>(x / n);
      k = static_cast<int>(x - static_cast<long long>(item) * n);
      return;
    }
    long long done = 0;
    for (int base = 0; base < sd.s.nb; base += 256) {
      int n[8];
      long long s = 0;
#pragma unroll
      for (int e = 0; e < 8; ++e) {
        const int b = base + lane * 8 + e;
        n[e] = b < sd.s.nb ? fw_cost(A, fw_tiles(sd, b)) : 0;
        s += n[e];
      }
      long long inc = s;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const long long v = __shfl_up_sync(0xffffffffu, inc, o);
        if (lane >= o) inc += v;
      }
      const long long all = __shfl_sync(0xffffffffu, inc, 31);
      if ((done + all) * per > x) {
        const unsigned hit = __ballot_sync(0xffffffffu, (done + inc) * per > x);
        const int src = __ffs(hit) - 1;
        long long at = done + inc - s;
        int fi = 0, fk = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) {
          const long long end = at + n[e];
          if (at * per <= x && x < end * per) {
            const long long rel = x - at * per;
            fi = (base + lane * 8 + e) * per + static_cast<int>(rel / n[e]);
            fk = static_cast<int>(rel % n[e]);
          }
          at = end;
        }
        item = __shfl_sync(0xffffffffu, fi, src);
        k = __shfl_sync(0xffffffffu, fk, src);
        return;
      }
      done += all;
    }
    item = sd.items;  // past the end: never reached for x below the total
    k = 0;
  }
};

// This CTA's run, by one warp: [W c / G, W (c + 1) / G) of the cost W behind the whole items, G the CTAs that get any
// (a piece list has no gaps).
struct FwRun {
  long long W, G;
};
__device__ __forceinline__ FwRun fw_start(const FwArgs& A, FwCursor& cur, int lane) {
  const int first = A.whole * static_cast<int>(gridDim.x);
  const long long t0 = FwScan::before(A, A.side[0], A.side[0].items, lane);
  const long long t1 = A.sides > 1 ? FwScan::before(A, A.side[1], A.side[1].items, lane) : 0;
  const long long s0 = first ? FwScan::before(A, A.side[0], first, lane) : 0;
  const long long W = t0 + t1 - s0;
  const long long G = W < gridDim.x ? W : gridDim.x, c = blockIdx.x;
  const long long lo = c < G ? W * c / G : W, hi = c < G ? W * (c + 1) / G : W;
  cur.begin = lo;
  cur.left = hi - lo;
  cur.at = 0;
  cur.w = cur.side = cur.item = cur.k = 0;
  if (hi > lo) {
    long long x = s0 + lo;
    if (x >= t0) {
      cur.side = 1;
      x -= t0;
    }
    FwScan::locate(A, A.side[cur.side], x, lane, cur.item, cur.k);
  }
  return FwRun{W, G};
}
// Notes which CTAs hold the pieces of the item `g` that begins in this run.
__device__ __forceinline__ void fw_note_pieces(const FwArgs& A, const FwCursor& cur, const FwRun& run, const FwSeg& g) {
  const FwSide& sd = A.side[g.side];
  sd.pieces[g.item - sd.first] = make_int2(blockIdx.x, static_cast<int>(((cur.at + g.n) * run.G - 1) / run.W));
}

}  // namespace

// The few-rows form (cross_attention_rows.cu): all sides of `A` have items of at most kFewRows rows. `behind`: it
// may run beside the launch before it in the stream, whose results it does not need, and ends after it.
constexpr int kFewRows = 16;
constexpr int kFewKeyShift = 6;
int few_rows_grid();
int few_rows_launch(const FwArgs& A, int grid, bool behind, cudaStream_t st);

}  // namespace tsb
