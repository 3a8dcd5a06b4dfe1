// Dense attention forward on the tensor cores (bf16 in and out, fp32 softmax
// and sums; head_dim a multiple of 8 up to 128): cross attention and
// shared-prefix attention, from one token per sequence to long prompts.
//
//   O = sum_j 2^(s_j - m) v_j / sum_j 2^(s_j - m),  s = scale log2(e) q.k
// in one pass over the key tiles with the running maximum m and sum l of every
// row. P = 2^(s - m) is rounded to bf16 for its product with V (half a step, at
// most 2^-8 relative, of the same size as the result's own rounding: the result's
// error grows from 1.7e-3 to 2.3e-3 of its size; unrounded P would take a second
// product for its low part); l sums the unrounded values in fp32. m moves only when
// a tile's maximum passes it by more than 2^8, so the accumulator in TMEM is rarely
// rescaled and P <= 2^8.
//
// An item is 256 packed rows (see xattn.cuh: query heads of one key head,
// tokens, and for a shared prefix all sequences) against the keys of one (batch
// entry, key head). One CTA per SM, 11 warps:
//   warps 0-3 / 4-7  softmax of rows 0-127 / 128-255, a thread per row: reads
//                    its 128 scores from TMEM, writes P over them as packed
//                    bf16 (the A operand of the second product), keeps m and l;
//                    loads the Q tile (any strides) and writes O.
//   warp 8           TMA producer: K0, V0, K1, V1, ... through one ring of
//                    tiles; a tile is read by both halves' products, so 64 KB
//                    of K / V feed 2 x 2 products of 128 x 128 x 128.
//   warp 10          the list of (item, key tiles) this CTA works through
//   warp 9           MMA issuer: for each key tile P_A V, next S_A, P_B V,
//                    next S_B; the tensor cores work on one half while the
//                    other half's exponentials run.
// The score and P columns of a half are the same TMEM columns: MMAs of a CTA
// run in issue order, so the next S follows the P V that reads them.
//
// Work split: with many items each CTA takes whole items round robin (CTAs that
// run at the same time share K / V in L2); the last one to two rounds - or all
// of it when items are few, as in decoding - are cut into equal runs of key
// tiles whatever the items' lengths, so every SM streams keys. A CTA has at
// most one item it continues and one it leaves unfinished: their (O / l,
// log-sum-exp) go to two slots of the workspace, joined by a second launch in
// tile order (no atomics, results repeat bit for bit). The split depends on the
// lengths, which stay on the device: no host synchronisation.
//
// What bounds it: long rows, the exponentials and the chain scores -> P -> product of
// a half (a quarter of them as a polynomial on the FMA pipe): 16 heads, 4096 x 4096 x
// 128 137 us, 1000 TFLOP/s; 4 x 16 heads, 2048 x 4096 x 128 with the row statistics 255
// us, 1078. Short or ragged items lose 3 to 5 us an item and CTA to its start and end
// and the join: prompts of 4 x 32/8 heads, 777 x up to 2049 keys 87 + 12 us. Few rows
// (a shared prefix, 256 rows a key head): memory and that same start and end.
//
// Hidden keys (past a length, or masked): scores become -inf by selection, and
// their V rows are zeroed in shared memory before the product, so NaN or
// infinity in padding never meets a zero P. Only tiles that hold hidden keys
// pay for it.
#include "xattn_items.cuh"

namespace tsb {
namespace {

constexpr int kFwThreads = 352;
constexpr int kFwRows = 256;  // rows of an item, two halves of 128
constexpr int kFwKeys = 128, kFwKeyShift = 7;
constexpr float kFwLazy = 8.f;
// Key tiles that an item's start and end count for: 1, 2, 4 take 109.2, 109.3, 108.8 us in ragged prompts of 777 tokens
// and 146.6, 147.3, 147.7 us in a step of 96 sequences over a shared prefix of 32768 keys.
constexpr int kFwItemCost = 2;
// Tiles after which a row's accumulator and sum are added to fp32 sums in memory and start from zero again. The tensor
// core cuts what it adds to the accumulator's last place, so sums of one sign shrink with the chain: 0.07% after 2^17
// keys, 0.25% after 2^19, 1% after 2^21 (values of mean 1), and terms below 2^-25 of the sum vanish. The row's sum is
// added to term by term, where terms below 2^-24 of it vanish.
constexpr int kFwFlushTiles = 1024;
// The list's writer, and the softmax warps of a half without rows, wait until the others are through with a segment. A
// tile takes 1 to 3 us, so an item of 50 million keys takes the second that bounds the waits for a pipeline stage: these
// two waits are bounded by 20 us a tile more.
constexpr uint64_t kFwTileNs = 20000;
// Key tiles that a CTA of the few-rows form walks at most: 2^21 keys, of which a warp's accumulators add 2^19 (0.25%
// low). It has no flushing (its registers are full); the calls beyond, milliseconds long, take the 256-row form.
constexpr int64_t kFewMostTiles = 1 << (21 - kFewKeyShift);
// Tiles of a CTA at least, see fw_plan. 4, 8, 16: 43.6, 50.2, 63.8 us for 64 sequences over a prefix of 2048 and own keys
// up to 512; 65.2, 65.7, 79.2 over 8192 and 1024; 89.4, 81.7, 92.7 for 96 sequences there; the same over 32768 and 2048.
constexpr int kFwLeast = 8;

template <int HD>
struct FwLayout {
  static constexpr int kChunks = HD / 64;
  static constexpr int kTile = 128 * HD * 2;
  static constexpr int kStages = HD == 128 ? 5 : 10;
  static constexpr int kQ = 0;
  static constexpr int kRing = 2 * kTile;
  static constexpr int kBar = kRing + kStages * kTile;
  static constexpr int kFlushed = kBar + 512;  // float [2][256]
  static constexpr int kSmem = kFlushed + 2048;
  static constexpr uint32_t kTmemO = 256;  // S / P: [0, 128) and [128, 256); O: [256, +HD) and [384, +HD)
};

struct FwBars {
  uint64_t full[10], empty[10], q_full[2], s_full[2], p_half[2], p_full[2], o_done[2];
  uint64_t seg_full[kFwSegs], seg_empty[kFwSegs];
  FwSeg seg[kFwSegs];
  uint32_t tmem_slot;
  int abort_flag;
};

static_assert(sizeof(FwBars) <= 512, "FwLayout::kFlushed");

template <int HD>
__global__ void __launch_bounds__(kFwThreads, 1)
xattn_fwd_tc_kernel(const __grid_constant__ CUtensorMap tk0, const __grid_constant__ CUtensorMap tv0,
                    const __grid_constant__ CUtensorMap tk1, const __grid_constant__ CUtensorMap tv1,
                    const __grid_constant__ FwArgs A) {
  using Lay = FwLayout<HD>;
  // No static shared memory: the dynamic window then starts 1024-byte aligned, as the swizzled tiles need.
  extern __shared__ __align__(16) uint8_t sb[];
  FwBars& B = *reinterpret_cast<FwBars*>(sb + Lay::kBar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  if (threadIdx.x == 0) {
    for (int i = 0; i < Lay::kStages; ++i) {
      mbar_init(&B.full[i], 1);
      mbar_init(&B.empty[i], 1);
    }
    for (int i = 0; i < 2; ++i) {
      mbar_init(&B.q_full[i], 128);
      mbar_init(&B.s_full[i], 1);
      mbar_init(&B.p_half[i], 128);
      mbar_init(&B.p_full[i], 128);
      mbar_init(&B.o_done[i], 1);
    }
    for (int i = 0; i < kFwSegs; ++i) {
      mbar_init(&B.seg_full[i], 1);
      mbar_init(&B.seg_empty[i], 10);  // producer, MMA issuer, eight softmax warps
    }
    B.abort_flag = (smem_u32(sb) & 1023u) ? 1 : 0;
    if (B.abort_flag) record_device_error(DEVERR_SELFCHECK_SMEM);
    fence_mbar_init();
  }
  if (warp == 9) {
    tmem_alloc(&B.tmem_slot, 512);
    tmem_relinquish();
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = B.tmem_slot;
  volatile int* abort_flag = &B.abort_flag;
  // The i-th segment of the list (false: the list was given up). One reader of each consumer then arrives on
  // seg_empty.
  auto read_seg = [&](int i, FwSeg& g) {
    if (!mbar_wait(&B.seg_full[i % kFwSegs], (i / kFwSegs) & 1, A.seg_ns)) return false;
    g = B.seg[i % kFwSegs];
    return true;
  };

  grid_dep_launch();  // the own keys' launch of a two-sided call may take SMs as they come free

  if (warp == 10) {
    // ---------------- the list of segments
    if (!*abort_flag) {
      FwCursor cur{A};
      const FwRun run = fw_start(A, cur, lane);
      if (lane == 0) {
        FwSeg g;
        for (int i = 0;; ++i) {
          const bool whole = cur.w < A.whole, more = cur.next(g);
          if (!more) g.side = -1;
          if (i >= kFwSegs && !mbar_wait(&B.seg_empty[i % kFwSegs], (i / kFwSegs - 1) & 1, A.seg_ns)) {
            atomicExch(&B.abort_flag, 1);
            break;
          }
          B.seg[i % kFwSegs] = g;
          mbar_arrive(&B.seg_full[i % kFwSegs]);
          if (!more || *abort_flag) break;
          if (!whole && g.k0 == 0) fw_note_pieces(A, cur, run, g);
        }
      }
    }
  } else if (warp == 8) {
    // ---------------- TMA producer
    if (lane == 0 && !*abort_flag) {
      FwSeg g;
      int slot = 0, use = 0;
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!read_seg(i, g)) { ok = false; break; }
        mbar_arrive(&B.seg_empty[i % kFwSegs]);
        if (g.side < 0) break;
        const FwSide& sd = A.side[g.side];
        const CUtensorMap* tk = g.side ? &tk1 : &tk0;
        const CUtensorMap* tv = g.side ? &tv1 : &tv0;
        const int kh = g.h * sd.mul_kh, kb = g.bi * sd.mul_kb, vh = g.h * sd.mul_vh, vb = g.bi * sd.mul_vb;
        for (int j = g.k0; ok && j < g.k1; ++j) {
#pragma unroll 1
          for (int kv = 0; kv < 2; ++kv) {
            if (*abort_flag || (use > 0 && !mbar_wait(&B.empty[slot], (use - 1) & 1))) {
              ok = false;
              break;
            }
            uint8_t* dst = sb + Lay::kRing + slot * Lay::kTile;
            mbar_arrive_expect_tx(&B.full[slot], Lay::kTile);
            for (int c = 0; c < Lay::kChunks; ++c)
              tma_load_4d(dst + c * 16384, kv ? tv : tk, c * 64, j * kFwKeys, kv ? vh : kh, kv ? vb : kb, &B.full[slot]);
            if (++slot == Lay::kStages) {
              slot = 0;
              ++use;
            }
          }
        }
      }
      if (!ok) {
        atomicExch(&B.abort_flag, 1);
        // copies in flight land before the CTA may end
        for (int i = 0; i < Lay::kStages; ++i) {
          const int u = use - (i < slot ? 0 : 1);
          if (u >= 0) mbar_wait(&B.full[i], u & 1);
        }
      }
    }
  } else if (warp == 9) {
    // ---------------- MMA issuer
    if (warp_all(!*abort_flag)) {
      constexpr uint32_t idesc_s = make_idesc(MmaKind::BF16, 128, 128);
      constexpr uint32_t idesc_o = make_idesc(MmaKind::BF16, 128, HD) | (1u << 16);  // V is MN-major
      const bool lead = elect_one();
      // Descriptors are formed once and moved by adding to their address field (16-byte units). The tensor
      // cores take the next MMA only a moment before they are through with the last (64 clocks each), so a
      // barrier is looked at before the last MMA of a burst is issued, and waited for only if it was not
      // complete then: a wait that is already over would cost more than an MMA each.
      const uint64_t k_desc = smem_desc_sw128(smem_u32(sb + Lay::kRing));
      const uint64_t v_desc = smem_desc_sw128_mn(smem_u32(sb + Lay::kRing), 16384);
      const uint32_t q_lo = static_cast<uint32_t>(smem_desc_sw128(smem_u32(sb + Lay::kQ)));
      constexpr uint32_t kStep = Lay::kTile >> 4;
      FwSeg g;
      int slot = 0, use = 0;
      uint32_t q_ph = 0, p_ph = 0;  // phase bit of each half (no arrays: an index would put them in local memory)
      auto advance = [&] {
        if (++slot == Lay::kStages) {
          slot = 0;
          ++use;
        }
      };
      auto ensure = [&](bool seen, uint64_t* bar, int parity) { return warp_all(seen || mbar_wait(bar, parity & 1)); };
      auto score = [&](int half, int ks, int kk) {
        const uint32_t off = ((kk >> 2) * 16384 + (kk & 3) * 32) >> 4;
        umma<MmaKind::BF16>(tmem + half * 128, desc_at(k_desc, q_lo + half * kStep + off),
                            desc_at(k_desc, static_cast<uint32_t>(k_desc) + ks * kStep + off), idesc_s, kk > 0);
      };
      bool ok = true;
      for (int i = 0; ok; ++i) {
        if (!warp_all(read_seg(i, g))) { ok = false; break; }
        if (lead) mbar_arrive(&B.seg_empty[i % kFwSegs]);
        if (g.side < 0) break;
        const int n = g.k1 - g.k0;
        if (n == 0) continue;
        const int halves = static_cast<int64_t>(g.rt) * kFwRows + 128 < side_rows(A.side[g.side].s) ? 2 : 1;
        // first scores
        if (!ensure(false, &B.full[slot], use)) { ok = false; break; }
        for (int half = 0; half < halves; ++half) {
          if (!ensure(false, &B.q_full[half], q_ph >> half)) { ok = false; break; }
          q_ph ^= 1u << half;
          tc_fence_after();
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk)
            if (lead) score(half, slot, kk);
          if (lead) umma_commit(&B.s_full[half]);
        }
        if (!ok) break;
        if (lead) umma_commit(&B.empty[slot]);
        advance();
        bool v_seen = false, p_seen = false;
        for (int j = 0; ok && j < n; ++j) {
          const int vs = slot, vu = use;
          advance();
          const bool more = j + 1 < n;
          if (!ensure(v_seen, &B.full[vs], vu)) { ok = false; break; }
          const uint32_t v_lo = static_cast<uint32_t>(v_desc) + vs * kStep;
          bool k_seen = !more;
          for (int half = 0; half < halves; ++half) {
            // P is packed at the start of its own 64 score columns; the last 64 keys come first
            auto pv = [&](int kk, bool add) {
              umma_ts_f16(tmem + Lay::kTmemO + half * 128, tmem + half * 128 + (kk >> 2) * 64 + (kk & 3) * 8,
                          desc_at(v_desc, v_lo + kk * (2048 >> 4)), idesc_o, add);
            };
            const int ph = (p_ph >> half) & 1;
            if (!ensure(p_seen, &B.p_half[half], ph)) { ok = false; break; }
            tc_fence_after();
            if (lead) {
              pv(4, j > 0);
              pv(5, true);
              pv(6, true);
            }
            bool f_seen = mbar_test_wait(&B.p_full[half], ph);
            if (!k_seen) k_seen = mbar_test_wait(&B.full[slot], use & 1);
            if (lead) pv(7, true);
            if (!ensure(f_seen, &B.p_full[half], ph)) { ok = false; break; }
            p_ph ^= 1u << half;
            tc_fence_after();
#pragma unroll
            for (int kk = 0; kk < 4; ++kk)
              if (lead) pv(kk, true);
            const int nh = half + 1 < halves ? half + 1 : 0;  // whose P comes next
            if (more) {
              if (!ensure(k_seen, &B.full[slot], use)) { ok = false; break; }
              k_seen = true;
#pragma unroll
              for (int kk = 0; kk < HD / 16 - 1; ++kk)
                if (lead) score(half, slot, kk);
              p_seen = mbar_test_wait(&B.p_half[nh], (p_ph >> nh) & 1);
              if (nh == 0) {
                const int ns = slot + 1 == Lay::kStages ? 0 : slot + 1;
                v_seen = mbar_test_wait(&B.full[ns], (ns == 0 ? use + 1 : use) & 1);
              }
              if (lead) {
                score(half, slot, HD / 16 - 1);
                umma_commit(&B.s_full[half]);
              }
            } else {
              if (lead) umma_commit(&B.o_done[half]);
              p_seen = nh > 0 && mbar_test_wait(&B.p_half[nh], (p_ph >> nh) & 1);
            }
          }
          if (!ok) break;
          if (lead) umma_commit(&B.empty[vs]);
          if (more) {
            if (lead) umma_commit(&B.empty[slot]);
            advance();
          }
        }
      }
      if (!ok && lead) atomicExch(&B.abort_flag, 1);
    }
  } else {
    // ---------------- softmax, a thread per row
    const int half = warp >> 2, r = threadIdx.x & 127;
    const uint32_t lane_base = static_cast<uint32_t>((warp & 3) * 32) << 16;
    const uint32_t t_s = tmem + half * 128 + lane_base, t_o = tmem + Lay::kTmemO + half * 128 + lane_base;
    const float sl = A.scale_log2;
    uint8_t* const q_tile = sb + Lay::kQ + half * Lay::kTile;
    // This row's flushed sum, the maximum it refers to, and its flushed accumulator (four elements in 16 bytes, a warp's
    // rows side by side).
    float* const flushed_l = reinterpret_cast<float*>(sb + Lay::kFlushed);
    float* const flushed_m = flushed_l + kFwRows;
    // The accumulator plus f times the flushed one: kept there with zeros in TMEM, or left in TMEM at the end of an item.
    auto move_sums = [&](float f, bool first, bool out) {
      float4* at = reinterpret_cast<float4*>(A.flush + static_cast<int64_t>(blockIdx.x) * kFwRows * HD) + threadIdx.x;
#pragma unroll 1
      for (int c = 0; c < HD; c += 4, at += kFwRows) {
        uint32_t o[4];
        tmem_ld4(t_o + c, o);
        tmem_wait_ld4(o);
        float4 a = first ? make_float4(0.f, 0.f, 0.f, 0.f) : *at;
        a = make_float4(fmaf(a.x, f, __uint_as_float(o[0])), fmaf(a.y, f, __uint_as_float(o[1])),
                        fmaf(a.z, f, __uint_as_float(o[2])), fmaf(a.w, f, __uint_as_float(o[3])));
        if (out) {
          *at = a;
          a = make_float4(0.f, 0.f, 0.f, 0.f);
        }
        tmem_st4(t_o + c, __float_as_uint(a.x), __float_as_uint(a.y), __float_as_uint(a.z), __float_as_uint(a.w));
      }
      tmem_wait_st();
    };
    // a wait that gave up ends the whole warp's work (its lanes vote and exchange below)
    int seg_no = 0, tile_no = 0;
    int v_slot = 1, v_use = 0;  // ring position of the current tile's V
    auto skip = [&](int tiles) {
      const int64_t p = static_cast<int64_t>(v_use) * Lay::kStages + v_slot + 2ll * tiles;
      v_use = static_cast<int>(p / Lay::kStages);
      v_slot = static_cast<int>(p - static_cast<int64_t>(v_use) * Lay::kStages);
    };
    // Q rows of an item into the swizzled tile, asynchronously: a warp copies its own 32 rows, HD / 8 lanes a row
    auto load_q = [&](const FwSeg& g) {
      const FwSide& sd = A.side[g.side];
      const XSide& s = sd.s;
      const int64_t R = side_rows(s), row = static_cast<int64_t>(g.rt) * kFwRows + half * 128 + r;
      const int64_t mine = row < R ? q_offset(s, g.bi, g.h, fw_row(sd, row)) : -1;
      constexpr int kLanes = HD / 8, kPer = 32 / kLanes;
      const int c = lane % kLanes;
      const __nv_bfloat16* q = static_cast<const __nv_bfloat16*>(s.q);
#pragma unroll
      for (int i = 0; i < 32 / kPer; ++i) {
        const int tr = (warp & 3) * 32 + i * kPer + lane / kLanes;
        const int64_t off = __shfl_sync(0xffffffffu, mine, i * kPer + lane / kLanes);
        const bool in = off >= 0 && c * 8 < A.D;
        cp_async16(q_tile + (c >> 3) * 16384 + tr * 128 + (((c & 7) ^ (tr & 7)) << 4), in ? q + off + c * 8 : q, in);
      }
    };
    auto finish_q = [&] {
      cp_async_wait_all();
      if (A.q_flip) {  // a negative scale: flip Q's signs, and scale by its magnitude
        __syncwarp();
        constexpr int kLanes = HD / 8, kPer = 32 / kLanes;
        const int c = lane % kLanes;
        for (int i = 0; i < 32 / kPer; ++i) {
          const int tr = (warp & 3) * 32 + i * kPer + lane / kLanes;
          uint4* p = reinterpret_cast<uint4*>(q_tile + (c >> 3) * 16384 + tr * 128 + (((c & 7) ^ (tr & 7)) << 4));
          const uint4 v = *p;
          *p = make_uint4(v.x ^ A.q_flip, v.y ^ A.q_flip, v.z ^ A.q_flip, v.w ^ A.q_flip);
        }
      }
      fence_proxy_async_smem();
      mbar_arrive(&B.q_full[half]);
    };
    auto active = [&](const FwSeg& g) {
      if (g.side < 0 || g.k0 == g.k1) return false;
      return half == 0 || static_cast<int64_t>(g.rt) * kFwRows + 128 < side_rows(A.side[g.side].s);
    };
    int seg_i = 0;
    auto next_seg = [&](FwSeg& x) {
      if (!warp_all(read_seg(seg_i, x))) return false;
      if (lane == 0) mbar_arrive(&B.seg_empty[seg_i % kFwSegs]);
      ++seg_i;
      return true;
    };

    FwSeg g, gn;
    bool ok = warp_all(!*abort_flag) && next_seg(g);
    if (ok && active(g)) {
      load_q(g);
      finish_q();
    }
    while (ok && g.side >= 0) {
      if (!active(g)) {
        if (g.k0 == g.k1) {  // a whole item without keys: zeros
          const XSide& s = A.side[0].s;
          const int64_t row = static_cast<int64_t>(g.rt) * kFwRows + half * 128 + r;
          if (row < side_rows(s)) {
            const XRow x = fw_row(A.side[0], row);
            __nv_bfloat16* ob = A.out + o_offset(s, g.bi, g.h, x);
            for (int d = 0; d < A.D; d += 8) *reinterpret_cast<uint4*>(ob + d) = make_uint4(0u, 0u, 0u, 0u);
            if (A.lse != nullptr) A.lse[flat_row(s, g.bi, g.h, x)] = -INFINITY;
          }
        }
        skip(g.k1 - g.k0);
        if (!next_seg(gn)) { ok = false; break; }
        if (active(gn)) {
          load_q(gn);
          finish_q();
        }
        g = gn;
        continue;
      }
      const FwSide& sd = A.side[g.side];
      const XSide& s = sd.s;
      const int64_t R = side_rows(s), row = static_cast<int64_t>(g.rt) * kFwRows + half * 128 + r;
      const bool live = row < R;
      const int len = g.len;
      int lim = 0;
      if (live) lim = s.causal ? row_limit(s, fw_row(sd, row), len) : len;
      const uint8_t* mask = s.mask ? s.mask + g.bi * s.mask_stride : nullptr;
      const bool warp_live = __any_sync(0xffffffffu, live);
      float m = -INFINITY, l = 0.f;
      for (int j = g.k0; j < g.k1; ++j, ++tile_no) {
        const int key0 = j * kFwKeys;
        // clean: every key of the tile counts; part: some are hidden from a row of this warp
        const bool clean = mask == nullptr && key0 + kFwKeys <= len;
        const bool part = !clean || __any_sync(0xffffffffu, live && key0 + kFwKeys > lim);
        if (!warp_all(!*abort_flag && mbar_wait(&B.s_full[half], tile_no & 1))) { ok = false; break; }
        tc_fence_after();
        if (j + 1 == g.k1) {
          // every score product of this item has run: the next item's Q takes the tile while the last P is formed
          if (!next_seg(gn)) { ok = false; break; }
          if (active(gn)) load_q(gn);
        }
        if (half == 0 && !clean) {
          // V rows of hidden keys become zeros before any product reads the tile (the second
          // half's P V is issued after the first half's)
          if (!warp_all(mbar_wait(&B.full[v_slot], v_use & 1))) { ok = false; break; }
          const int key = key0 + r;
          if (!(key < len && (mask == nullptr || mask[key] != 0))) {
            uint8_t* vr = sb + Lay::kRing + v_slot * Lay::kTile + r * 128;
#pragma unroll
            for (int c = 0; c < Lay::kChunks; ++c)
#pragma unroll
              for (int u = 0; u < 8; ++u) *reinterpret_cast<uint4*>(vr + c * 16384 + u * 16) = make_uint4(0u, 0u, 0u, 0u);
          }
          fence_proxy_async_smem();
        }
        if (warp_live) {
          // Hidden scores become -inf in place, in a loop of its own: the code below stays one, small and
          // without spills.
          if (part) {
#pragma unroll 1
            for (int c = 0; c < 4; ++c) {
              const int key = key0 + 32 * c + lane, n = min(max(lim - key0 - 32 * c, 0), 32);
              uint32_t vis = __ballot_sync(0xffffffffu, key < len && (mask == nullptr || mask[key] != 0));
              vis &= n == 32 ? ~0u : (1u << n) - 1u;
              uint32_t v[32];
              tmem_ld32(t_s + c * 32, v);
              tmem_wait_ld32(v);
#pragma unroll
              for (int i = 0; i < 32; ++i) v[i] = (vis >> i) & 1u ? v[i] : 0xff800000u;
              tmem_st32(t_s + c * 32, v);
            }
            tmem_wait_st();
          }
          // s_full of this tile implies the previous P V has completed
          if (j > g.k0 && (j - g.k0) % kFwFlushTiles == 0) {
            const bool first = j - g.k0 == kFwFlushTiles;
            const float was = first ? -INFINITY : flushed_m[threadIdx.x], f = was == -INFINITY ? 0.f : ex2(was - m);
            move_sums(f, first, true);
            flushed_l[threadIdx.x] = first ? l : fmaf(flushed_l[threadIdx.x], f, l);
            flushed_m[threadIdx.x] = m;
            l = 0.f;
          }
          // Scores come in chunks of 32 columns, and the first two are read again once the maximum is known:
          // all 128 do not fit beside the rest of a thread's 168 registers, and a spill is slow (224 KB of
          // shared memory leave local memory no L1). A chunk is in flight while the one before is used. One in
          // four exponentials runs on the FMA pipe: the special-function unit alone (16 a clock) needs 2048
          // clocks for the two halves' tile, as long as the products.
          uint32_t v0[32], v1[32], v2[32], v3[32];
          float a0 = -INFINITY, a1 = -INFINITY, a2 = -INFINITY, a3 = -INFINITY;
          auto maxes = [&](uint32_t (&v)[32]) {
#pragma unroll
            for (int i = 0; i < 32; i += 8) {
              a0 = max3_nan(a0, __uint_as_float(v[i]), __uint_as_float(v[i + 1]));
              a1 = max3_nan(a1, __uint_as_float(v[i + 2]), __uint_as_float(v[i + 3]));
              a2 = max3_nan(a2, __uint_as_float(v[i + 4]), __uint_as_float(v[i + 5]));
              a3 = max3_nan(a3, __uint_as_float(v[i + 6]), __uint_as_float(v[i + 7]));
            }
          };
          tmem_ld32(t_s, v0);
          tmem_wait_ld32(v0);
          tmem_ld32(t_s + 32, v1);
          maxes(v0);
          tmem_wait_ld32(v1);
          tmem_ld32(t_s + 64, v2);
          maxes(v1);
          tmem_wait_ld32(v2);
          tmem_ld32(t_s + 96, v3);
          maxes(v2);
          tmem_wait_ld32(v3);
          maxes(v3);
          a0 = max3_nan(max3_nan(a0, a1, a2), a3, a3);
          const float bmax = a0 == -INFINITY ? a0 : a0 * sl;
          const float mnew = bmax <= m + kFwLazy ? m : bmax;  // a NaN moves in and stays
          const float mu = mnew == -INFINITY ? 0.f : mnew;
          const float corr = ex2(m - mu);  // 1 when m stays, 0 before the first key
          // s_full of this tile implies the previous P V has completed: O may be rescaled
          if (j > g.k0 && __any_sync(0xffffffffu, mnew != m)) {
#pragma unroll 1
            for (int c = 0; c < HD / 16; ++c) {
              uint32_t o[16];
              tmem_ld16(t_o + c * 16, o);
              tmem_wait_ld16(o);
#pragma unroll
              for (int i = 0; i < 16; ++i) o[i] = __float_as_uint(__uint_as_float(o[i]) * corr);
              tmem_st16(t_o + c * 16, o);
            }
          }
          m = mnew;
          uint64_t sum_a = pack2(l * corr, 0.f), sum_b = pack2(0.f, 0.f);
          const uint64_t sl2 = pack2(sl, sl), mu2 = pack2(-mu, -mu);
          uint32_t pk[32];
          auto probs = [&](uint32_t (&v)[32], uint32_t* out) {
#pragma unroll
            for (int i = 0; i < 32; i += 2) {
              const uint64_t x = fma2(pack2(__uint_as_float(v[i]), __uint_as_float(v[i + 1])), sl2, mu2);
              float e0, e1;
              if (i % 8 == 6) {
                exp2_poly2(x, e0, e1);
              } else {
                unpack2(x, e0, e1);
                e0 = ex2(e0);
                e1 = ex2(e1);
              }
              if (i & 2) sum_b = add2(sum_b, pack2(e0, e1));
              else sum_a = add2(sum_a, pack2(e0, e1));
              out[i / 2] = pack_bf16(e0, e1);
            }
          };
          // P of the last 64 keys goes over their scores first, so that its product starts half a tile early
          probs(v2, pk);
          tmem_ld32(t_s, v0);
          probs(v3, pk + 16);
          tmem_st32(t_s + 64, pk);
          tmem_wait_st();
          tc_fence_before();
          mbar_arrive(&B.p_half[half]);
          tmem_wait_ld32(v0);
          tmem_ld32(t_s + 32, v1);
          probs(v0, pk);
          tmem_wait_ld32(v1);
          probs(v1, pk + 16);
          tmem_st32(t_s, pk);
          float s0, s1, s2, s3;
          unpack2(sum_a, s0, s1);
          unpack2(sum_b, s2, s3);
          l = (s0 + s1) + (s2 + s3);
          tmem_wait_st();
        } else {
          mbar_arrive(&B.p_half[half]);
        }
        tc_fence_before();
        mbar_arrive(&B.p_full[half]);
        skip(1);
      }
      if (!ok) break;
      if (active(gn)) finish_q();
      if (!warp_all(mbar_wait(&B.o_done[half], seg_no & 1) && !*abort_flag)) { ok = false; break; }
      ++seg_no;
      tc_fence_after();
      if (warp_live) {
        if (g.k1 - g.k0 > kFwFlushTiles) {
          const float was = flushed_m[threadIdx.x], f = was == -INFINITY ? 0.f : ex2(was - m);
          l = fmaf(flushed_l[threadIdx.x], f, l);
          move_sums(f, false, false);
        }
        const float inv = m == -INFINITY ? 0.f : 1.f / l;  // no key: zero
        const float ls = m == -INFINITY ? -INFINITY : m + log2f(l);
        const XRow x = fw_row(sd, live ? row : 0);
        const bool all = g.k0 == 0 && g.k1 == g.n;
        const bool to_slot = !all || A.keep;
        float* po = nullptr;
        __nv_bfloat16* ob = nullptr;
        int slot_stride = 0;
        if (to_slot) {
          const int64_t slot = all ? g.item : 2ll * blockIdx.x + (g.k0 == 0 ? 1 : 0);
          slot_stride = all ? sd.item_rows : sd.slot_rows;
          po = (all ? sd.item_slots : sd.slots) + slot * slot_stride * A.D;
          if (live) (all ? sd.item_lse : sd.slot_lse)[slot * slot_stride + half * 128 + r] = ls;
          po += (half * 128 + r) * 4;
        } else if (live) {
          ob = A.out + o_offset(s, g.bi, g.h, x);
          if (A.lse != nullptr) A.lse[flat_row(s, g.bi, g.h, x)] = ls;
        }
#pragma unroll 1
        for (int c = 0; c < HD / 32; ++c) {
          uint32_t o[32];
          tmem_ld32(t_o + c * 32, o);
          tmem_wait_ld32(o);
          auto f = [&](int i) { return __uint_as_float(o[i]) * inv; };
          if (to_slot) {
#pragma unroll
            for (int i = 0; i < 32; i += 4)
              if (live && c * 32 + i < A.D)
                *reinterpret_cast<float4*>(po + static_cast<int64_t>(c * 8 + i / 4) * slot_stride * 4) =
                    make_float4(f(i), f(i + 1), f(i + 2), f(i + 3));
          } else {
            // four lanes exchange their four 16-byte pieces, so that a store writes 64 contiguous bytes of a row
            uint4 q[4];
#pragma unroll
            for (int i = 0; i < 4; ++i)
              q[i] = make_uint4(pack_bf16(f(8 * i), f(8 * i + 1)), pack_bf16(f(8 * i + 2), f(8 * i + 3)),
                                pack_bf16(f(8 * i + 4), f(8 * i + 5)), pack_bf16(f(8 * i + 6), f(8 * i + 7)));
            quad_transpose(q, lane & 3);
            const int d = c * 32 + (lane & 3) * 8;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
              __nv_bfloat16* row = reinterpret_cast<__nv_bfloat16*>(
                  __shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(ob), (lane & ~3) + k));
              if (row != nullptr && d < A.D) *reinterpret_cast<uint4*>(row + d) = q[k];
            }
          }
        }
      }
      tc_fence_before();  // O is read before the next item's first P V (ordered by p_full)
      g = gn;
    }
    if (!ok) atomicExch(&B.abort_flag, 1);
  }
  __syncwarp();
  tc_fence_before();
  __syncthreads();
  if (warp == 9) {
    tc_fence_after();
    tmem_dealloc(tmem, 512);
  }
}

// Joins the pieces of every row of the split part. A thread has 4 elements of a row in U places 32 elements apart, rows
// fastest, as the slots are laid out (whole lines for 32 rows); a block has up to 32 rows and 8 U groups of 4 elements.
// One side: rows of a split item (items that one CTA finished are done). Two sides: 32 packed rows of the prefix's
// items of a key head, which are rows of one or more sequences' own items.
// A load takes about a microsecond here, so what counts is how many follow one another: BATCH pieces of a thread are in
// flight together, 8 where an item has few rows and many pieces, or a prefix's; 2 in U = 4 places where large items
// were cut once.
template <int BATCH, int U>
__global__ void __launch_bounds__(256, U > 1 ? 3 : 2) xattn_join_kernel(const __grid_constant__ FwArgs A) {
  __shared__ __align__(16) uint2 tile[32][8 * U];
  const FwSide& L = A.side[0];  // whose rows the blocks walk
  const FwSide& S = A.side[A.sides - 1];
  const int item = A.sides == 1 ? blockIdx.x + L.first : blockIdx.x;
  const int per = L.s.hkv * L.row_tiles, bi = item / per, rem = item - bi * per, h = rem / L.row_tiles;
  const int rt = rem - h * L.row_tiles;
  const int64_t R = side_rows(L.s), row0 = static_cast<int64_t>(rt) * L.tile_rows + blockIdx.y * 32;
  const int rows = static_cast<int>(min(static_cast<int64_t>(32), min(R, static_cast<int64_t>(rt + 1) * L.tile_rows) - row0));
  if (rows <= 0) return;
  const int c0 = blockIdx.z * 8 * U, cw = min(8 * U, A.D / 4 - c0);
  grid_dep_wait();
  const int n = fw_tiles(L, bi);
  const int2 p = n > 0 ? L.pieces[item - L.first] : make_int2(0, -1);
  if (A.sides == 1 && n > 0 && p.x == p.y) return;
  for (int i = threadIdx.x; i < rows * min(8, cw); i += blockDim.x) {
    const int c = i / rows, r = i - c * rows;
    const int64_t row = row0 + r;
    float mx = -INFINITY, den = 0.f;
    float4 acc[U];
#pragma unroll
    for (int u = 0; u < U; ++u) acc[u] = make_float4(0.f, 0.f, 0.f, 0.f);
    auto add = [&](const float* slots, const float* lse, int stride, int at, int count, auto&& slot_of) {
      for (int k0 = 0; k0 < count; k0 += BATCH) {
        float ls[BATCH];
        float4 o[BATCH][U];
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          ls[k] = -INFINITY;
#pragma unroll
          for (int u = 0; u < U; ++u) o[k][u] = make_float4(0.f, 0.f, 0.f, 0.f);
          if (k0 + k < count) {
            const int64_t slot = slot_of(k0 + k);
            ls[k] = lse[slot * stride + at];
#pragma unroll
            for (int u = 0; u < U; ++u)
              if (U == 1 || c + 8 * u < cw)
                o[k][u] = *reinterpret_cast<const float4*>(
                    slots + slot * stride * A.D + (static_cast<int64_t>(c0 + c + 8 * u) * stride + at) * 4);
          }
        }
        float mn = mx;
#pragma unroll
        for (int k = 0; k < BATCH; ++k) mn = max3_nan(mn, mn, ls[k]);
        const float base = mn == -INFINITY ? 0.f : mn, f = exp2f(mx - base);
        den *= f;
#pragma unroll
        for (int u = 0; u < U; ++u) acc[u] = make_float4(acc[u].x * f, acc[u].y * f, acc[u].z * f, acc[u].w * f);
#pragma unroll
        for (int k = 0; k < BATCH; ++k) {
          const float w = exp2f(ls[k] - base);
          den += w;
#pragma unroll
          for (int u = 0; u < U; ++u)
            acc[u] = make_float4(fmaf(w, o[k][u].x, acc[u].x), fmaf(w, o[k][u].y, acc[u].y),
                                 fmaf(w, o[k][u].z, acc[u].z), fmaf(w, o[k][u].w, acc[u].w));
        }
        mx = mn;
      }
    };
    auto pieces = [&](int2 q, const FwSide& sd, int it, int at) {
      const bool single = A.sides > 1 && q.x == q.y;
      add(single ? sd.item_slots : sd.slots, single ? sd.item_lse : sd.slot_lse, single ? sd.item_rows : sd.slot_rows, at,
          q.y - q.x + 1, [&](int k) { return single ? static_cast<int64_t>(it) : 2ll * (q.x + k) + (k == 0 ? 1 : 0); });
    };
    int own_item = 0, own_at = 0;
    int2 own = make_int2(0, -1);
    XRow x = fw_row(L, row);
    int ob = bi;
    if (A.sides > 1) {
      // packed row (b, g, t) of the prefix is row (g, t) of sequence b
      const int orow = x.g * S.s.T + x.t, ort = orow / S.tile_rows;
      ob = x.b2;
      x.b2 = 0;
      own_item = (ob * S.s.hkv + h) * S.row_tiles + ort;
      own_at = orow - ort * S.tile_rows;
      if (side_len(S.s, ob) > 0) own = S.pieces[own_item];
    }
    pieces(p, L, item, blockIdx.y * 32 + r);
    if (A.sides > 1) pieces(own, S, own_item, own_at);
    const float inv = den == 0.f ? 0.f : 1.f / den;
#pragma unroll
    for (int u = 0; u < U; ++u) {
      const uint2 v =
          make_uint2(pack_bf16(acc[u].x * inv, acc[u].y * inv), pack_bf16(acc[u].z * inv, acc[u].w * inv));
      if (rows == 32) tile[r][c + 8 * u] = v;
      else if (c + 8 * u < cw) *reinterpret_cast<uint2*>(A.out + o_offset(S.s, ob, h, x) + (c0 + c + 8 * u) * 4) = v;
    }
    if (A.lse != nullptr && c0 + c == 0) A.lse[flat_row(S.s, ob, h, x)] = den == 0.f ? -INFINITY : mx + log2f(den);
  }
  if (rows < 32) return;
  __syncthreads();
  // 32 rows leave in 64 U contiguous bytes each
  for (int i = threadIdx.x; i < 32 * (cw / 2); i += blockDim.x) {
    const int r = i / (cw / 2), u = i - r * (cw / 2);
    XRow x = fw_row(L, row0 + r);
    int ob = bi;
    if (A.sides > 1) {
      ob = x.b2;
      x.b2 = 0;
    }
    *reinterpret_cast<uint4*>(A.out + o_offset(S.s, ob, h, x) + c0 * 4 + u * 8) =
        *reinterpret_cast<const uint4*>(&tile[r][u * 2]);
  }
}

// One launch: the sides it takes (all of the call's, or one of two), in the form their rows ask for.
struct FwLaunch {
  bool few;
  int sides, side[2], grid, whole, split_items, slot_rows;
  int64_t items[2];
  size_t o, lse, flush, item_o[2], item_lse[2], pieces[2];  // byte offsets in the workspace
};
struct FwPlan {
  int launches;
  FwLaunch l[2];
  size_t total;
};

FwPlan fw_plan(const trnsparse_attention_args* a, const XSide (&s)[2], int n) {
  FwPlan p = {};
  bool few[2] = {false, false};
  for (int i = 0; i < n; ++i) {
    const int64_t item = (s[i].klen + (1ll << kFewKeyShift) - 1) >> kFewKeyShift;
    const int64_t run = item * s[i].nb * s[i].hkv / few_rows_grid();  // where it is below an item, no CTA has a whole one
    few[i] = side_rows(s[i]) <= kFewRows && (item < run ? item : run) <= kFewMostTiles;
  }
  p.launches = n > 1 && few[0] != few[1] ? 2 : 1;
  size_t at = 0;
  const size_t D = static_cast<size_t>(a->head_dim);
  for (int i = 0; i < p.launches; ++i) {
    FwLaunch& l = p.l[i];
    l.sides = p.launches == 2 ? 1 : n;
    l.few = few[p.launches == 2 ? i : 0];
    const int64_t tile_rows = l.few ? kFewRows : kFwRows, shift = l.few ? kFewKeyShift : kFwKeyShift;
    int64_t most = 0, tiles = 0, items = 0, longest = 0;
    for (int j = 0; j < l.sides; ++j) {
      const XSide& x = s[l.side[j] = p.launches == 2 ? i : j];
      const int64_t R = side_rows(x);
      l.items[j] = (R + tile_rows - 1) / tile_rows * x.nb * x.hkv;
      items += l.items[j];
      longest = longest > (x.klen >> shift) ? longest : x.klen >> shift;
      tiles += l.items[j] * ((x.klen + (1ll << shift) - 1) >> shift);
      most = most > R ? most : R;
    }
    // Beside the own keys' launch the prefix's takes as many SMs as give a CTA kFwLeast tiles: each of its pieces is
    // written and joined (256 rows in fp32), and the other launch has work for the rest of the SMs.
    const int64_t least = tiles / kFwLeast > 0 ? tiles / kFwLeast : 1, sms = sm_count();
    const int64_t full = l.few ? few_rows_grid() : p.launches == 2 && least < sms ? least : sms;
    l.grid = static_cast<int>(tiles < full ? (tiles > 0 ? tiles : 1) : full);
    // One side: whole items for all but the last round (items of one length), or the last one to two rounds, which
    // then even out what unequal lengths left.
    const XSide& x0 = s[l.side[0]];
    const int last = x0.lengths != nullptr && x0.nb > 1 ? 1 : 0;
    if (n == 1 && items >= (1 + last) * static_cast<int64_t>(l.grid)) l.whole = static_cast<int>(items / l.grid - last);
    l.split_items = static_cast<int>(items - static_cast<int64_t>(l.whole) * l.grid);
    l.slot_rows = static_cast<int>(most < tile_rows ? most : tile_rows);
    auto take = [&](size_t bytes) {
      const size_t was = at;
      at += align256(bytes);
      return was;
    };
    l.o = take(sizeof(float) * 2 * l.grid * l.slot_rows * D);
    l.lse = take(sizeof(float) * 2 * l.grid * l.slot_rows);
    l.flush = take(!l.few && longest >= kFwFlushTiles ? sizeof(float) * l.grid * kFwRows * (D <= 64 ? 64 : 128) : 0);
    for (int j = 0; j < l.sides; ++j) {
      const int64_t R = side_rows(s[l.side[j]]), rows = R < tile_rows ? R : tile_rows;
      l.item_o[j] = take(n > 1 ? sizeof(float) * l.items[j] * rows * D : 0);
      l.item_lse[j] = take(n > 1 ? sizeof(float) * l.items[j] * rows : 0);
      l.pieces[j] = take(sizeof(int2) * (n > 1 ? l.items[j] : l.split_items));
    }
  }
  p.total = at;
  return p;
}

template <int HD>
int fw_launch(const FwArgs& A, const XMap (&m)[4], int grid, cudaStream_t st) {
  using Lay = FwLayout<HD>;
  auto kern = xattn_fwd_tc_kernel<HD>;
  static unsigned long long done = 0;  // a bit per device; setting the attribute again is harmless
  int rc = allow_smem(kern, Lay::kSmem, &done, "attention (tensor cores): set smem");
  if (rc) return rc;
  kern<<<grid, kFwThreads, Lay::kSmem, st>>>(m[0].map, m[1].map, m[2].map, m[3].map, A);
  TSB_CHECK_LAUNCH("attention (tensor cores) launch");
  return debug_sync(st, "attention (tensor cores)");
}

}  // namespace

bool xattn_tc_ok(const trnsparse_attention_args* a, bool prefix) {
  if (a->dtype != TRNSPARSE_BF16 || a->head_dim % 8 || a->head_dim > 128) return false;
  if (prefix ? a->prefix_len + a->k_len == 0 : a->k_len == 0) return false;
  if (!aligned16(a->q) || !aligned16(a->out)) return false;
  if (!strides_ok(a->q_strides, a->batch, a->q_heads, a->q_len, false) ||
      !strides_ok(a->out_strides, a->batch, a->q_heads, a->q_len, false))
    return false;
  if (a->k_len > 0 && (!aligned16(a->k) || !aligned16(a->v) ||
                       !strides_ok(a->k_strides, a->batch, a->kv_heads, a->k_len, true) ||
                       !strides_ok(a->v_strides, a->batch, a->kv_heads, a->k_len, true)))
    return false;
  if (prefix && a->prefix_len > 0) {
    const int64_t ks[3] = {0, a->prefix_k_strides[0], a->prefix_k_strides[1]};
    const int64_t vs[3] = {0, a->prefix_v_strides[0], a->prefix_v_strides[1]};
    if (!aligned16(a->prefix_k) || !aligned16(a->prefix_v) || !strides_ok(ks, 1, a->kv_heads, a->prefix_len, true) ||
        !strides_ok(vs, 1, a->kv_heads, a->prefix_len, true))
      return false;
  }
  return true;
}

size_t xattn_tc_workspace(const trnsparse_attention_args* a, bool prefix) {
  XSide s[2];
  int n = 0;
  if (make_sides(a, prefix, s, &n)) return 0;
  return fw_plan(a, s, n).total;
}

int xattn_tc_forward(const trnsparse_attention_args* a, bool prefix, void* ws, cudaStream_t st) {
  XSide s[2];
  int n = 0;
  int rc = make_sides(a, prefix, s, &n);
  if (rc) return rc;
  const FwPlan p = fw_plan(a, s, n);
  char* w = static_cast<char*>(ws);
  const int64_t D = a->head_dim;
  FwArgs J = {};  // the call as a whole, for the join
  J.sides = n;
  J.D = static_cast<int>(D);
  J.out = static_cast<__nv_bfloat16*>(a->out);
  J.lse = a->lse;
  // a scale of 0 (or too small for fp32) stays above 0, so that a hidden score of -inf stays -inf
  J.scale_log2 = fmaxf(static_cast<float>(fabs(a->scale) * 1.4426950408889634), 1e-37f);
  J.q_flip = a->scale < 0 ? 0x80008000u : 0u;
  J.keep = n > 1;
  for (int i = 0; i < p.launches; ++i) {
    const FwLaunch& l = p.l[i];
    FwArgs A = J;
    A.sides = l.sides;
    A.whole = l.whole;
    for (int j = 0; j < l.sides; ++j) {
      FwSide& S = A.side[j];
      S.s = s[l.side[j]];
      S.tile_rows = l.few ? kFewRows : kFwRows;
      S.key_shift = l.few ? kFewKeyShift : kFwKeyShift;
      const int64_t R = side_rows(S.s);
      S.row_tiles = static_cast<int>((R + S.tile_rows - 1) / S.tile_rows);
      S.items = static_cast<int>(l.items[j]);
      S.by_T = fast_div(S.s.T);
      S.by_G = fast_div(S.s.G);
      S.slots = reinterpret_cast<float*>(w + l.o);
      S.slot_lse = reinterpret_cast<float*>(w + l.lse);
      S.slot_rows = l.slot_rows;
      S.item_slots = reinterpret_cast<float*>(w + l.item_o[j]);
      S.item_lse = reinterpret_cast<float*>(w + l.item_lse[j]);
      S.item_rows = static_cast<int>(R < S.tile_rows ? R : S.tile_rows);
      S.pieces = reinterpret_cast<int2*>(w + l.pieces[j]);
      S.first = l.whole * l.grid;
    }
    if (l.few) {
      rc = few_rows_launch(A, l.grid, i > 0, st);
    } else {
      A.item_cost = kFwItemCost;
      A.flush = reinterpret_cast<float*>(w + l.flush);
      A.seg_ns = kWaitNs;
      for (int j = 0; j < l.sides; ++j)
        A.seg_ns += kFwTileNs * static_cast<uint64_t>((A.side[j].s.klen >> kFwKeyShift) + 1);
      XMap m[4];
      for (int j = 0; j < l.sides && !rc; ++j) {
        FwSide& S = A.side[j];
        const XSide& x = S.s;
        rc = make_xmap(&m[2 * j], x.k, D, x.klen, x.hkv, x.nb, x.k_t, x.k_h, x.k_b, 128);
        if (!rc) rc = make_xmap(&m[2 * j + 1], x.v, D, x.klen, x.hkv, x.nb, x.v_t, x.v_h, x.v_b, 128);
        S.mul_kh = m[2 * j].mul_h;
        S.mul_kb = m[2 * j].mul_b;
        S.mul_vh = m[2 * j + 1].mul_h;
        S.mul_vb = m[2 * j + 1].mul_b;
      }
      for (int j = 2 * l.sides; j < 4; ++j) m[j] = m[j - 2];
      if (!rc) rc = D <= 64 ? fw_launch<64>(A, m, l.grid, st) : fw_launch<128>(A, m, l.grid, st);
    }
    if (rc) return rc;
    for (int j = 0; j < l.sides; ++j) J.side[l.side[j]] = A.side[j];
  }
  const FwLaunch& l = p.l[p.launches - 1];
  const FwSide& W = J.side[0];
  const int blocks = n == 1 ? l.split_items : W.items;
  if (blocks == 0) return TRNSPARSE_OK;
  const int threads = W.item_rows >= 32 ? 256 : (W.item_rows * 8 + 31) & ~31;
  const bool large = n == 1 && W.item_rows >= 32;
  auto kern = large ? xattn_join_kernel<2, 4> : xattn_join_kernel<8, 1>;
  const unsigned groups = large ? 32 : 8;  // of 4 elements a block
  cudaError_t e = launch_pdl(kern, dim3(blocks, (W.item_rows + 31) / 32, (a->head_dim / 4 + groups - 1) / groups),
                             dim3(threads), 0, st, J);
  if (e != cudaSuccess) return cuda_status(e, "attention (tensor cores): join");
  return debug_sync(st, "attention (tensor cores): join");
}

}  // namespace tsb
