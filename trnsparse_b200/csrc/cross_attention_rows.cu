// Attention forward for few rows (at most 16 packed rows an item: decoding), bf16 in and out, fp32 softmax and
// sums, head_dim a multiple of 8 up to 128. The mathematics, the hidden keys and the work split are those of
// cross_attention_tc.cu; the result of an item is joined from its pieces by the same kernel.
//
// What bounds it: memory, K and V read once (at 4 query heads a key head one key of head_dim 128 is 512 bytes and
// 1024 multiply-adds). A 128-row tcgen05 tile would be padding and one chain S -> softmax -> P V per 128 keys; here
// the rows are the 16 of an m16n8k16 product and every warp has keys of its own, so four chains run in a CTA and
// eight on an SM, and nothing but the loads is waited for:
//   warp 4       the list of (item, keys), and TMA: tiles of 64 keys, K and V together, through a ring (80 KB in
//                flight a CTA at head_dim 64, 64 KB at 128; two CTAs an SM)
//   warps 0-3    16 keys each of a tile: S by ldmatrix and mma, softmax in registers with the warp's own running
//                maximum and sum, P V with P as it lies in registers; the four partial results of an item are
//                joined through shared memory.
// Measured against the 128-row kernel at 32 x 16 heads, 1500 keys, head_dim 64: 41 against 81 us (197 MB).
#include "xattn_items.cuh"

namespace tsb {
namespace {

constexpr int kFrThreads = 160;
constexpr int kFrKeys = 1 << kFewKeyShift;
constexpr float kFrLazy = 8.f;
constexpr int kFrItemCost = 2;  // in key tiles

template <int HD>
struct FrLayout {
  static constexpr int kChunks = HD / 64;
  static constexpr int kTile = kFrKeys * HD * 2;     // K or V of a tile
  static constexpr int kStages = HD == 128 ? 2 : 5;  // two CTAs an SM
  static constexpr int kMerge = kStages * 2 * kTile;  // float [4 warps][16 rows][HD]
  static constexpr int kStat = kMerge + 4 * kFewRows * HD * 4;  // float [2][4][16]: maximum, sum
  static constexpr int kBar = kStat + 2 * 4 * kFewRows * 4;
  static constexpr int kSmem = kBar + 384;
};

struct FrBars {
  uint64_t full[5], empty[5], seg_full[kFwSegs], seg_empty[kFwSegs], merge_full, merge_empty;
  FwSeg seg[kFwSegs];
  int abort_flag;
};
static_assert(sizeof(FrBars) <= 384, "FrLayout::kSmem");

__device__ __forceinline__ void ldmatrix4(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void ldmatrix4_trans(uint32_t addr, uint32_t (&r)[4]) {
  asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0, %1, %2, %3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(addr)
               : "memory");
}
__device__ __forceinline__ void mma16816(float (&c)[4], const uint32_t (&a)[4], uint32_t b0, uint32_t b1) {
  asm volatile(
      "mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0, %1, %2, %3}, {%4, %5, %6, %7}, {%8, %9}, {%0, %1, %2, "
      "%3};\n"
      : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
      : "r"(a[0]), "r"(a[1]), "r"(a[2]), "r"(a[3]), "r"(b0), "r"(b1));
}
__device__ __forceinline__ float quad_max(float v) {
  v = max3_nan(v, v, __shfl_xor_sync(0xffffffffu, v, 1));
  return max3_nan(v, v, __shfl_xor_sync(0xffffffffu, v, 2));
}

template <int HD>
__global__ void __launch_bounds__(kFrThreads, 2)
xattn_rows_kernel(const __grid_constant__ CUtensorMap tk0, const __grid_constant__ CUtensorMap tv0,
                  const __grid_constant__ CUtensorMap tk1, const __grid_constant__ CUtensorMap tv1,
                  const __grid_constant__ FwArgs A) {
  using Lay = FrLayout<HD>;
  extern __shared__ __align__(16) uint8_t sb[];  // no static shared memory: 1024-byte aligned
  FrBars& B = *reinterpret_cast<FrBars*>(sb + Lay::kBar);
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  if (threadIdx.x == 0) {
    for (int i = 0; i < Lay::kStages; ++i) {
      mbar_init(&B.full[i], 1);
      mbar_init(&B.empty[i], 4);
    }
    for (int i = 0; i < kFwSegs; ++i) {
      mbar_init(&B.seg_full[i], 1);
      mbar_init(&B.seg_empty[i], 4);
    }
    mbar_init(&B.merge_full, 128);
    mbar_init(&B.merge_empty, 128);
    B.abort_flag = (smem_u32(sb) & 1023u) ? 1 : 0;
    if (B.abort_flag) record_device_error(DEVERR_SELFCHECK_SMEM);
    fence_mbar_init();
  }
  __syncthreads();
  volatile int* abort_flag = &B.abort_flag;

  if (warp == 4) {
    // ---------------- the list of segments, and their tiles
    if (!*abort_flag) {
      FwCursor cur{A};
      const FwRun run = fw_start(A, cur, lane);
      if (lane == 0) {
        int slot = 0, use = 0;
        bool ok = true;
        FwSeg g;
        for (int i = 0; ok; ++i) {
          const bool whole = cur.w < A.whole, more = cur.next(g);
          if (!more) g.side = -1;
          if (i >= kFwSegs && !mbar_wait(&B.seg_empty[i % kFwSegs], (i / kFwSegs - 1) & 1)) {
            ok = false;
            break;
          }
          B.seg[i % kFwSegs] = g;
          mbar_arrive(&B.seg_full[i % kFwSegs]);
          if (!more) break;
          const FwSide& sd = A.side[g.side];
          if (!whole && g.k0 == 0) fw_note_pieces(A, cur, run, g);
          const CUtensorMap* tk = g.side ? &tk1 : &tk0;
          const CUtensorMap* tv = g.side ? &tv1 : &tv0;
          const int kh = g.h * sd.mul_kh, kb = g.bi * sd.mul_kb, vh = g.h * sd.mul_vh, vb = g.bi * sd.mul_vb;
          for (int j = g.k0; j < g.k1; ++j) {
            if (*abort_flag || (use > 0 && !mbar_wait(&B.empty[slot], (use - 1) & 1))) {
              ok = false;
              break;
            }
            uint8_t* dst = sb + slot * 2 * Lay::kTile;
            mbar_arrive_expect_tx(&B.full[slot], 2 * Lay::kTile);
            for (int c = 0; c < Lay::kChunks; ++c) {
              tma_load_4d(dst + c * (kFrKeys * 128), tk, c * 64, j * kFrKeys, kh, kb, &B.full[slot]);
              tma_load_4d(dst + Lay::kTile + c * (kFrKeys * 128), tv, c * 64, j * kFrKeys, vh, vb, &B.full[slot]);
            }
            if (++slot == Lay::kStages) {
              slot = 0;
              ++use;
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
    }
  } else {
    // ---------------- four warps, 16 keys of a tile each
    const int gr = lane >> 2, t4 = lane & 3;
    const float sl = A.scale_log2;
    float* const merge = reinterpret_cast<float*>(sb + Lay::kMerge);
    float* const stat = reinterpret_cast<float*>(sb + Lay::kStat);
    // lane's row of the 8 x 8 matrices an ldmatrix gathers: K (key, d half), V (key half, d)
    const int mi = lane >> 3, mr = lane & 7;
    const int k_key = warp * 16 + (mi >> 1) * 8 + mr, k_d8 = mi & 1;
    const int v_key = warp * 16 + (mi & 1) * 8 + mr, v_d8 = mi >> 1;
    int slot = 0, use = 0, seg_no = 0;
    bool ok = warp_all(!*abort_flag);
    for (int i = 0; ok; ++i) {
      if (!warp_all(mbar_wait(&B.seg_full[i % kFwSegs], (i / kFwSegs) & 1))) { ok = false; break; }
      const FwSeg g = B.seg[i % kFwSegs];
      __syncwarp();
      if (lane == 0) mbar_arrive(&B.seg_empty[i % kFwSegs]);
      if (g.side < 0) break;
      const FwSide& sd = A.side[g.side];
      const XSide& s = sd.s;
      const int R = static_cast<int>(side_rows(s));
      // Q as the A operand: rows gr and gr + 8, elements 2 t4, 2 t4 + 1 and eight further
      uint32_t q[HD / 16][4];
      int lim[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = gr + 8 * e;
        const bool live = row < R;
        const XRow x = fw_row(sd, live ? row : 0);
        lim[e] = live ? row_limit(s, x, g.len) : 0;
        const __nv_bfloat16* qp = static_cast<const __nv_bfloat16*>(s.q) + q_offset(s, g.bi, g.h, x);
#pragma unroll
        for (int kk = 0; kk < HD / 16; ++kk)
#pragma unroll
          for (int f = 0; f < 2; ++f) {
            const int d = kk * 16 + f * 8 + t4 * 2;
            uint32_t v = 0;
            if (live && d < A.D) v = __ldg(reinterpret_cast<const uint32_t*>(qp + d));
            q[kk][f * 2 + e] = v ^ A.q_flip;
          }
      }
      const uint8_t* mask = s.mask ? s.mask + g.bi * s.mask_stride : nullptr;
      float m[2] = {-INFINITY, -INFINITY}, l[2] = {0.f, 0.f};
      float o[HD / 8][4];
#pragma unroll
      for (int n = 0; n < HD / 8; ++n)
#pragma unroll
        for (int c = 0; c < 4; ++c) o[n][c] = 0.f;
      for (int j = g.k0; j < g.k1; ++j) {
        const int key0 = j * kFrKeys + warp * 16;
        if (!warp_all(!*abort_flag && mbar_wait(&B.full[slot], use & 1))) { ok = false; break; }
        uint8_t* const kt = sb + slot * 2 * Lay::kTile;
        uint8_t* const vt = kt + Lay::kTile;
        const bool clean = mask == nullptr && key0 + 16 <= g.len;
        if (key0 < g.len) {
          uint32_t kept = 0xffffu;
          if (!clean) {
            // V rows of hidden keys become zeros (this warp alone reads them)
            const int key = key0 + (lane & 15);
            kept = __ballot_sync(0xffffffffu, key < g.len && (mask == nullptr || mask[key] != 0)) & 0xffffu;
#pragma unroll 1
            for (int u = lane; u < 16 * (HD / 8); u += 32) {
              const int r = u / (HD / 8), c = u % (HD / 8);
              if (!((kept >> r) & 1u))
                *reinterpret_cast<uint4*>(vt + (c >> 3) * (kFrKeys * 128) + (warp * 16 + r) * 128 + (c & 7) * 16) =
                    make_uint4(0u, 0u, 0u, 0u);
            }
            fence_proxy_async_smem();  // the slot's next copy comes after these writes
            __syncwarp();
          }
          float sc[2][4] = {{0.f, 0.f, 0.f, 0.f}, {0.f, 0.f, 0.f, 0.f}};
          const uint32_t ka = smem_u32(kt) + k_key * 128, va = smem_u32(vt) + v_key * 128;
#pragma unroll
          for (int kk = 0; kk < HD / 16; ++kk) {
            uint32_t b[4];
            const int c8 = kk * 2 + k_d8;  // 16-byte unit of the key's row
            ldmatrix4(ka + (c8 >> 3) * (kFrKeys * 128) + (((c8 & 7) ^ (k_key & 7)) << 4), b);
            mma16816(sc[0], q[kk], b[0], b[1]);
            mma16816(sc[1], q[kk], b[2], b[3]);
          }
          // hidden scores: key 8 n + 2 t4 + c of the warp's 16, row gr + 8 e
          const bool part = !clean || __any_sync(0xffffffffu, (gr < R && key0 + 16 > lim[0]) || (gr + 8 < R && key0 + 16 > lim[1]));
          if (part) {
#pragma unroll
            for (int n = 0; n < 2; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) {
                const int k = n * 8 + t4 * 2 + (c & 1);
                if (!((kept >> k) & 1u) || key0 + k >= lim[c >> 1]) sc[n][c] = -INFINITY;
              }
          }
          float mu[2], corr[2];
          bool moved = false;
#pragma unroll
          for (int e = 0; e < 2; ++e) {
            float mx = max3_nan(sc[0][2 * e], sc[0][2 * e + 1], max3_nan(sc[1][2 * e], sc[1][2 * e + 1], sc[1][2 * e]));
            mx = quad_max(mx);
            mx = mx == -INFINITY ? mx : mx * sl;
            const float mn = mx <= m[e] + kFrLazy ? m[e] : mx;  // a NaN moves in and stays
            mu[e] = mn == -INFINITY ? 0.f : mn;
            corr[e] = ex2(m[e] - mu[e]);
            moved |= mn != m[e];
            m[e] = mn;
          }
          if (__any_sync(0xffffffffu, moved)) {
#pragma unroll
            for (int e = 0; e < 2; ++e) l[e] *= corr[e];
#pragma unroll
            for (int n = 0; n < HD / 8; ++n)
#pragma unroll
              for (int c = 0; c < 4; ++c) o[n][c] *= corr[c >> 1];
          }
          uint32_t p[4];
#pragma unroll
          for (int n = 0; n < 2; ++n)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
              const float e0 = ex2(fmaf(sc[n][2 * e], sl, -mu[e])), e1 = ex2(fmaf(sc[n][2 * e + 1], sl, -mu[e]));
              l[e] += e0 + e1;
              p[n * 2 + e] = pack_bf16(e0, e1);
            }
#pragma unroll
          for (int dd = 0; dd < HD / 16; ++dd) {
            uint32_t b[4];
            const int c8 = dd * 2 + v_d8;
            ldmatrix4_trans(va + (c8 >> 3) * (kFrKeys * 128) + (((c8 & 7) ^ (v_key & 7)) << 4), b);
            mma16816(o[2 * dd], p, b[0], b[1]);
            mma16816(o[2 * dd + 1], p, b[2], b[3]);
          }
        }
        __syncwarp();
        if (lane == 0) mbar_arrive(&B.empty[slot]);
        if (++slot == Lay::kStages) {
          slot = 0;
          ++use;
        }
      }
      if (!ok) break;
      // ---- the four warps' parts of the item, joined
      if (seg_no > 0 && !warp_all(mbar_wait(&B.merge_empty, (seg_no - 1) & 1))) { ok = false; break; }
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        const int row = gr + 8 * e;
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 1);
        l[e] += __shfl_xor_sync(0xffffffffu, l[e], 2);
        if (row < R) {
          float* po = merge + (warp * kFewRows + row) * HD + t4 * 2;
#pragma unroll
          for (int n = 0; n < HD / 8; ++n) *reinterpret_cast<float2*>(po + n * 8) = make_float2(o[n][2 * e], o[n][2 * e + 1]);
          if (t4 == 0) {
            stat[warp * kFewRows + row] = m[e];
            stat[(4 + warp) * kFewRows + row] = l[e];
          }
        }
      }
      mbar_arrive(&B.merge_full);
      if (!warp_all(mbar_wait(&B.merge_full, seg_no & 1))) { ok = false; break; }
      const bool all = g.k0 == 0 && g.k1 == g.n;
      const bool to_slot = !all || A.keep;
      const int64_t sidx = all ? g.item : 2ll * blockIdx.x + (g.k0 == 0 ? 1 : 0);
      const int stride = all ? sd.item_rows : sd.slot_rows;
      float* const slots = all ? sd.item_slots : sd.slots;
      float* const slot_lse = all ? sd.item_lse : sd.slot_lse;
      const int q4 = A.D / 4;
      for (int u = threadIdx.x; u < R * q4; u += 128) {
        // slots: rows fastest, as they are laid out; the output: elements fastest
        const int row = to_slot ? u % R : u / q4, c4 = to_slot ? u / R : u - row * q4;
        float mx = -INFINITY;
#pragma unroll
        for (int w = 0; w < 4; ++w) mx = max3_nan(mx, mx, stat[w * kFewRows + row]);
        const float base = mx == -INFINITY ? 0.f : mx;
        float den = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
        for (int w = 0; w < 4; ++w) {
          const float f = ex2(stat[w * kFewRows + row] - base);
          const float4 v = *reinterpret_cast<const float4*>(merge + (w * kFewRows + row) * HD + c4 * 4);
          den = fmaf(f, stat[(4 + w) * kFewRows + row], den);
          acc = make_float4(fmaf(f, v.x, acc.x), fmaf(f, v.y, acc.y), fmaf(f, v.z, acc.z), fmaf(f, v.w, acc.w));
        }
        const float inv = mx == -INFINITY ? 0.f : 1.f / den;  // no key: zero
        const float ls = mx == -INFINITY ? -INFINITY : mx + log2f(den);
        acc = make_float4(acc.x * inv, acc.y * inv, acc.z * inv, acc.w * inv);
        if (to_slot) {
          *reinterpret_cast<float4*>(slots + sidx * stride * A.D + (static_cast<int64_t>(c4) * stride + row) * 4) = acc;
          if (c4 == 0) slot_lse[sidx * stride + row] = ls;
        } else {
          const XRow x = fw_row(sd, row);
          *reinterpret_cast<uint2*>(A.out + o_offset(s, g.bi, g.h, x) + c4 * 4) =
              make_uint2(pack_bf16(acc.x, acc.y), pack_bf16(acc.z, acc.w));
          if (A.lse != nullptr && c4 == 0) A.lse[flat_row(s, g.bi, g.h, x)] = ls;
        }
      }
      mbar_arrive(&B.merge_empty);
      ++seg_no;
    }
    if (!ok) atomicExch(&B.abort_flag, 1);
  }
  // launched beside the launch before it: what follows this kernel needs that one's results too
  grid_dep_wait();
}

template <int HD>
int fr_launch(const FwArgs& A, const XMap (&m)[4], int grid, bool behind, cudaStream_t st) {
  using Lay = FrLayout<HD>;
  auto kern = xattn_rows_kernel<HD>;
  static unsigned long long done = 0;  // a bit per device; setting the attribute again is harmless
  int rc = allow_smem(kern, Lay::kSmem, &done, "attention (few rows): set smem");
  if (rc) return rc;
  if (behind) {
    cudaError_t e = launch_pdl(kern, dim3(grid), dim3(kFrThreads), Lay::kSmem, st, m[0].map, m[1].map, m[2].map, m[3].map, A);
    if (e != cudaSuccess) return cuda_status(e, "attention (few rows) launch");
  } else {
    kern<<<grid, kFrThreads, Lay::kSmem, st>>>(m[0].map, m[1].map, m[2].map, m[3].map, A);
    TSB_CHECK_LAUNCH("attention (few rows) launch");
  }
  return debug_sync(st, "attention (few rows)");
}

}  // namespace

int few_rows_grid() { return 2 * sm_count(); }

int few_rows_launch(const FwArgs& args, int grid, bool behind, cudaStream_t st) {
  FwArgs A = args;
  A.item_cost = kFrItemCost;
  XMap m[4];
  for (int j = 0; j < A.sides; ++j) {
    FwSide& S = A.side[j];
    const XSide& x = S.s;
    int rc = make_xmap(&m[2 * j], x.k, A.D, x.klen, x.hkv, x.nb, x.k_t, x.k_h, x.k_b, kFrKeys);
    if (!rc) rc = make_xmap(&m[2 * j + 1], x.v, A.D, x.klen, x.hkv, x.nb, x.v_t, x.v_h, x.v_b, kFrKeys);
    if (rc) return rc;
    S.mul_kh = m[2 * j].mul_h;
    S.mul_kb = m[2 * j].mul_b;
    S.mul_vh = m[2 * j + 1].mul_h;
    S.mul_vb = m[2 * j + 1].mul_b;
  }
  for (int j = 2 * A.sides; j < 4; ++j) m[j] = m[j - 2];
  return A.D <= 64 ? fr_launch<64>(A, m, grid, behind, st) : fr_launch<128>(A, m, grid, behind, st);
}

}  // namespace tsb
