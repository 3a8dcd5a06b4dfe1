// Shared by the tensor-core dense attention kernels: 4-D tensor maps over
// strided (batch, head, token, head_dim) operands, TMA loads through them, and
// the rule for which calls the tensor cores take.
#pragma once

#include "tc_common.cuh"
#include "xattn.cuh"

namespace tsb {
namespace {

// 4-D tiled load of the box at element coordinates (d, token, head, batch).
__device__ __forceinline__ void tma_load_4d(void* dst, const CUtensorMap* map, int d, int t, int h, int b,
                                            uint64_t* bar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];\n" ::"r"(smem_u32(dst)),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(d), "r"(t), "r"(h), "r"(b), "r"(smem_u32(bar))
      : "memory");
}

// A bf16 operand as a tensor map with boxes of 64 elements x `box_rows` tokens. Elements past D and
// tokens past len read as zeros, so any D up to the tile's width and any length load whole tiles. A head
// or batch dimension of one entry, or of stride 0 (expanded), is not part of the map: its coordinate is
// multiplied by mul = 0.
struct XMap {
  CUtensorMap map;
  int mul_h, mul_b;
};

inline int make_xmap(XMap* m, const void* base, int64_t D, int64_t len, int64_t heads, int64_t batch, int64_t s_t,
                     int64_t s_h, int64_t s_b, uint32_t box_rows) {
  static PFN_cuTensorMapEncodeTiled_v12000 encode = nullptr;
  if (!encode) {
    void* fn = nullptr;
    cudaDriverEntryPointQueryResult q;
    cudaError_t e = cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &fn, cudaEnableDefault, &q);
    if (e != cudaSuccess || q != cudaDriverEntryPointSuccess || !fn)
      return fail(TRNSPARSE_ERR_CUDA, "cuTensorMapEncodeTiled unavailable");
    encode = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(fn);
  }
  m->mul_h = heads > 1 && s_h != 0;
  m->mul_b = batch > 1 && s_b != 0;
  const int64_t row = len > 1 && s_t != 0 ? s_t * 2 : ((D * 2 + 15) & ~15ll);
  if (len > 1 && s_t == 0) return fail(TRNSPARSE_ERR_ALIGN, "tensor map: token stride 0");
  cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)len, m->mul_h ? (cuuint64_t)heads : 1,
                        m->mul_b ? (cuuint64_t)batch : 1};
  cuuint64_t strides[3] = {(cuuint64_t)row, m->mul_h ? (cuuint64_t)s_h * 2 : (cuuint64_t)row,
                           m->mul_b ? (cuuint64_t)s_b * 2 : (cuuint64_t)row};
  cuuint32_t box[4] = {64, box_rows, 1, 1}, estr[4] = {1, 1, 1, 1};
  CUresult r = encode(&m->map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                      CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  if (r != CUDA_SUCCESS) return fail(TRNSPARSE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return TRNSPARSE_OK;
}

// tcgen05.wait::ld that also orders the loaded registers: nothing that uses them moves above it.
__device__ __forceinline__ void tmem_wait_ld32(uint32_t (&r)[32]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15]),
                 "+r"(r[16]), "+r"(r[17]), "+r"(r[18]), "+r"(r[19]), "+r"(r[20]), "+r"(r[21]), "+r"(r[22]),
                 "+r"(r[23]), "+r"(r[24]), "+r"(r[25]), "+r"(r[26]), "+r"(r[27]), "+r"(r[28]), "+r"(r[29]),
                 "+r"(r[30]), "+r"(r[31])
               :
               : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Strides (batch, head, token) the tensor maps and 16-byte accesses take: multiples of 8 elements, not
// negative, below 2^39 elements; a dimension of one entry has no stride to look at.
inline bool strides_ok(const int64_t* s, int64_t nb, int64_t nh, int64_t nt, bool keys) {
  const int64_t n[3] = {nb, nh, nt};
  for (int i = 0; i < 3; ++i) {
    if (n[i] <= 1) continue;
    if (s[i] % 8 || s[i] < 0 || s[i] >= (1ll << 38)) return false;
    if (keys && i == 2 && s[i] == 0) return false;
  }
  return true;
}

}  // namespace
}  // namespace tsb
