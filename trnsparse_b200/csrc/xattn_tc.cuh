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
  auto run = [&] {
    return encode(&m->map, CU_TENSOR_MAP_DATA_TYPE_BFLOAT16, 4, const_cast<void*>(base), dims, strides, box, estr,
                  CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                  CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
  };
  CUresult r = run();
  if (r == CUDA_ERROR_INVALID_CONTEXT) {
    // a driver call, and this host thread (autograd's, for one) has made no runtime call yet
    int dev = 0;
    cudaError_t e = cudaGetDevice(&dev);
    if (e == cudaSuccess) e = cudaSetDevice(dev);
    if (e != cudaSuccess) return cuda_status(e, "tensor map: make the device's context current");
    r = run();
  }
  if (r != CUDA_SUCCESS) return fail(TRNSPARSE_ERR_CUDA, "cuTensorMapEncodeTiled failed (%d)", (int)r);
  return TRNSPARSE_OK;
}

__device__ __forceinline__ void tmem_ld16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];\n"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr)
      : "memory");
}

__device__ __forceinline__ void tmem_ld4(uint32_t taddr, uint32_t (&r)[4]) {
  asm volatile("tcgen05.ld.sync.aligned.32x32b.x4.b32 {%0,%1,%2,%3}, [%4];\n"
               : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3])
               : "r"(taddr)
               : "memory");
}
__device__ __forceinline__ void tmem_st4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1,%2,%3,%4};\n" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}

// The MMA warp stays converged: all lanes wait and vote, one elected lane issues. The addresses of its MMAs are
// then uniform values, which the compiler keeps in uniform registers; one lane walking the loop alone moves them
// there for every MMA (2340 clocks against 2080 for 32 MMAs of 64 clocks with their waits).
__device__ __forceinline__ bool elect_one() {
  uint32_t p;
  asm volatile("{\n.reg .pred P;\nelect.sync _|P, 0xffffffff;\nselp.u32 %0, 1, 0, P;\n}\n" : "=r"(p));
  return p != 0;
}
__device__ __forceinline__ bool warp_all(bool b) { return __all_sync(0xffffffffu, b) != 0; }
// A shared-memory descriptor's low word holds the address (16-byte units), which moves; the high word stays.
__device__ __forceinline__ uint64_t desc_at(uint64_t desc, uint32_t lo) {
  uint64_t d;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(d) : "r"(lo), "r"(static_cast<uint32_t>(desc >> 32)));
  return d;
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

__device__ __forceinline__ void tmem_wait_ld16(uint32_t (&r)[16]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n"
               : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]), "+r"(r[4]), "+r"(r[5]), "+r"(r[6]), "+r"(r[7]),
                 "+r"(r[8]), "+r"(r[9]), "+r"(r[10]), "+r"(r[11]), "+r"(r[12]), "+r"(r[13]), "+r"(r[14]), "+r"(r[15])
               :
               : "memory");
}
__device__ __forceinline__ void tmem_wait_ld4(uint32_t (&r)[4]) {
  asm volatile("tcgen05.wait::ld.sync.aligned;\n" : "+r"(r[0]), "+r"(r[1]), "+r"(r[2]), "+r"(r[3]) : : "memory");
}

__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;\n" : "=f"(y) : "f"(x));
  return y;
}

// Pairs of floats in one 64-bit register: the packed fp32 instructions of sm_100 do two elements an issue slot.
__device__ __forceinline__ uint64_t pack2(float a, float b) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};\n" : "=l"(r) : "f"(a), "f"(b));
  return r;
}
__device__ __forceinline__ void unpack2(uint64_t v, float& a, float& b) {
  asm("mov.b64 {%0, %1}, %2;\n" : "=f"(a), "=f"(b) : "l"(v));
}
__device__ __forceinline__ uint64_t fma2(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;\n" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t add2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
// The larger of three, NaN if any is.
__device__ __forceinline__ float max3_nan(float a, float b, float c) {
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;\n" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}

__device__ __forceinline__ uint64_t mul2(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("mul.rn.f32x2 %0, %1, %2;\n" : "=l"(r) : "l"(a), "l"(b));
  return r;
}

// 2^x of two elements on the FMA pipe, x <= 120 or so: x = n + f with n the nearest integer (adding 1.5 2^23
// leaves it in the low mantissa bits), 2^f on [-1/2, 1/2] by a degree-4 minimax polynomial (relative error
// 2.6e-6, fitted by weighted least squares for this file; P is rounded to bf16, half a step up to 2^-8, afterwards, the
// row's sum takes it as it is), and n added
// to the exponent. x below -126 gives 0, NaN gives NaN.
__device__ __forceinline__ void exp2_poly2(uint64_t x2, float& a, float& b) {
  float xa, xb, la, lb;
  unpack2(x2, xa, xb);
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;\n" : "=f"(la) : "f"(xa));  // -127
  asm("max.NaN.f32 %0, %1, 0fC2FE0000;\n" : "=f"(lb) : "f"(xb));
  const uint64_t x = pack2(la, lb);
  const float magic = 12582912.f;
  const uint64_t t = add2(x, pack2(magic, magic));
  const uint64_t n = add2(t, pack2(-magic, -magic));
  const uint64_t f = fma2(n, pack2(-1.f, -1.f), x);
  uint64_t p = fma2(f, pack2(0x1.3997d6p-7f, 0x1.3997d6p-7f), pack2(0x1.ca1440p-5f, 0x1.ca1440p-5f));
  p = fma2(f, p, pack2(0x1.ec06dap-3f, 0x1.ec06dap-3f));
  p = fma2(f, p, pack2(0x1.62e0dcp-1f, 0x1.62e0dcp-1f));
  p = fma2(f, p, pack2(0x1.ffffe8p-1f, 0x1.ffffe8p-1f));
  float ta, tb, pa, pb, za, zb;
  unpack2(t, ta, tb);
  unpack2(p, pa, pb);
  unpack2(mul2(x, pack2(0.f, 0.f)), za, zb);
  a = xa >= -126.f ? __uint_as_float((__float_as_uint(ta) << 23) + __float_as_uint(pa)) : za;
  b = xb >= -126.f ? __uint_as_float((__float_as_uint(tb) << 23) + __float_as_uint(pb)) : zb;
}

__device__ __forceinline__ uint4 shfl_xor4(uint4 v, int m) {
  return make_uint4(__shfl_xor_sync(0xffffffffu, v.x, m), __shfl_xor_sync(0xffffffffu, v.y, m),
                    __shfl_xor_sync(0xffffffffu, v.z, m), __shfl_xor_sync(0xffffffffu, v.w, m));
}
// Lane i of four holds q[0..3]; afterwards q[k] is what lane k held as q[i].
__device__ __forceinline__ void quad_transpose(uint4 (&q)[4], int i) {
#pragma unroll
  for (int m = 1; m <= 2; m <<= 1) {
    const bool up = i & m;
#pragma unroll
    for (int a = 0; a < 4; ++a) {
      if (a & m) continue;
      // swap q[a | m] of the lower lane with q[a] of the upper lane
      const uint4 give = up ? q[a] : q[a | m];
      const uint4 got = shfl_xor4(give, m);
      if (up) q[a] = got;
      else q[a | m] = got;
    }
  }
}

// Asynchronous 16-byte copy global -> shared, zeros when !in (then nothing is read).
__device__ __forceinline__ void cp_async16(void* dst, const void* src, bool in) {
  asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;\n" ::"r"(smem_u32(dst)), "l"(src), "r"(in ? 16 : 0)
               : "memory");
}
__device__ __forceinline__ void cp_async_wait_all() { asm volatile("cp.async.wait_all;\n" ::: "memory"); }

// Dynamic shared memory above the default, asked for once per device (`done`: a bit each).
template <typename K>
int allow_smem(K kern, int bytes, unsigned long long* done, const char* what) {
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess) return cuda_status(e, what);
  const unsigned long long bit = dev < 64 ? 1ull << dev : 0;
  if (__atomic_load_n(done, __ATOMIC_ACQUIRE) & bit) return TRNSPARSE_OK;
  e = cudaFuncSetAttribute(kern, cudaFuncAttributeMaxDynamicSharedMemorySize, bytes);
  if (e != cudaSuccess) return cuda_status(e, what);
  __atomic_fetch_or(done, bit, __ATOMIC_RELEASE);
  return TRNSPARSE_OK;
}

// Strides (batch, head, token) the tensor maps and 16-byte accesses take: multiples of 8 elements, not
// negative, below 2^38 elements; a dimension of one entry has no stride to look at.
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
