// Tensor-core plumbing of the attention kernels: tensor maps over [B,T,H,D] operands, TMA
// loads of 128-row tiles, tensor-memory moves, and products of 16-bit tiles.
//
// An operand tile is [D/64 blocks][128 rows][64 values] in 128-byte-swizzled rows (the
// K-major layout of tc.cuh).  Read with the head dimension as K it gives A B^T products
// (scores); read MN-major, with its rows as K, it is the right factor of P V, dS K and so on.
// Head sizes below a multiple of 64 are filled with zeros by TMA, as rows beyond T are.
#pragma once

#include <atomic>
#include <cuda.h>

#include "attn_common.cuh"
#include "pipe.cuh"

namespace gdnx {
namespace attn {

constexpr int TM = 128;                 // rows of a tile
constexpr uint32_t BLOCK_BYTES = TM * 128;  // 64 values of every row

GDNX_DEV void tma_load_4d(uint32_t dst, const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t mbar) {
  asm volatile(
      "cp.async.bulk.tensor.4d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5}], "
      "[%6];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(mbar)
      : "memory");
}

// A tensor map and which of its head and batch coordinates count (a broadcast one is 0).
struct TileMap {
  CUtensorMap map;
  int use_h, use_b;
};

// Rows t0..t0+127 of head h into a tile of DB blocks.
template <int DB>
GDNX_DEV void load_rows(uint32_t dst, const TileMap& m, int t0, int64_t h, int64_t b, uint32_t mbar) {
#pragma unroll
  for (int d = 0; d < DB; ++d)
    tma_load_4d(dst + d * BLOCK_BYTES, &m.map, d * 64, m.use_h ? (int)h : 0, t0, m.use_b ? (int)b : 0, mbar);
}

// Instruction descriptor of a 16-bit product with fp32 sums (bf16: format 1, f16: format 0).
__host__ __device__ constexpr uint32_t idesc16(bool bf16, int M, int N, bool a_mn, bool b_mn) {
  return (1u << 4) | ((bf16 ? 1u : 0u) << 7) | ((bf16 ? 1u : 0u) << 10) | ((a_mn ? 1u : 0u) << 15) |
         ((b_mn ? 1u : 0u) << 16) | ((uint32_t)(N >> 3) << 17) | ((uint32_t)(M >> 4) << 24);
}

// A value that all lanes of a converged warp hold alike, in a form that the compiler knows to be
// uniform (what is loaded from memory or found from the thread index it does not).
template <typename T>
GDNX_DEV T uniform(T x) { return __shfl_sync(0xffffffffu, x, 0); }

// One lane of a converged warp.  Products are issued by a whole warp that keeps its state
// uniform, with only the instructions themselves under the elected lane: their operands then
// stay in uniform registers (issued from a divergent thread, each product waits for its
// operands to be moved there, and the issue takes longer than the product runs).
GDNX_DEV bool elect_one() {
  uint32_t ok;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok));
  return ok != 0;
}

// Descriptors are built once and stepped by constants (their address field counts 16-byte units), which
// keeps a product's issue well below its run time.

// D[128 x N] = A B^T over the head dimension: both tiles K-major in shared memory.
template <int DB>
GDNX_DEV void mma_abt(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc) {
  const uint64_t da = tc::smem_desc(a, 16, 1024), db = tc::smem_desc(b, 16, 1024);
#pragma unroll
  for (int k = 0; k < 4 * DB; ++k) {
    const uint32_t at = ((k / 4) * BLOCK_BYTES + (k % 4) * 32) >> 4;
    tc::mma_bf16(d, da + at, db + at, idesc, k > 0);
  }
}

// D[128 x 64 DB] (+)= P X over 16 STEPS keys: P packed 16-bit in tensor memory, X rows of a tile
// read with its rows as K.  `acc`: whether D holds a sum already.
template <int STEPS>
GDNX_DEV void mma_px(uint32_t d, uint32_t p, uint32_t x, uint32_t idesc, bool acc) {
  const uint64_t dx = tc::smem_desc(x, BLOCK_BYTES, 1024);
#pragma unroll
  for (int k = 0; k < STEPS; ++k) tc::mma_bf16_ts(d, p + 8 * k, dx + k * (2048 >> 4), idesc, acc || k > 0);
}

// Bounded wait by a whole warp, which leaves together.
GDNX_DEV bool warp_wait(uint64_t* bar, uint32_t parity, volatile int* abort_flag) {
  return __all_sync(0xffffffffu, pipe::wait_or_abort(bar, parity, abort_flag));
}

// Registers of the executing warpgroup from here on (the block's sum stays within its launch's).
template <int N>
GDNX_DEV void regs_up() { asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N)); }
template <int N>
GDNX_DEV void regs_down() { asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N)); }

template <bool BF16>
GDNX_DEV uint32_t pack2(float lo, float hi) {
  if (BF16) return tc::pack_bf16(lo, hi);
  const __half2 t = __floats2half2_rn(lo, hi);
  return *reinterpret_cast<const uint32_t*>(&t);
}

GDNX_DEV float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}

// 32 lanes x 128 consecutive 32-bit columns of tensor memory (the wait is in the same statement, as in tc.cuh).
GDNX_DEV void tmem_ld128(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x128.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63,"
      "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"
      "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95,"
      "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"
      "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127"
      "}, [%128];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63]),
        "=f"(v[64]), "=f"(v[65]), "=f"(v[66]), "=f"(v[67]), "=f"(v[68]), "=f"(v[69]), "=f"(v[70]), "=f"(v[71]),
        "=f"(v[72]), "=f"(v[73]), "=f"(v[74]), "=f"(v[75]), "=f"(v[76]), "=f"(v[77]), "=f"(v[78]), "=f"(v[79]),
        "=f"(v[80]), "=f"(v[81]), "=f"(v[82]), "=f"(v[83]), "=f"(v[84]), "=f"(v[85]), "=f"(v[86]), "=f"(v[87]),
        "=f"(v[88]), "=f"(v[89]), "=f"(v[90]), "=f"(v[91]), "=f"(v[92]), "=f"(v[93]), "=f"(v[94]), "=f"(v[95]),
        "=f"(v[96]), "=f"(v[97]), "=f"(v[98]), "=f"(v[99]), "=f"(v[100]), "=f"(v[101]), "=f"(v[102]), "=f"(v[103]),
        "=f"(v[104]), "=f"(v[105]), "=f"(v[106]), "=f"(v[107]), "=f"(v[108]), "=f"(v[109]), "=f"(v[110]), "=f"(v[111]),
        "=f"(v[112]), "=f"(v[113]), "=f"(v[114]), "=f"(v[115]), "=f"(v[116]), "=f"(v[117]), "=f"(v[118]), "=f"(v[119]),
        "=f"(v[120]), "=f"(v[121]), "=f"(v[122]), "=f"(v[123]), "=f"(v[124]), "=f"(v[125]), "=f"(v[126]), "=f"(v[127])
      : "r"(taddr)
      : "memory");
}

// 32 lanes x 64 consecutive 32-bit columns of tensor memory (the wait is in the same statement, as in tc.cuh).
GDNX_DEV void tmem_ld64(uint32_t taddr, float* v) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x64.b32 {"
      "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"
      "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,"
      "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"
      "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63"
      "}, [%64];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=f"(v[0]), "=f"(v[1]), "=f"(v[2]), "=f"(v[3]), "=f"(v[4]), "=f"(v[5]), "=f"(v[6]), "=f"(v[7]),
        "=f"(v[8]), "=f"(v[9]), "=f"(v[10]), "=f"(v[11]), "=f"(v[12]), "=f"(v[13]), "=f"(v[14]), "=f"(v[15]),
        "=f"(v[16]), "=f"(v[17]), "=f"(v[18]), "=f"(v[19]), "=f"(v[20]), "=f"(v[21]), "=f"(v[22]), "=f"(v[23]),
        "=f"(v[24]), "=f"(v[25]), "=f"(v[26]), "=f"(v[27]), "=f"(v[28]), "=f"(v[29]), "=f"(v[30]), "=f"(v[31]),
        "=f"(v[32]), "=f"(v[33]), "=f"(v[34]), "=f"(v[35]), "=f"(v[36]), "=f"(v[37]), "=f"(v[38]), "=f"(v[39]),
        "=f"(v[40]), "=f"(v[41]), "=f"(v[42]), "=f"(v[43]), "=f"(v[44]), "=f"(v[45]), "=f"(v[46]), "=f"(v[47]),
        "=f"(v[48]), "=f"(v[49]), "=f"(v[50]), "=f"(v[51]), "=f"(v[52]), "=f"(v[53]), "=f"(v[54]), "=f"(v[55]),
        "=f"(v[56]), "=f"(v[57]), "=f"(v[58]), "=f"(v[59]), "=f"(v[60]), "=f"(v[61]), "=f"(v[62]), "=f"(v[63])
      : "r"(taddr)
      : "memory");
}

// 32 lanes x 32 columns of raw words.
GDNX_DEV void tmem_st32u(uint32_t taddr, const uint32_t (&v)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {"
      "%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16,"
      "%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31,%32"
      "};\n\t"
      "tcgen05.wait::st.sync.aligned;"
      :
      : "r"(taddr),
        "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]), "r"(v[5]), "r"(v[6]), "r"(v[7]),
        "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15]),
        "r"(v[16]), "r"(v[17]), "r"(v[18]), "r"(v[19]), "r"(v[20]), "r"(v[21]), "r"(v[22]), "r"(v[23]),
        "r"(v[24]), "r"(v[25]), "r"(v[26]), "r"(v[27]), "r"(v[28]), "r"(v[29]), "r"(v[30]), "r"(v[31])
      : "memory");
}

GDNX_DEV void tma_store_4d(const CUtensorMap* map, int c0, int c1, int c2, int c3, uint32_t src) {
  asm volatile("cp.async.bulk.tensor.4d.global.shared::cta.tile.bulk_group [%0, {%1, %2, %3, %4}], [%5];" ::"l"(
                   reinterpret_cast<uint64_t>(map)),
               "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(src)
               : "memory");
}

// Bits lo..hi (inclusive, any integers) of the 32-bit word that holds columns 32w..32w+31.
GDNX_DEV uint32_t range_bits(int lo, int hi, int w) {
  lo = max(lo - 32 * w, 0);
  hi = min(hi - 32 * w, 31);
  return lo > hi ? 0u : (0xffffffffu >> (31 - hi)) & (0xffffffffu << lo);
}

// Two fp32 operations in one instruction.
GDNX_DEV float2 fma2(float2 a, float2 b, float2 c) {
  float2 d;
  asm("{\n\t.reg .b64 x, y, z;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\tmov.b64 z, {%6, %7};\n\t"
      "fma.rn.f32x2 x, x, y, z;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y), "f"(c.x), "f"(c.y));
  return d;
}
GDNX_DEV float2 add2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "add.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

GDNX_DEV float2 mul2(float2 a, float2 b) {
  float2 d;
  asm("{\n\t.reg .b64 x, y;\n\tmov.b64 x, {%2, %3};\n\tmov.b64 y, {%4, %5};\n\t"
      "mul.rn.f32x2 x, x, y;\n\tmov.b64 {%0, %1}, x;\n\t}"
      : "=f"(d.x), "=f"(d.y)
      : "f"(a.x), "f"(a.y), "f"(b.x), "f"(b.y));
  return d;
}

// The larger of two values, NaN if either is.
GDNX_DEV float max_nan(float a, float b) {
  float m;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(m) : "f"(a), "f"(b));
  return m;
}

// 2^x of two values on the FMA pipes, for x <= 120; below -125 it stays at 2^-125.  x = n + f with
// |f| <= 1/2 (n by rounding x + 1.5 2^23), 2^f by the polynomial of degree 4 whose relative
// error over the interval is least (2.6e-6, Remez exchange), n added to the exponent.  NaN gives 2^-125 too, or with
// KEEP_NAN NaN, for one more multiplication (n added to its bits would make a number of it).
template <bool KEEP_NAN>
GDNX_DEV float2 ex2_poly(float2 x) {
  constexpr float kRound = 12582912.f;
  x.x = KEEP_NAN ? max_nan(x.x, -125.f) : fmaxf(x.x, -125.f);
  x.y = KEEP_NAN ? max_nan(x.y, -125.f) : fmaxf(x.y, -125.f);
  const float2 r = add2(x, make_float2(kRound, kRound));
  const float2 n = add2(r, make_float2(-kRound, -kRound));
  const float2 f = fma2(n, make_float2(-1.f, -1.f), x);
  float2 p = fma2(f, make_float2(0.009570102207f, 0.009570102207f), make_float2(0.05591785908f, 0.05591785908f));
  p = fma2(p, f, make_float2(0.2402474433f, 0.2402474433f));
  p = fma2(p, f, make_float2(0.6931217909f, 0.6931217909f));
  p = fma2(p, f, make_float2(0.9999992847f, 0.9999992847f));
  if (KEEP_NAN)
    return mul2(p, make_float2(__int_as_float((__float_as_int(r.x) << 23) + 0x3f800000),
                               __int_as_float((__float_as_int(r.y) << 23) + 0x3f800000)));
  p.x = __int_as_float(__float_as_int(p.x) + (__float_as_int(r.x) << 23));
  p.y = __int_as_float(__float_as_int(p.y) + (__float_as_int(r.y) << 23));
  return p;
}

// ------------------------------- host side ----------------------------------
using EncodeTiledFn = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                   const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                   CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

inline EncodeTiledFn encode_fn() {
  static const EncodeTiledFn fn = [] {
    void* f = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &f, cudaEnableDefault, &q) == cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      return reinterpret_cast<EncodeTiledFn>(f);
    cudaGetLastError();
    return EncodeTiledFn(nullptr);
  }();
  return fn;
}

// Whether a kernel may use `smem` bytes of dynamic shared memory on the current device (set on its first launch
// there: `done` has a bit for each).
template <typename F>
bool allow_smem(F kernel, int smem, std::atomic<uint64_t>& done) {
  int dev = 0;
  if (cudaGetDevice(&dev) != cudaSuccess) return false;
  if (dev < 64 && (done.load(std::memory_order_relaxed) >> dev & 1)) return true;
  if (cudaFuncSetAttribute(kernel, cudaFuncAttributeMaxDynamicSharedMemorySize, smem) != cudaSuccess) {
    cudaGetLastError();
    return false;
  }
  if (dev < 64) done.fetch_or(1ull << dev);
  return true;
}

// 4-D map {D, head, token, batch} over a [B,T,H,D] view of 16-bit values, box {64, 1, rows, 1},
// 128-byte swizzle, zeros outside.  False where TMA cannot address the view.
inline bool make_tile_map(const gdnx_view& v, int64_t B, int64_t T, int64_t H, int64_t D, TileMap* m,
                          int rows = TM) {
  if ((v.dtype != GDNX_BF16 && v.dtype != GDNX_F16) || reinterpret_cast<uintptr_t>(v.ptr) % 16 || D % 8) return false;
  const EncodeTiledFn enc = encode_fn();
  if (!enc) return false;
  m->use_h = H > 1 && v.sh != 0;
  m->use_b = B > 1 && v.sb != 0;
  const cuuint64_t dims[4] = {(cuuint64_t)D, (cuuint64_t)(m->use_h ? H : 1), (cuuint64_t)T,
                              (cuuint64_t)(m->use_b ? B : 1)};
  // dimensions of one element may carry any stride: give them a valid one
  const cuuint64_t row = (cuuint64_t)((D + 7) / 8 * 16);
  const cuuint64_t strides[3] = {m->use_h ? (cuuint64_t)v.sh * 2 : row, T > 1 ? (cuuint64_t)v.st * 2 : row,
                                 m->use_b ? (cuuint64_t)v.sb * 2 : row};
  for (int i = 0; i < 3; ++i)
    if (strides[i] == 0 || strides[i] % 16 || strides[i] >= (1ull << 40)) return false;
  const cuuint32_t box[4] = {64, 1, (cuuint32_t)rows, 1};
  const cuuint32_t es[4] = {1, 1, 1, 1};
  return enc(&m->map, v.dtype == GDNX_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 4,
             const_cast<void*>(v.ptr), dims, strides, box, es, CU_TENSOR_MAP_INTERLEAVE_NONE,
             CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
             CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

}  // namespace attn
}  // namespace gdnx
