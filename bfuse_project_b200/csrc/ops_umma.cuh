// Tensor-core bodies for dense / batch_matmul on sm_100a: TMA loads into a shared-memory ring,
// tcgen05.mma issued by one thread with the fp32 accumulator in tensor memory, tcgen05.ld back to
// registers for the epilogue (bias, causal mask, bf16 down-convert).  They compute the operators
// of the reference's dense / batch_matmul kernels (NT layout, scripts/configure_kernels.py:14-26)
// with tf32 or bf16 operands instead of CUDA-core fp32 FMAs.
//
// BlockDim = (192, 1, 1): warps 0-3 read the accumulator (one TMEM lane quadrant each), warp 4 is
// the TMA producer, warp 5 allocates tensor memory and issues the MMAs.  One 128 x BN output tile
// belongs to `split` CTAs that each multiply a slice of K: GridDim = (split * ceil(M/128),
// ceil(N/BN), batch).  A tcgen05.mma of 128 x N x 32 bytes takes about the same time for N = 32
// as for N = 256, so narrow problems are fast only with wide tiles whose K loop is spread over
// several SMs.  With split > 1 the CTAs of a tile form a thread-block cluster and every CTA owns a
// share of the tile's 128-byte column chunks: after one cluster barrier (all MMAs of the tile are
// done, so every ring is free) each CTA pushes its fp32 partial sums of a chunk straight from
// tensor memory into the owner's shared memory with st.async, the owner waits on an mbarrier that
// counts the delivered bytes, sums the k-slices in order (deterministic) and stores the chunk.
// The ring depth comes from the shared-memory size the caller registered.
//
// Every wait on an mbarrier is bounded: when it gives up it writes a code to the status word and
// the body falls through to its normal exit (barrier, TMEM free) instead of spinning.
#pragma once

#include <cuda.h>
#include <float.h>

#include <type_traits>

#include "tile.h"

namespace bfuse {

constexpr int kUmmaThreads = 192;
constexpr int kUmmaBM = 128;
constexpr int kUmmaRowBytes = 128;                      // one swizzle-128B row of K per stage
constexpr int kUmmaABytes = kUmmaBM * kUmmaRowBytes;    // 16 KB of A per stage
constexpr int kUmmaHeaderBytes = 2048;                  // barriers, tmem pointer, bias slice; keeps tiles 1 KB aligned
constexpr int kUmmaMaxStages = 8;

enum UmmaStatus : int {
  UMMA_WAIT_EMPTY_TIMEOUT = 0x101,
  UMMA_WAIT_FULL_TIMEOUT = 0x102,
  UMMA_WAIT_ACC_TIMEOUT = 0x103,
  UMMA_WAIT_PEERS_TIMEOUT = 0x104,
  UMMA_WAIT_OTHER_TIMEOUT = 0x105,
};

// bm: rows of A (and of the output tile) per CTA, 128 or 256
__host__ __device__ constexpr int umma_stage_bytes(int bn, int bm = kUmmaBM) { return (bm + bn) * kUmmaRowBytes; }
__host__ __device__ constexpr int umma_smem_bytes(int bn, int stages, int bm = kUmmaBM) {
  return kUmmaHeaderBytes + stages * umma_stage_bytes(bn, bm);
}

// ---- PTX wrappers ----------------------------------------------------------------------------
__device__ __forceinline__ uint32_t smem_u32(const void *p) { return (uint32_t)__cvta_generic_to_shared(p); }

__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_inval(uint32_t bar) {
  asm volatile("mbarrier.inval.shared::cta.b64 [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ float ld_shared_f32(uint32_t addr) {
  float v;
  asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ uint64_t global_ns() {
  uint64_t t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Wait for phase `parity` of an mbarrier, for at most ~1 s.  Returns false after reporting.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity, int *status, int code) {
  uint64_t t0 = 0;
  for (uint32_t it = 0;; ++it) {
    uint32_t ok;
    asm volatile(
        "{\n\t.reg .pred p;\n\t"
        "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
        "selp.b32 %0, 1, 0, p;\n\t}"
        : "=r"(ok)
        : "r"(bar), "r"(parity)
        : "memory");
    if (ok) return true;
    if ((it & 1023u) == 1023u) {
      // once any wait of the launch has given up, the others follow at once: a failed launch then ends
      // after about one second in all, not one second per CTA (negative: refused data, and nothing to give up for)
      if (status && *reinterpret_cast<volatile int *>(status) > 0) return false;
      const uint64_t now = global_ns();
      if (t0 == 0) t0 = now;
      if (now - t0 > 1000000000ull) {
        if (status) atomicExch(status, code);
        return false;
      }
    }
  }
}

__device__ __forceinline__ void tma_load_3d(uint32_t dst, const CUtensorMap *map, uint32_t bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];"
      ::"r"(dst), "l"(map), "r"(bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void tmem_alloc(uint32_t dst_smem, uint32_t cols) {
  asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(dst_smem), "r"(cols) : "memory");
}
// Lets co-resident CTAs allocate while this one still holds its columns.  A CTA that will allocate
// again (a persistent CTA, once per tile) must NOT call this: allocating after it is illegal.
__device__ __forceinline__ void tmem_relinquish() {
  asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;" ::: "memory");
}
__device__ __forceinline__ void tmem_dealloc(uint32_t taddr, uint32_t cols) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(taddr), "r"(cols) : "memory");
}
__device__ __forceinline__ void tc_fence_before() { asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void tc_fence_after() { asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory"); }
__device__ __forceinline__ void umma_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar) : "memory");
}
// One thread of a warp, chosen by the hardware; every lane of the (converged) warp must call it.
__device__ __forceinline__ bool elect_one() {
  uint32_t pred;
  asm volatile("{\n\t.reg .pred p;\n\telect.sync _|p, 0xffffffff;\n\tselp.b32 %0, 1, 0, p;\n\t}" : "=r"(pred));
  return pred != 0;
}
// High word of the shared-memory matrix descriptor of a K-major, 128B-swizzled operand tile whose
// rows are 128 bytes: 8-row groups 1024 bytes apart (stride byte offset, bits 32-45), version 1
// (bit 46), layout SWIZZLE_128B (bits 61-63).  The low word is (address >> 4) | 1 << 16.
constexpr uint32_t kUmmaDescHi = (1024u >> 4) | (1u << 14) | (2u << 29);
template <int KIND>  // 0: tf32, 1: bf16; a_lo / b_lo: low descriptor words
__device__ __forceinline__ void umma_ss(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  if (KIND == 0) {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::tf32 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(accumulate)
        : "memory");
  } else {
    asm volatile(
        "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
        "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(accumulate)
        : "memory");
  }
}
// The same MMA with the A operand in tensor memory: 128 lanes (rows of A) x one 32-bit column per tf32
// value of k, 8 columns per instruction; B from shared memory as above.
__device__ __forceinline__ void umma_ts_tf32(uint32_t d_tmem, uint32_t a_tmem, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::1.kind::tf32 [%0], [%1], db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_tmem), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// Registers -> tensor memory, 32 lanes x 32 consecutive 32-bit columns: thread i of the warp writes
// lane i (a warp reaches the 32 lanes of its quadrant, warp index mod 4).  Asynchronous: complete
// after tmem_st_wait().
__device__ __forceinline__ void tmem_st_32x32(uint32_t taddr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], "
      "{%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};" ::"r"(taddr),
      "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]), "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]), "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]), "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// the same, 4 columns
__device__ __forceinline__ void tmem_st_32x4(uint32_t taddr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("tcgen05.st.sync.aligned.32x32b.x4.b32 [%0], {%1, %2, %3, %4};" ::"r"(taddr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}
__device__ __forceinline__ void tmem_st_wait() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }
// 32 lanes x 16 consecutive fp32 columns of the accumulator: thread i of the warp gets lane i.
// Asynchronous: the registers are valid after tmem_ld_wait().
__device__ __forceinline__ void tmem_ld_32x16(uint32_t taddr, uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x16.b32 "
      "{%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15}, [%16];"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]), "=r"(r[8]),
        "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15])
      : "r"(taddr));
}
__device__ __forceinline__ void tmem_ld_wait() { asm volatile("tcgen05.wait::ld.sync.aligned;" ::: "memory"); }

__device__ __forceinline__ void cluster_sync_all() {
  asm volatile("barrier.cluster.arrive.release.aligned;\n\tbarrier.cluster.wait.acquire.aligned;" ::: "memory");
}
// address of `local` (a shared::cta address of this CTA) in the shared memory of cluster rank `rank`
__device__ __forceinline__ uint32_t peer_smem(uint32_t local, uint32_t rank) {
  uint32_t r;
  asm volatile("mapa.shared::cluster.u32 %0, %1, %2;" : "=r"(r) : "r"(local), "r"(rank));
  return r;
}
// 16-byte store into a peer's shared memory that also credits 16 bytes to the peer's mbarrier
__device__ __forceinline__ void st_async_u4(uint32_t peer_addr, uint32_t peer_bar, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.async.weak.shared::cluster.mbarrier::complete_tx::bytes.v4.b32 [%0], {%2, %3, %4, %5}, [%1];" ::"r"(peer_addr),
               "r"(peer_bar), "r"(a), "r"(b), "r"(c), "r"(d)
               : "memory");
}
__device__ __forceinline__ float4 ld_shared_f4(uint32_t addr) {
  float4 v;
  asm volatile("ld.shared.v4.f32 {%0,%1,%2,%3}, [%4];" : "=f"(v.x), "=f"(v.y), "=f"(v.z), "=f"(v.w) : "r"(addr) : "memory");
  return v;
}
__device__ __forceinline__ void st_shared_u4(uint32_t addr, uint32_t a, uint32_t b, uint32_t c, uint32_t d) {
  asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(addr), "r"(a), "r"(b), "r"(c), "r"(d) : "memory");
}

// Instruction descriptor: fp32 accumulate, both operands K-major, M = 128, N = bn.
__host__ __device__ constexpr uint32_t umma_idesc(int kind, int bn) {
  return (1u << 4) | ((kind == 0 ? 2u : 1u) << 7) | ((kind == 0 ? 2u : 1u) << 10) | ((uint32_t)(bn >> 3) << 17) |
         ((uint32_t)(kUmmaBM >> 4) << 24);
}

struct GemmUmmaParams {
  alignas(64) CUtensorMap map_a;    // {K, M, batch}, box {128 B of K, BM, 1}, 128B swizzle
  alignas(64) CUtensorMap map_b;    // {K, N, batch}, box {128 B of K, BN, 1}, 128B swizzle
  alignas(64) CUtensorMap map_out;  // {N, M, batch}, box {128 B of N, 32, 1}, 128B swizzle (stores)
  const float *bias;                // [N] or nullptr
  void *out;                        // [batch, M, N] fp32 (tf32 kind) or bf16 (bf16 kind)
  int batch, M, N, K;
  int causal;
  int stages;
  int bn;            // output-tile width: 32, 64, 128 or 256 (also the TMEM columns allocated)
  int split;         // CTAs (k-slices) per output tile = cluster width; 1: no split
  int kb_per_slice;  // K blocks (of 128 bytes per row) per k-slice
  int bm;            // output-tile height: 128, or 256 (two MMAs per k-step share the W tile; split == 1 only)
  long long *timeline;  // diagnostic: when non-null, CTA 0 records globaltimer marks here (see UmmaMark)
};

// The product with more in its epilogue: out = act(A W^T + bias) + other, or * other.  `other` has the output's shape, so
// its tiles come and go in the same boxes.
struct GemmActParams : GemmUmmaParams {
  alignas(64) CUtensorMap map_other;   // as map_out, for loads
  const uint16_t *other;
  int has_other;                       // 0: no residual / gate
  int mul;                             // 1: act(...) * other, 0: act(...) + other
  int act;                             // BFUSE_ACT_*
};

enum GemmAct : int { ACT_NONE = 0, ACT_RELU = 1, ACT_GELU = 2, ACT_GELU_TANH = 3, ACT_SILU = 4 };

// The activations, two values at a time and without branches: an epilogue has one warp per scheduler, and erff's two ways cost
// 137 clocks a value where this takes about 20.
__device__ __forceinline__ float rcp_approx(float x) {   // 1 ulp; 0 from 2^126 on
  float y;
  asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float exp2_approx(float x) {   // 2 ulp
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float d;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
  return d;
}
// x / (1 + 2^-z), of y = -8 - z: the sum is taken 2^-8 smaller, so that its reciprocal leaves the normal range only where the
// result does (SiLU: below -92; with the sum as it is at -87, which lost values of up to 5e-37)
__device__ __forceinline__ float2 over_one_plus_exp2(float2 x, float2 y) {
  constexpr float k = 1.f / 256.f;
  return mul2(mul2(x, make_float2(k, k)), make_float2(rcp_approx(k + exp2_approx(y.x)), rcp_approx(k + exp2_approx(y.y))));
}
template <int ACT>
__device__ __forceinline__ float2 activate(float2 x) {
  const float2 m8 = make_float2(-8.f, -8.f);
  if (ACT == ACT_RELU) return make_float2(x.x > 0.f ? x.x : (x.x != x.x ? x.x : 0.f), x.y > 0.f ? x.y : (x.y != x.y ? x.y : 0.f));
  if (ACT == ACT_SILU) return over_one_plus_exp2(x, fma2(x, make_float2(-1.4426950408889634f, -1.4426950408889634f), m8));
  if (ACT == ACT_GELU_TANH) {   // 1/2 (1 + tanh u) = 1 / (1 + e^-2u), u = sqrt(2 / pi) (x + 0.044715 x^3)
    constexpr float a = -2.302208198f, b = -0.10294324f;   // -2 sqrt(2 / pi) log2(e), and 0.044715 times that
    return over_one_plus_exp2(x, fma2(x, fma2(mul2(x, x), make_float2(b, b), make_float2(a, a)), m8));
  }
  if (ACT == ACT_GELU) {
    // x Phi(x) = max(x, 0) - a Phi(-a), a = |x|.  Phi(-a) = e^(-a^2 / 2) R(a) with R(a) = erfcx(a / sqrt(2)) / 2 = t (c1 + ... + c8 t^7),
    // t = 1 / (1 + 0.305 a): fitted for this kernel by reweighted least squares to the largest RELATIVE error over 0 <= a <= 14,
    // 9.4e-8.  The exponent's roundings add a few 2^-24 of it: 2^-20 of Phi for a < 2, 2^-17 at 13; below that Phi leaves the
    // normal range.  (a: at most 16, where Phi is 0, so that nothing is infinite.)
    const float2 a = make_float2(fminf(fabsf(x.x), 16.f), fminf(fabsf(x.y), 16.f));
    const float2 d = fma2(a, make_float2(0.305f, 0.305f), make_float2(1.f, 1.f)), t = make_float2(rcp_approx(d.x), rcp_approx(d.y));
    const float2 s = mul2(mul2(a, a), make_float2(-0.5f * 1.4426950408889634f, -0.5f * 1.4426950408889634f));
    float2 q = fma2(t, make_float2(0.0366991801f, 0.0366991801f), make_float2(-0.152988269f, -0.152988269f));
    q = fma2(t, q, make_float2(0.185716826f, 0.185716826f));
    q = fma2(t, q, make_float2(-0.0379767573f, -0.0379767573f));
    q = fma2(t, q, make_float2(0.121021641f, 0.121021641f));
    q = fma2(t, q, make_float2(0.103420877f, 0.103420877f));
    q = fma2(t, q, make_float2(0.122466815f, 0.122466815f));
    q = fma2(t, q, make_float2(0.121639733f, 0.121639733f));
    q = mul2(mul2(q, t), make_float2(exp2_approx(s.x), exp2_approx(s.y)));   // Phi(-a)
    return fma2(make_float2(-a.x, -a.y), q, make_float2(max_nan(x.x, 0.f), max_nan(x.y, 0.f)));
  }
  return x;
}
template <int ACT, int N>
__device__ __forceinline__ void activate_each(float (&v)[N]) {
#pragma unroll
  for (int j = 0; j < N; j += 2) {
    const float2 y = activate<ACT>(make_float2(v[j], v[j + 1]));
    v[j] = y.x, v[j + 1] = y.y;
  }
}
template <int N>
__device__ __forceinline__ void activate_all(int act, float (&v)[N]) {
  if (act == ACT_RELU) activate_each<ACT_RELU>(v);
  else if (act == ACT_GELU) activate_each<ACT_GELU>(v);
  else if (act == ACT_GELU_TANH) activate_each<ACT_GELU_TANH>(v);
  else if (act == ACT_SILU) activate_each<ACT_SILU>(v);
}

// marks of the diagnostic timeline (nanoseconds on the global timer), written by virtual block 0
enum UmmaMark : int {
  MARK_START = 0, MARK_SETUP_DONE, MARK_FIRST_LOAD_ISSUED, MARK_LAST_LOAD_ISSUED, MARK_FIRST_FULL, MARK_LAST_MMA_ISSUED,
  MARK_ACC_READY, MARK_PARTIAL_WRITTEN, MARK_CLUSTER_SYNC1, MARK_REDUCED, MARK_CLUSTER_SYNC2, MARK_END, MARK_COUNT
};

constexpr int kUmmaStagingBytes = 4 * 4096;  // one 32-row x 128-byte store buffer per epilogue warp
// bytes of the ring that the epilogue needs: for split GEMMs the receive area -- per owned 128-byte
// output chunk one fp32 partial (128 rows x chunk columns) from every k-slice -- plus the store buffers
__host__ __device__ constexpr int umma_recv_bytes(int bn, int split, int elem) {
  return split > 1 ? ((bn * elem / 128 + split - 1) / split) * split * (128 / elem) * kUmmaBM * 4 : 0;
}
__host__ __device__ constexpr int umma_epilogue_bytes(int bn, int split, int elem) {
  return umma_recv_bytes(bn, split, elem) + kUmmaStagingBytes;
}

__device__ __forceinline__ void tma_store_3d(const CUtensorMap *map, uint32_t src, int c0, int c1, int c2) {
  asm volatile("cp.async.bulk.tensor.3d.global.shared::cta.bulk_group [%0, {%2, %3, %4}], [%1];" ::"l"(map), "r"(src),
               "r"(c0), "r"(c1), "r"(c2)
               : "memory");
}
__device__ __forceinline__ void tma_store_commit() { asm volatile("cp.async.bulk.commit_group;" ::: "memory"); }
template <int PENDING>
__device__ __forceinline__ void tma_store_wait_read() {
  asm volatile("cp.async.bulk.wait_group.read %0;" ::"n"(PENDING) : "memory");
}
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// The epilogue of one warp: 32 rows x 128-byte chunks go through 128B-swizzled staging buffers and
// leave with one TMA store per chunk (full lines, clipped at the tensor's edges by the hardware).
// Chunks are staged in groups: one proxy fence, one warp barrier and one bulk group per GROUP of
// chunks, because each of those costs a few hundred nanoseconds of latency that a per-chunk
// sequence would pay serially.  With a buffer for every chunk of the warp nothing is ever waited
// for before the end; otherwise the buffers form two half-groups that alternate (one being filled
// while the other's stores read it).
template <int KIND>
struct ChunkWriter {
  const CUtensorMap *map_out;
  int M, N, causal;  // output rows / columns (clipping, mask) of the tensor the map describes
  uint32_t buf0;   // staging buffers of this warp (nbuf x 4096 bytes)
  int nbuf, lane, issued;  // issued: bulk groups committed so far
  int m_base, bz;  // first output row of this warp's 32 rows, batch index
  int n_tile0;     // first output column of the tile
  int nb_step;     // columns between consecutive chunks this warp writes
  int group;       // chunks per bulk group: nbuf (single group) or nbuf / 2
  // Output rows that are not 16-byte multiples cannot be described to the TMA: the staged chunks
  // then leave with 4-byte stores, 32 lanes writing 32 consecutive elements of one row (fp32 only).
  float *direct = nullptr;  // element (0, 0) of this batch entry's output matrix, or nullptr: TMA stores
  int slot = 0, pending = 0, first_nb = 0;

  __device__ __forceinline__ uint32_t begin_chunk() {
    if (!direct && pending == 0 && issued * group >= nbuf) {
      // the half-group about to be overwritten must have been read by its stores
      if (lane == 0) {
        if (group < nbuf) tma_store_wait_read<1>();
        else tma_store_wait_read<0>();
      }
      __syncwarp();
    }
    return buf0 + (uint32_t)slot * 4096u;
  }
  // 16 finished fp32 values of this lane's row: columns [nb + sub*16, +16) of the chunk at column nb;
  // bias_tile: this tile's slice of the bias vector in shared memory (zeros without a bias)
  __device__ __forceinline__ void put16(uint32_t buf, int sub, int nb, float (&v)[16], const float *bias_tile) {
    const int col0 = nb + sub * 16, m = m_base + lane;
    if (bias_tile) {
      // all four loads first: the shared-memory stores below are ordered asm statements, and a load
      // placed between them would wait out its latency there
      const float4 *b4 = reinterpret_cast<const float4 *>(bias_tile + (col0 - n_tile0));
      const float4 ba = b4[0], bb = b4[1], bc = b4[2], bd = b4[3];
      v[0] += ba.x, v[1] += ba.y, v[2] += ba.z, v[3] += ba.w;
      v[4] += bb.x, v[5] += bb.y, v[6] += bb.z, v[7] += bb.w;
      v[8] += bc.x, v[9] += bc.y, v[10] += bc.z, v[11] += bc.w;
      v[12] += bd.x, v[13] += bd.y, v[14] += bd.z, v[15] += bd.w;
    }
    if (causal && col0 + 15 > m) {
#pragma unroll
      for (int j = 0; j < 16; ++j)
        if (col0 + j > m) v[j] = -FLT_MAX;
    }
    const uint32_t row = buf + (uint32_t)lane * 128u;
    if (KIND == 0) {
#pragma unroll
      for (int j = 0; j < 4; ++j)
        st_shared_u4(row + (uint32_t)(((sub * 4 + j) ^ (lane & 7)) * 16), __float_as_uint(v[4 * j]), __float_as_uint(v[4 * j + 1]),
                     __float_as_uint(v[4 * j + 2]), __float_as_uint(v[4 * j + 3]));
    } else {
#pragma unroll
      for (int j = 0; j < 2; ++j)
        st_shared_u4(row + (uint32_t)(((sub * 2 + j) ^ (lane & 7)) * 16), f2_to_bf16x2(v[8 * j], v[8 * j + 1]),
                     f2_to_bf16x2(v[8 * j + 2], v[8 * j + 3]), f2_to_bf16x2(v[8 * j + 4], v[8 * j + 5]),
                     f2_to_bf16x2(v[8 * j + 6], v[8 * j + 7]));
    }
  }
  __device__ __forceinline__ void end_chunk(uint32_t buf, int nb) {
    (void)buf;
    if (pending == 0) first_nb = nb;
    ++pending;
    if (++slot == nbuf) slot = 0;
    if (pending == group) flush();
  }
  // hands the staged chunks to the TMA: every lane fences its own writes, lane 0 issues the stores
  __device__ __forceinline__ void flush() {
    if (pending == 0) return;
    if (direct) {
      __syncwarp();
      const int first_slot = (slot == 0 ? nbuf : slot) - pending;
      for (int i = 0; i < pending; ++i) {
        const int col = first_nb + i * nb_step + lane;
        const uint32_t b = buf0 + (uint32_t)(first_slot + i) * 4096u;
        if (col < N) {
#pragma unroll 4
          for (int row = 0; row < 32; ++row) {
            float v;
            asm volatile("ld.shared.f32 %0, [%1];" : "=f"(v) : "r"(b + (uint32_t)(row * 128 + (((lane >> 2) ^ (row & 7)) << 4) + ((lane & 3) << 2))) : "memory");
            if (m_base + row < M) direct[(size_t)(m_base + row) * N + col] = v;
          }
        }
      }
      __syncwarp();  // the buffers may be overwritten
      ++issued;
      pending = 0;
      return;
    }
    fence_async_smem();
    __syncwarp();
    if (lane == 0) {
      const int first_slot = (slot == 0 ? nbuf : slot) - pending;
      for (int i = 0; i < pending; ++i) {
        const int nb = first_nb + i * nb_step;
        if (nb < N && m_base < M) tma_store_3d(map_out, buf0 + (uint32_t)(first_slot + i) * 4096u, nb, m_base, bz);
      }
      tma_store_commit();
    }
    ++issued;
    pending = 0;
  }
  __device__ __forceinline__ void finish() {
    flush();
    if (!direct && lane == 0) tma_store_wait_read<0>();
    __syncwarp();
  }
};

// Few rows of A (tokens being decoded): multiplied the other way round, out^T = W A^T.  A stage then holds 128 rows of W and
// only `bm` (16 or 32) of A instead of 128, so that eight stages are 128 KB of weights on their way per SM; the accumulator has
// output columns in its lanes and rows in its columns, and what the k-slices exchange is 128 x bm.
__host__ __device__ constexpr bool umma_few_rows(int bm) { return bm < kUmmaBM; }
__host__ __device__ constexpr int umma_few_recv_bytes(int bm, int split) { return split > 1 ? kUmmaBM * bm * 4 : 0; }

constexpr int kActBarOffset = 256;   // in the window's header: a barrier per epilogue warp and staging buffer
constexpr int kActBars = 4;          // staging buffers of a warp at most (staging_plan: 64 bf16 columns a chunk, 256 a tile)

// The writer of GemmUmma<KIND, true>: `other` is loaded into the very staging buffer that its chunk of the output leaves
// from, so it costs no shared memory; the loads of all buffers are under way before the first chunk is worked on, and
// the tile's lines were asked into L2 while the MMAs ran (512 x 4096 x 4096 with a residual: 24 us, as the product without one).
struct ActWriter : ChunkWriter<1> {
  const GemmActParams *pa;
  uint32_t bar0;                  // this warp's barriers, one per staging buffer
  int *status;
  int col0, m0, per_half, total;  // first chunk's column and row; chunks of 128 rows; chunks in all
  int next = 0, loaded = 0;       // chunks begun; chunks whose load has been issued

  __device__ __forceinline__ void load(int q, int half_end) {   // lane 0: chunk q into its buffer, unless it is another half's
    if (q >= total || q >= half_end) return;
    const uint32_t s = (uint32_t)(q % nbuf), bar = bar0 + 8 * s;
    mbar_expect_tx(bar, 4096u);
    tma_load_3d(buf0 + s * 4096u, &pa->map_other, bar, col0 + (q % per_half) * nb_step, m0 + (q / per_half) * kUmmaBM, bz);
  }
  __device__ __forceinline__ void prefetch() const {   // one lane
    if (!pa->has_other) return;
    for (int q = 0; q < total; ++q)
      asm volatile("cp.async.bulk.prefetch.tensor.3d.L2.global.tile [%0, {%1, %2, %3}];" ::"l"(&pa->map_other),
                   "r"(col0 + (q % per_half) * nb_step), "r"(m0 + (q / per_half) * kUmmaBM), "r"(bz)
                   : "memory");
  }
  // the ring is idle: every buffer starts with its first chunk
  __device__ __forceinline__ void start() {
    if (!pa->has_other) return;
    loaded = min(nbuf, min(per_half, total));
    if (lane == 0)
      for (int q = 0; q < loaded; ++q) load(q, per_half);
    __syncwarp();
  }
  __device__ __forceinline__ uint32_t begin_chunk() {
    const uint32_t buf = ChunkWriter<1>::begin_chunk();
    if (pa->has_other) {
      if (next >= loaded) {   // a buffer's later use: the whole group that is free now
        const int half_end = (next / per_half + 1) * per_half, end = min(next + group, min(half_end, total));
        if (lane == 0)
          for (int q = next; q < end; ++q) load(q, half_end);
        loaded = end;
        __syncwarp();
      }
      mbar_wait(bar0 + 8 * (uint32_t)(next % nbuf), (next / nbuf) & 1, status, UMMA_WAIT_OTHER_TIMEOUT);
      __syncwarp();
    }
    ++next;
    return buf;
  }
  __device__ __forceinline__ void put16(uint32_t buf, int sub, int nb, float (&v)[16], const float *bias_tile) {
    const float4 *b4 = reinterpret_cast<const float4 *>(bias_tile + (nb + sub * 16 - n_tile0));
    const float4 ba = b4[0], bb = b4[1], bc = b4[2], bd = b4[3];
    v[0] += ba.x, v[1] += ba.y, v[2] += ba.z, v[3] += ba.w;
    v[4] += bb.x, v[5] += bb.y, v[6] += bb.z, v[7] += bb.w;
    v[8] += bc.x, v[9] += bc.y, v[10] += bc.z, v[11] += bc.w;
    v[12] += bd.x, v[13] += bd.y, v[14] += bd.z, v[15] += bd.w;
    activate_all(pa->act, v);
    const uint32_t row = buf + (uint32_t)lane * 128u;
    if (pa->has_other) {
#pragma unroll
      for (int j = 0; j < 2; ++j) {
        const float4 o = ld_shared_f4(row + (uint32_t)(((sub * 2 + j) ^ (lane & 7)) * 16));
        const float u[4] = {o.x, o.y, o.z, o.w};
#pragma unroll
        for (int i = 0; i < 4; ++i) {
          const float2 f = bf16x2_to_f2(__float_as_uint(u[i]));
          float &a = v[8 * j + 2 * i], &b = v[8 * j + 2 * i + 1];
          a = pa->mul ? a * f.x : a + f.x;
          b = pa->mul ? b * f.y : b + f.y;
        }
      }
    }
#pragma unroll
    for (int j = 0; j < 2; ++j)
      st_shared_u4(row + (uint32_t)(((sub * 2 + j) ^ (lane & 7)) * 16), f2_to_bf16x2(v[8 * j], v[8 * j + 1]),
                   f2_to_bf16x2(v[8 * j + 2], v[8 * j + 3]), f2_to_bf16x2(v[8 * j + 4], v[8 * j + 5]),
                   f2_to_bf16x2(v[8 * j + 6], v[8 * j + 7]));
  }
  // no load may be in flight when the window is handed on (a wait before the last chunk gave up)
  __device__ __forceinline__ void drain() {
    for (; next < loaded; ++next) mbar_wait(bar0 + 8 * (uint32_t)(next % nbuf), (next / nbuf) & 1, status, UMMA_WAIT_OTHER_TIMEOUT);
    __syncwarp();
  }
};

// staging buffers (per epilogue warp) and chunks per bulk group for `total` chunks when `free_bufs`
// buffers fit: a buffer per chunk in groups of two (the stores of one pair run while the next pair
// is staged, and nothing is reused), else two alternating half-groups of up to 4, else one buffer
__device__ __forceinline__ void staging_plan(int free_bufs, int total, int &nbuf, int &group) {
  if (free_bufs >= total) nbuf = total, group = min(2, total);
  else if (free_bufs >= 2) group = min(4, free_bufs / 2), nbuf = 2 * group;
  else nbuf = 1, group = 1;
}


// The cross-CTA reduction of a tile whose K range is split over the `split` CTAs of a cluster
// (k-slice = rank in the cluster); called by every thread of the operator after the MMAs.  The
// tile's 128-byte output chunks are dealt to the k-slices round-robin; `tiles` (the ring, idle by
// now) receives, per owned chunk, one fp32 partial from every k-slice, laid out
// [16-column group][quarter][row][4 floats].  After one cluster barrier (every k-slice has finished
// its MMAs, so every ring is free) each CTA pushes its partials straight from tensor memory into
// the owners' shared memory; an owner waits on its mbarrier, which counts the delivered bytes,
// sums the k-slices in order (deterministic) and stores the chunk through `w`.
template <int KIND, class Writer>
__device__ __forceinline__ void umma_split_reduce(const TileCtx &c, int BN, int split, int kslice, uint32_t tiles, uint32_t recv_bar,
                                                  uint32_t tmem_row, bool acc_ok, Writer &w, int n0,
                                                  const float *bias_tile, long long *tl) {
  constexpr int kElem = KIND == 0 ? 4 : 2, kOutCols = 128 / kElem, kSub = kOutCols / 16;
  constexpr uint32_t kChunkPartial = (uint32_t)kOutCols * kUmmaBM * 4;
  const int warp = c.tid >> 5, lane = c.tid & 31, quad = (threadIdx.x >> 5) & 3;
  const int chunks = BN / kOutCols, max_owned = (chunks + split - 1) / split;
  auto mark = [&](int what, bool who) {
    if (tl && who) tl[what] = (long long)global_ns();
  };
  cluster_sync_all();
  mark(MARK_CLUSTER_SYNC1, c.tid == 0);
  if (warp >= 4) return;
  const int row = quad * 32 + lane;
  if (acc_ok) {
#pragma unroll 1
    for (int cc = 0; cc < BN / 16; cc += 2) {
      uint32_t r0[16], r1[16];
      tmem_ld_32x16(tmem_row + cc * 16, r0);
      tmem_ld_32x16(tmem_row + (cc + 1) * 16, r1);
      tmem_ld_wait();
      const int ch = cc / kSub, owner = ch % split;
      const uint32_t slot = tiles + (uint32_t)((ch / split) * split + kslice) * kChunkPartial;
      const uint32_t dst0 = peer_smem(slot + (uint32_t)((((cc % kSub) * 4) * kUmmaBM + row) * 16), (uint32_t)owner);
      const uint32_t dst1 = dst0 + 4u * kUmmaBM * 16u;
      const uint32_t bar = peer_smem(recv_bar, (uint32_t)owner);
#pragma unroll
      for (int j = 0; j < 4; ++j) {
        st_async_u4(dst0 + (uint32_t)(j * kUmmaBM * 16), bar, r0[4 * j], r0[4 * j + 1], r0[4 * j + 2], r0[4 * j + 3]);
        st_async_u4(dst1 + (uint32_t)(j * kUmmaBM * 16), bar, r1[4 * j], r1[4 * j + 1], r1[4 * j + 2], r1[4 * j + 3]);
      }
    }
  }
  mark(MARK_PARTIAL_WRITTEN, c.tid == 0);
  // all partials of the chunks this CTA owns have landed (a CTA that owns none expected no bytes)
  int owned = 0;
  for (int ch = kslice; ch < chunks; ch += split) ++owned;
  const bool got = owned == 0 || mbar_wait(recv_bar, 0, c.status, UMMA_WAIT_PEERS_TIMEOUT);
  mark(MARK_CLUSTER_SYNC2, c.tid == 0);
  if (got) {
#pragma unroll 1
    for (int li = 0; li < max_owned; ++li) {
      const int ch = li * split + kslice;
      if (ch >= chunks) break;
      const uint32_t buf = w.begin_chunk();
#pragma unroll 1
      for (int sub = 0; sub < kSub; ++sub) {
        float acc[16];
#pragma unroll
        for (int j = 0; j < 16; ++j) acc[j] = 0.f;
#pragma unroll 1
        for (int peer = 0; peer < split; ++peer) {  // k-slice order: the sum is deterministic
          const uint32_t src = tiles + (uint32_t)(li * split + peer) * kChunkPartial + (uint32_t)(((sub * 4) * kUmmaBM + row) * 16);
#pragma unroll
          for (int j = 0; j < 4; ++j) {
            const float4 v = ld_shared_f4(src + (uint32_t)(j * kUmmaBM * 16));
            acc[4 * j] += v.x, acc[4 * j + 1] += v.y, acc[4 * j + 2] += v.z, acc[4 * j + 3] += v.w;
          }
        }
        w.put16(buf, sub, n0 + ch * kOutCols, acc, bias_tile);
      }
      w.end_chunk(buf, n0 + ch * kOutCols);
    }
    w.finish();
  }
  mark(MARK_REDUCED, c.tid == 0);
}

// ACT: with activation and a residual or gate in the epilogue (bf16)
template <int KIND, bool ACT = false>
struct GemmUmma {
  static_assert(!ACT || KIND == 1, "the activating epilogue is built for bf16");
  using Params = typename std::conditional<ACT, GemmActParams, GemmUmmaParams>::type;
  using Writer = typename std::conditional<ACT, ActWriter, ChunkWriter<KIND>>::type;
  static constexpr int kMaxThreads = kUmmaThreads;
  static constexpr int kMinBlocks = 1;
  static constexpr bool kMemoryBound = false;
  static constexpr bool kUsesTmem = true;   // allocates tensor memory (see fused_block_kernel)
  static constexpr int kElem = KIND == 0 ? 4 : 2;
  static constexpr int kBK = kUmmaRowBytes / kElem;  // K elements per stage
  static constexpr int kOutCols = 128 / kElem;       // output columns per 128-byte store chunk
  static constexpr int kSub = kOutCols / 16;         // 16-column accumulator reads per chunk

  // The MMA issue loop of one k-slice, run by a single thread.  TALL: 256-row tile -- rows 128..255
  // of A (16 KB further on in the stage) against the same W tile into a second accumulator BN
  // columns on.  A separate instantiation keeps the common loop free of the extra branch and of a
  // run-time W offset: it is a chain of dependent instructions whose length sets the MMA rate of
  // narrow tiles.  Returns false when a wait gave up.
  template <bool TALL>
  __device__ __forceinline__ static bool issue_mmas(const TileCtx &c, uint32_t tiles, int stage_bytes, int stages, int num_kb,
                                                    uint32_t full0, uint32_t empty0, uint32_t tmem_acc, uint32_t idesc, int bn,
                                                    long long *tl) {
    // low descriptor word of stage 0; a stage is stage_bytes / 16 further on
    const uint32_t lo0 = ((tiles >> 4) & 0x3fffu) | (1u << 16), stage16 = (uint32_t)stage_bytes >> 4;
    constexpr uint32_t b_off = (uint32_t)(TALL ? 2 : 1) * (kUmmaABytes >> 4);
    uint32_t s = 0, ph = 0, lo = lo0, accumulate = 0;
    for (int kb = 0; kb < num_kb; ++kb) {
      if (!mbar_wait(full0 + 8 * s, ph, c.status, UMMA_WAIT_FULL_TIMEOUT)) return false;
      tc_fence_after();
      if (kb == 0 && tl) tl[MARK_FIRST_FULL] = (long long)global_ns();
#pragma unroll
      for (int j = 0; j < 4; ++j) {  // 4 x 32 bytes of K per stage; +2 = 32 bytes in descriptor units
        umma_ss<KIND>(tmem_acc, lo + 2 * j, lo + b_off + 2 * j, idesc, accumulate);
        if (TALL) umma_ss<KIND>(tmem_acc + (uint32_t)bn, lo + (kUmmaABytes >> 4) + 2 * j, lo + b_off + 2 * j, idesc, accumulate);
        accumulate = 1;
      }
      umma_commit(empty0 + 8 * s);  // frees the stage once these MMAs have read it
      if (++s == (uint32_t)stages) s = 0, ph ^= 1, lo = lo0;
      else lo += stage16;
    }
    return true;
  }

  // The tile of few rows: split (1, 2, 4 or 8) CTAs of a cluster, each a slice of K.  Every rank pushes its sums to the rank that
  // owns the output column, into memory kept for that, so no one waits for the others' rings.
  __device__ __forceinline__ static void run_few(const Params &p, const TileCtx &c) {
    const int warp = c.tid >> 5, lane = c.tid & 31, quad = (threadIdx.x >> 5) & 3, at = quad * 32 + lane;   // at: output column of the tile
    const int BM = p.bm, split = p.split, stages = p.stages, stage_bytes = umma_stage_bytes(kUmmaBM, BM);
    const int kslice = c.block_x() % split, m0 = c.block_x() / split * BM, n0 = c.block_y() * kUmmaBM, bz = c.block_z();
    const uint32_t full0 = smem_u32(c.smem), empty0 = full0 + 8 * kUmmaMaxStages, acc_bar = empty0 + 8 * kUmmaMaxStages, recv_bar = acc_bar + 8;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(c.smem + 8 * (2 * kUmmaMaxStages + 2));
    const uint32_t tiles = full0 + kUmmaHeaderBytes, recv = tiles + (uint32_t)(stages * stage_bytes);
    const int cols = BM < 32 ? 32 : BM;
    if (warp == 5 && !c.tmem_given) {
      tmem_alloc(smem_u32(tmem_slot), cols);
      if (!c.persistent) tmem_relinquish();
    }
    const int total_kb = (p.K + kBK - 1) / kBK, kb0 = kslice * p.kb_per_slice, num_kb = min(p.kb_per_slice, total_kb - kb0), npre = min(stages, num_kb);
    auto load = [&](int kb, uint32_t s) {
      const uint32_t dst = tiles + s * stage_bytes, bar = full0 + 8 * s;
      mbar_expect_tx(bar, (uint32_t)stage_bytes);
      tma_load_3d(dst + BM * kUmmaRowBytes, &p.map_b, bar, (kb0 + kb) * kBK, n0, bz);
      tma_load_3d(dst, &p.map_a, bar, (kb0 + kb) * kBK, m0, bz);
    };
    if (warp == 4) {
      if (lane < stages) {
        mbar_init(full0 + 8 * lane, 1);
        mbar_init(empty0 + 8 * lane, 1);
      }
      if (lane == 0) {
        mbar_init(acc_bar, 1);
        mbar_init(recv_bar, 1);
      }
      if (lane < 2) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &p.map_a : &p.map_b) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      __syncwarp();
      c.dependency_wait();
      if (elect_one()) {
        if (split > 1) mbar_expect_tx(recv_bar, (uint32_t)umma_few_recv_bytes(BM, split));
        for (int kb = 0; kb < npre; ++kb) load(kb, (uint32_t)kb);
      }
      __syncwarp();
    } else {
      c.dependency_wait();
    }
    tc_fence_before();
    c.sync();
    tc_fence_after();
    if (split > 1) asm volatile("barrier.cluster.arrive.release.aligned;" ::: "memory");   // this CTA's barriers are up: its peers may push
    const uint32_t tmem = c.tmem_given ? c.tmem_base : *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    const int per = kUmmaBM / split;   // output columns a rank owns
    bool ok = true;
    if (warp == 4) {
      if (elect_one()) {
        uint32_t s = 0, ph = 0;
        for (int kb = npre; kb < num_kb; ++kb) {
          if (!mbar_wait(empty0 + 8 * s, ph, c.status, UMMA_WAIT_EMPTY_TIMEOUT)) break;
          load(kb, s);
          if (++s == (uint32_t)stages) s = 0, ph ^= 1;
        }
      }
      __syncwarp();
    } else if (warp == 5) {
      if (elect_one()) {
        const uint32_t idesc = umma_idesc(KIND, BM), lo0 = ((tiles >> 4) & 0x3fffu) | (1u << 16), w_off = (uint32_t)(BM * kUmmaRowBytes) >> 4;
        uint32_t s = 0, ph = 0, lo = lo0;
        for (int kb = 0; kb < num_kb && ok; ++kb) {
          ok = mbar_wait(full0 + 8 * s, ph, c.status, UMMA_WAIT_FULL_TIMEOUT);
          if (!ok) break;
          tc_fence_after();
#pragma unroll
          for (int j = 0; j < 4; ++j) umma_ss<KIND>(tmem, lo + w_off + 2 * j, lo + 2 * j, idesc, kb > 0 || j > 0);
          umma_commit(empty0 + 8 * s);
          if (++s == (uint32_t)stages) s = 0, ph ^= 1, lo = lo0;
          else lo += (uint32_t)stage_bytes >> 4;
        }
        umma_commit(acc_bar);
        // (as in run(): no release may be in flight when the barriers go)
        for (int kb = max(0, num_kb - stages); kb < num_kb && ok; ++kb)
          ok = mbar_wait(empty0 + 8 * (kb % stages), (kb / stages) & 1, c.status, UMMA_WAIT_EMPTY_TIMEOUT);
      }
      __syncwarp();
    }
    // R sums of output column n, rows m, m + step ...: the loads of `other` first, then one after the other
    const size_t batch_at = (size_t)bz * p.M * p.N;
    auto finish = [&](auto &v, int m, int step, int n, float bias) {
      constexpr int R = sizeof(v) / sizeof(v[0]);
      const size_t i0 = batch_at + (size_t)m * p.N + n, next = (size_t)step * p.N;
      float o[R];
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (p.has_other && m + j * step < p.M) o[j] = __uint_as_float((uint32_t)__ldcg(p.other + i0 + j * next) << 16);
#pragma unroll
      for (int j = 0; j < R; ++j) v[j] += bias;
      activate_all(p.act, v);
#pragma unroll
      for (int j = 0; j < R; ++j)
        if (m + j * step < p.M) {
          if (p.has_other) v[j] = p.mul ? v[j] * o[j] : v[j] + o[j];
          reinterpret_cast<__nv_bfloat16 *>(p.out)[i0 + j * next] = __float2bfloat16_rn(v[j]);
        }
    };
    auto ask_other = [&](int m, int n) {
      if (p.has_other && m < p.M && n < p.N) prefetch_l2(p.other + batch_at + (size_t)m * p.N + n);
    };
    if (warp < 4) {
      const int n = n0 + (split > 1 ? kslice * per + at % per : at), m_first = m0 + (split > 1 ? at / per : 0), m_step = split > 1 ? split : 1;
      const float bias = p.bias && n < p.N ? __ldg(p.bias + n) : 0.f;
      if ((at & 31) == 0 || split > 1)
        for (int m = m_first; m < m0 + BM; m += m_step) ask_other(m, n);   // (one lane a line; with k-slices a warp's lanes are in several rows)
      ok = __all_sync(0xffffffffu, mbar_wait(acc_bar, 0, c.status, UMMA_WAIT_ACC_TIMEOUT));
      tc_fence_after();
      const uint32_t trow = tmem + ((uint32_t)(quad * 32) << 16);
      if (split == 1) {
#pragma unroll 1
        for (int mb = 0; mb < BM && m0 + mb < p.M && ok; mb += 16) {
          uint32_t r[16];
          tmem_ld_32x16(trow + mb, r);
          tmem_ld_wait();
          float v[16];
#pragma unroll
          for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r[j]);
          if (n < p.N) finish(v, m0 + mb, 1, n, bias);
        }
      } else {
        asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
        const int owner = at / per;
        const uint32_t dst = peer_smem(recv + (uint32_t)((kslice * per + at - owner * per) * BM) * 4, owner), bar = peer_smem(recv_bar, owner);
#pragma unroll 1
        for (int mb = 0; mb < BM; mb += 16) {
          uint32_t r[16];
          tmem_ld_32x16(trow + mb, r);
          tmem_ld_wait();
#pragma unroll
          for (int j = 0; j < 4; ++j) st_async_u4(dst + 4 * mb + 16 * j, bar, r[4 * j], r[4 * j + 1], r[4 * j + 2], r[4 * j + 3]);
        }
        ok = __all_sync(0xffffffffu, mbar_wait(recv_bar, 0, c.status, UMMA_WAIT_PEERS_TIMEOUT)) && ok;
        // (BM >= 16 and split <= 8: at least two rows a thread)
        for (int m = m_first; m < min(m0 + BM, p.M) && ok && n < p.N; m += 2 * split) {
          float v[2] = {0.f, 0.f};
          for (int r = 0; r < split; ++r) {   // k-slice order
            const uint32_t src = recv + (uint32_t)((r * per + at % per) * BM + m - m0) * 4;
            v[0] += ld_shared_f32(src), v[1] += ld_shared_f32(src + 4 * split);
          }
          finish(v, m, split, n, bias);
        }
      }
    } else if (split > 1) {
      asm volatile("barrier.cluster.wait.acquire.aligned;" ::: "memory");
    }
    __syncwarp();
    tc_fence_before();
    c.sync();
    if (warp == 5 && !c.tmem_given) tmem_dealloc(tmem, cols);
    if (c.persistent && c.tid < stages) {
      mbar_inval(full0 + 8 * c.tid);
      mbar_inval(empty0 + 8 * c.tid);
      if (c.tid == 0) {
        mbar_inval(acc_bar);
        mbar_inval(recv_bar);
      }
    }
  }
  __device__ __forceinline__ static void run(const Params &p, const TileCtx &c) {
    if constexpr (ACT) {
      if (umma_few_rows(p.bm)) return run_few(p, c);
    }
    const int warp = c.tid >> 5, lane = c.tid & 31;
    const int quad = (threadIdx.x >> 5) & 3;  // hardware warp w may only touch TMEM lanes [32 * (w % 4), +32)
    const int BN = p.bn, BM = p.bm, halves = BM / kUmmaBM, kABytes = BM * kUmmaRowBytes, kStageBytes = umma_stage_bytes(BN, BM);
    const uint32_t idesc = umma_idesc(KIND, BN);
    const int split = p.split, kslice = c.block_x() % split;
    // M tiles vary fastest: the (usually few) CTAs that share a W tile are launched next to each
    // other, so the tile is fetched from HBM once and the others hit L2
    const int m0 = (c.block_x() / split) * BM, n0 = c.block_y() * BN, bz = c.block_z();
    const int stages = p.stages;
    const int chunks = BN / kOutCols;

    // operator window: [0,1024) barriers + tmem pointer, then `stages` x (A tile, B tile); once the
    // MMAs are done the ring holds the partial tile (split GEMMs) and the store buffers
    uint64_t *bars = reinterpret_cast<uint64_t *>(c.smem);
    const uint32_t full0 = smem_u32(bars), empty0 = full0 + 8 * kUmmaMaxStages, acc_bar = empty0 + 8 * kUmmaMaxStages;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(c.smem + 8 * (2 * kUmmaMaxStages + 2));
    // Tensor memory first: the SM starts its next CTA of this kernel only when this one has given up
    // its permit to allocate, so every instruction before that delays a co-resident CTA.  A tile
    // entirely above the diagonal of a causal product needs no accumulator.
    const bool masked_tile = !ACT && p.causal && n0 > m0 + BM - 1;
    if (warp == 5) {
      if (!c.tmem_given) {   // (a persistent CTA of the work queue holds its columns already)
        if (!masked_tile) tmem_alloc(smem_u32(tmem_slot), BN * halves);
        if (!c.persistent) tmem_relinquish();
      }
    }
    const uint32_t tiles = smem_u32(c.smem) + kUmmaHeaderBytes;
    const uint32_t recv_bar = acc_bar + 8;                                  // counts partial sums delivered by peers
    float *bias_tile = reinterpret_cast<float *>(c.smem + 1024);            // BN floats
    const int max_owned = (chunks + split - 1) / split;                     // store chunks a k-slice finishes
    constexpr uint32_t kChunkPartial = (uint32_t)kOutCols * kUmmaBM * 4;    // fp32 partial of one chunk from one k-slice
    const uint32_t staging = tiles + (uint32_t)umma_recv_bytes(BN, split, kElem);
    // store buffers per epilogue warp, as many as the idle ring has room for (see staging_plan)
    const int free_bufs = (stages * kStageBytes - (int)(staging - tiles)) / kUmmaStagingBytes;
    int nbuf, group;
    staging_plan(free_bufs, max_owned, nbuf, group);
    Writer w = Writer{ChunkWriter<KIND>{&p.map_out, p.M, p.N, p.causal, staging + (uint32_t)(quad * nbuf) * 4096u, nbuf, lane, 0, m0 + quad * 32, bz, n0,
                                        split * kOutCols, group}};
    if constexpr (ACT) {
      w.pa = &p;
      w.bar0 = full0 + kActBarOffset + 8 * kActBars * quad;
      w.status = c.status;
      w.col0 = n0 + (split > 1 ? kslice * kOutCols : 0);
      w.m0 = m0 + quad * 32;
      w.per_half = split > 1 ? max(0, (chunks - kslice + split - 1) / split) : chunks;
      w.total = w.per_half * halves;
    }
    long long *const tl = (p.timeline && c.vblock == 0) ? p.timeline : nullptr;
    auto mark = [&](int what, bool who) {
      if (tl && who) tl[what] = (long long)global_ns();
    };
    mark(MARK_START, c.tid == 0);

    if (masked_tile) {
      c.dependency_wait();
      // tile entirely above the diagonal (for every k-slice of it): only the mask value to write;
      // k-slice 0 fills one buffer once and stores it to every chunk
      if (warp < 4 && kslice == 0) {
        const uint32_t buf = w.begin_chunk();
        const uint32_t mask = KIND == 0 ? __float_as_uint(-FLT_MAX) : f2_to_bf16x2(-FLT_MAX, -FLT_MAX);
#pragma unroll
        for (int j = 0; j < 8; ++j) st_shared_u4(buf + (uint32_t)lane * 128u + j * 16, mask, mask, mask, mask);
        fence_async_smem();
        __syncwarp();
        if (lane == 0) {
          for (int h = 0; h < halves; ++h) {
            const int mb = w.m_base + h * kUmmaBM;
            for (int ch = 0; ch < chunks && mb < p.M; ++ch)
              if (n0 + ch * kOutCols < p.N) tma_store_3d(&p.map_out, buf, n0 + ch * kOutCols, mb, bz);
          }
          tma_store_commit();
        }
        w.finish();
      }
      return;
    }

    const int total_kb = (p.K + kBK - 1) / kBK;
    const int kb0 = kslice * p.kb_per_slice;                 // first K block of this k-slice
    const int num_kb = min(p.kb_per_slice, total_kb - kb0);  // K blocks this CTA multiplies (>= 1)

    // The producer warp sets the barriers up itself and starts the first ring pass (every slot is
    // free, nothing to wait for) before the CTA-wide barrier, so the first operands are already on
    // their way from HBM while warp 5 allocates tensor memory.
    const int npre = min(stages, num_kb);
    if (warp == 4) {
      if (lane < stages) {
        mbar_init(full0 + 8 * lane, 1);
        mbar_init(empty0 + 8 * lane, 1);
      }
      if (lane == 0) {
        mbar_init(acc_bar, 1);
        mbar_init(recv_bar, 1);
      }
      if (ACT && lane < 4 * kActBars) mbar_init(full0 + kActBarOffset + 8 * lane, 1);
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      __syncwarp();
      if (lane == 0) {
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.map_a) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.map_b) : "memory");
        asm volatile("prefetch.tensormap [%0];" ::"l"(&p.map_out) : "memory");
        if (split > 1) {
          // bytes this CTA will receive: one partial per owned chunk from every k-slice (itself included)
          int owned = 0;
          for (int ch = kslice; ch < chunks; ch += split) ++owned;
          mbar_expect_tx(recv_bar, (uint32_t)owned * (uint32_t)split * kChunkPartial);
        }
      }
      c.dependency_wait();   // all of the above ran while the previous kernel drained; the loads below read its output
      if (elect_one()) {
        for (int kb = 0; kb < npre; ++kb) {
          const uint32_t dst = tiles + kb * kStageBytes, bar = full0 + 8 * kb;
          mbar_expect_tx(bar, kStageBytes);
          tma_load_3d(dst, &p.map_a, bar, (kb0 + kb) * kBK, m0, bz);
          tma_load_3d(dst + kABytes, &p.map_b, bar, (kb0 + kb) * kBK, n0, bz);
          if (kb == 0) mark(MARK_FIRST_LOAD_ISSUED, true);
        }
      }
      __syncwarp();
    } else {
      c.dependency_wait();
    }
    tc_fence_before();
    c.sync();
    tc_fence_after();
    const uint32_t tmem_acc = c.tmem_given ? c.tmem_base : *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    const uint32_t tmem_row = tmem_acc + ((uint32_t)(quad * 32) << 16);
    mark(MARK_SETUP_DONE, c.tid == 0);

    // The producer and the MMA issuer are ONE elected thread each (elect.sync, so the compiler knows
    // the branch is taken by a single thread and keeps descriptors in uniform registers).  Their
    // loops carry the ring slot, its phase and the low descriptor word incrementally: the issue
    // loop is a chain of dependent instructions on one thread, and every instruction saved in it is
    // time the tensor pipe does not idle (4 MMAs of N <= 128 execute faster than a careless loop
    // iteration issues them).  The other lanes wait at the __syncwarp below.
    bool acc_ok = true;
    if (warp == 4) {
      if (elect_one()) {
        // second and later ring passes (the first was issued before the barrier): slot 0 again
        uint32_t s = 0, ph = 0, dst = tiles, bar = full0;
        int kcoord = (kb0 + npre) * kBK;
        for (int kb = npre; kb < num_kb; ++kb) {
          if (!mbar_wait(empty0 + 8 * s, ph, c.status, UMMA_WAIT_EMPTY_TIMEOUT)) break;
          mbar_expect_tx(bar, kStageBytes);
          tma_load_3d(dst, &p.map_a, bar, kcoord, m0, bz);
          tma_load_3d(dst + kABytes, &p.map_b, bar, kcoord, n0, bz);
          kcoord += kBK;
          if (++s == (uint32_t)stages) s = 0, ph ^= 1, dst = tiles, bar = full0;
          else dst += kStageBytes, bar += 8;
        }
        mark(MARK_LAST_LOAD_ISSUED, true);
      }
      __syncwarp();
    } else if (warp == 5) {
      if (elect_one()) {
        bool ok = halves == 2 ? issue_mmas<true>(c, tiles, kStageBytes, stages, num_kb, full0, empty0, tmem_acc, idesc, BN, tl)
                              : issue_mmas<false>(c, tiles, kStageBytes, stages, num_kb, full0, empty0, tmem_acc, idesc, BN, tl);
        umma_commit(acc_bar);  // accumulator complete (also arrives if the loop bailed out)
        mark(MARK_LAST_MMA_ISSUED, true);
        // The stage-release arrivals of the last ring pass are asynchronous and nobody consumes them;
        // wait for them here so that none is still in flight when the barriers are invalidated and
        // the shared memory is handed to the next tile or the next CTA.
        for (int kb = max(0, num_kb - stages); kb < num_kb && ok; ++kb)
          ok = mbar_wait(empty0 + 8 * (kb % stages), (kb / stages) & 1, c.status, UMMA_WAIT_EMPTY_TIMEOUT);
      }
      __syncwarp();
    } else {
      // the epilogue warps are idle during the main loop: they fetch the tile's bias slice meanwhile
      // (only they read it, after their own named-barrier-free hand-off below)
      for (int i = c.tid; i < BN; i += 128) bias_tile[i] = (p.bias && n0 + i < p.N) ? __ldg(p.bias + n0 + i) : 0.f;
      if constexpr (ACT) {
        if (lane == 0) w.prefetch();
      }
      asm volatile("bar.sync %0, 128;" ::"r"(c.bar_id + 8) : "memory");  // the four epilogue warps only (ids 9 / 10)
      acc_ok = mbar_wait(acc_bar, 0, c.status, UMMA_WAIT_ACC_TIMEOUT);
      tc_fence_after();
      mark(MARK_ACC_READY, c.tid == 0);
      if constexpr (ACT) {
        if (acc_ok) w.start();
      }
      if (acc_ok && split == 1) {
#pragma unroll 1
        for (int h = 0; h < halves; ++h) {  // accumulator h holds output rows [m0 + 128 h, +128)
          const uint32_t trow = tmem_row + (uint32_t)(h * BN);
          w.m_base = m0 + h * kUmmaBM + quad * 32;
#pragma unroll 1
          for (int ch = 0; ch < chunks; ++ch) {
            const uint32_t buf = w.begin_chunk();
#pragma unroll
            for (int sub = 0; sub < kSub; sub += 2) {  // two accumulator reads in flight per wait
              uint32_t r0[16], r1[16];
              tmem_ld_32x16(trow + (ch * kSub + sub) * 16, r0);
              tmem_ld_32x16(trow + (ch * kSub + sub + 1) * 16, r1);
              tmem_ld_wait();
              float v[16];
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r0[j]);
              w.put16(buf, sub, n0 + ch * kOutCols, v, bias_tile);
#pragma unroll
              for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r1[j]);
              w.put16(buf, sub + 1, n0 + ch * kOutCols, v, bias_tile);
            }
            w.end_chunk(buf, n0 + ch * kOutCols);
          }
          w.flush();  // a group never spans two row blocks
        }
        w.finish();
        mark(MARK_PARTIAL_WRITTEN, c.tid == 0);
      }
    }
    if (split > 1) umma_split_reduce<KIND>(c, BN, split, kslice, tiles, recv_bar, tmem_row, acc_ok, w, n0, bias_tile, tl);
    if constexpr (ACT) {
      if (warp < 4) w.drain();
    }
    tc_fence_before();
    c.sync();
    if (warp == 5 && !c.tmem_given) tmem_dealloc(tmem_acc, BN * halves);
    if (c.persistent && c.tid < stages) {  // the next tile of a persistent CTA initialises them again
      mbar_inval(full0 + 8 * c.tid);
      mbar_inval(empty0 + 8 * c.tid);
      if (c.tid == 0) {
        mbar_inval(acc_bar);
        mbar_inval(recv_bar);
      }
    }
    if (ACT && c.persistent && c.tid < 4 * kActBars) mbar_inval(full0 + kActBarOffset + 8 * c.tid);
    mark(MARK_END, c.tid == 0);
  }
};

// ---- large products: pairs of CTAs that walk tiles of 256 rows ----
//
// With a whole-SM tile per CTA the tensor pipe idles while the epilogue turns the accumulator into the output: 4096 x 14336 x
// 4096 with SiLU and a gate took 480 us, 357 without any epilogue to speak of; in pairs it takes 320 to 345.  Here two CTAs of a cluster multiply a
// 256 x 256 tile together (tcgen05 cta_group::2: each holds 128 rows of A, 128 rows of W and 128 rows of the accumulator, so
// the operands cost no more traffic per flop than a 256 x 256 tile on one SM), which leaves tensor memory for a second
// accumulator: one tile's epilogue runs under the next one's MMAs.  A pair takes every pairs-th tile, rows of tiles
// fastest; the rings go on across tiles.
//
// BlockDim = (192, 1, 1), warps as in GemmUmma; the MMAs are issued by the cluster's first CTA.  Every CTA loads its own
// operands and reports them to the first one's barriers; a stage is given up, and an accumulator announced, in both.
//
// What bounds them: the tensor pipe, 81 % busy in the SMs' active clocks (4096 x 14336 x 2048), at the clock that the power limit
// leaves.  Tiles of 256 x 128 are for products of few tiles, which then spread over twice the SMs: a K block's MMAs are half as
// long (256 clocks), but it takes 400 clocks of 24 KB of loads, so not where the wide tiles fill the device.
constexpr int kPairRows = 256, kPairBufs = 3;
__host__ __device__ constexpr int pair_stages(int bn) { return bn == 256 ? 5 : 7; }
__host__ __device__ constexpr int pair_stage_bytes(int bn) { return kUmmaABytes + bn / 2 * kUmmaRowBytes; }   // 128 rows of A, half of W's
__host__ __device__ constexpr int pair_smem_bytes(int bn) { return kUmmaHeaderBytes + pair_stages(bn) * pair_stage_bytes(bn) + kPairBufs * kUmmaStagingBytes; }

__device__ __forceinline__ void tma_load_3d_pair(uint32_t dst, const CUtensorMap *map, uint32_t cluster_bar, int c0, int c1, int c2) {
  asm volatile(
      "cp.async.bulk.tensor.3d.cta_group::2.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%3, %4, %5}], [%2];" ::"r"(dst),
      "l"(map), "r"(cluster_bar), "r"(c0), "r"(c1), "r"(c2)
      : "memory");
}
__device__ __forceinline__ void umma_ss_pair(uint32_t d_tmem, uint32_t a_lo, uint32_t b_lo, uint32_t idesc, uint32_t accumulate) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 da, db;\n\tsetp.ne.b32 p, %5, 0;\n\tmov.b64 da, {%1, %3};\n\tmov.b64 db, {%2, %3};\n\t"
      "tcgen05.mma.cta_group::2.kind::f16 [%0], da, db, %4, p;\n\t}" ::"r"(d_tmem),
      "r"(a_lo), "r"(b_lo), "r"(kUmmaDescHi), "r"(idesc), "r"(accumulate)
      : "memory");
}
// arrives at the barrier at this address in both CTAs of the pair once the MMAs issued so far are done
__device__ __forceinline__ void umma_commit_pair(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::2.mbarrier::arrive::one.shared::cluster.multicast::cluster.b64 [%0], %1;" ::"r"(bar), "h"((uint16_t)3) : "memory");
}
__device__ __forceinline__ void mbar_arrive_cluster(uint32_t cluster_bar) {
  asm volatile("mbarrier.arrive.release.cluster.shared::cluster.b64 _, [%0];" ::"r"(cluster_bar) : "memory");
}

// As ActWriter, tile after tile through three buffers: the next chunk's `other` is on its way while this one is worked on.
struct PairWriter : ActWriter {
  int base = 0;   // chunks of the tiles before this one
  __device__ __forceinline__ void load_chunk(int q) {
    const uint32_t s = (uint32_t)(q % kPairBufs), bar = bar0 + 8 * s;
    mbar_expect_tx(bar, 4096u);
    tma_load_3d(buf0 + s * 4096u, &pa->map_other, bar, col0 + (q - base) * nb_step, m0, bz);
  }
  __device__ __forceinline__ uint32_t begin_chunk() {
    if (lane == 0) {
      tma_store_wait_read<1>();   // all but the last chunk's store have read their buffers: this one's and the next one's are free
      if (pa->has_other) {
        if (next >= loaded) load_chunk(next);
        if (next + 1 < total) load_chunk(next + 1);
      }
    }
    __syncwarp();
    if (pa->has_other) {
      loaded = min(next + 2, total);
      mbar_wait(bar0 + 8 * (uint32_t)(next % kPairBufs), (next / kPairBufs) & 1, status, UMMA_WAIT_OTHER_TIMEOUT);
      __syncwarp();
    }
    ++next;
    return buf0 + (uint32_t)slot * 4096u;
  }
};

struct GemmActPairs {
  using Params = GemmActParams;
  static constexpr int kMaxThreads = kUmmaThreads;
  static constexpr int kMinBlocks = 1;
  static constexpr bool kMemoryBound = false;
  static constexpr bool kUsesTmem = true;
  static constexpr int kBK = 64;

  __device__ __forceinline__ static void run(const Params &p, const TileCtx &c) {
    const int warp = c.tid >> 5, lane = c.tid & 31, quad = (threadIdx.x >> 5) & 3;
    const int rank = c.vblock & 1, pair = c.vblock >> 1, pairs = c.gx >> 1;
    const int BN = p.bn, stages = p.stages, stage_bytes = pair_stage_bytes(BN);
    const int tiles_m = (p.M + kPairRows - 1) / kPairRows, tiles_n = (p.N + BN - 1) / BN, total = p.batch * tiles_m * tiles_n;
    const int num_kb = (p.K + kBK - 1) / kBK;
    const uint32_t full0 = smem_u32(c.smem), empty0 = full0 + 8 * kUmmaMaxStages, acc_full = empty0 + 8 * kUmmaMaxStages, acc_empty = acc_full + 16;
    uint32_t *tmem_slot = reinterpret_cast<uint32_t *>(c.smem + 8 * (2 * kUmmaMaxStages + 4));
    float *bias_tile = reinterpret_cast<float *>(c.smem + 1024);
    const uint32_t ring = full0 + kUmmaHeaderBytes, staging = ring + (uint32_t)(stages * stage_bytes);
    if (warp == 5) {
      asm volatile("tcgen05.alloc.cta_group::2.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(smem_u32(tmem_slot)), "r"(512) : "memory");
      asm volatile("tcgen05.relinquish_alloc_permit.cta_group::2.sync.aligned;" ::: "memory");
    }
    if (warp == 4) {
      if (lane < stages) {
        mbar_init(full0 + 8 * lane, 1);
        mbar_init(empty0 + 8 * lane, 1);
      }
      if (lane < 2) {
        mbar_init(acc_full + 8 * lane, 1);
        mbar_init(acc_empty + 8 * lane, 256);
      }
      if (lane < 4 * kActBars) mbar_init(full0 + kActBarOffset + 8 * lane, 1);
      if (lane < 3 + p.has_other) asm volatile("prefetch.tensormap [%0];" ::"l"(lane == 0 ? &p.map_a : lane == 1 ? &p.map_b : lane == 2 ? &p.map_out : &p.map_other) : "memory");
      asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
      __syncwarp();
    }
    c.dependency_wait();
    tc_fence_before();
    cluster_sync_all();   // both CTAs' barriers are up, both have their tensor memory
    tc_fence_after();
    const uint32_t tmem = *reinterpret_cast<volatile uint32_t *>(tmem_slot);
    // tile i of this pair: M tiles vary fastest, so that the pairs at work share their W
    auto place = [&](int t, int &m0, int &n0, int &bz) {
      m0 = t % tiles_m * kPairRows;
      n0 = t / tiles_m % tiles_n * BN;
      bz = t / (tiles_m * tiles_n);
    };
    bool ok = true;
    if (warp == 4) {
      if (elect_one()) {
        uint32_t s = 0, ph = 1;
        for (int t = pair; t < total && ok; t += pairs) {
          int m0, n0, bz;
          place(t, m0, n0, bz);
          m0 += rank * kUmmaBM, n0 += rank * (BN / 2);
          for (int kb = 0; kb < num_kb; ++kb) {
            ok = mbar_wait(empty0 + 8 * s, ph, c.status, UMMA_WAIT_EMPTY_TIMEOUT);
            if (!ok) break;
            const uint32_t dst = ring + s * (uint32_t)stage_bytes, bar = peer_smem(full0 + 8 * s, 0);
            if (rank == 0) mbar_expect_tx(full0 + 8 * s, 2u * (uint32_t)stage_bytes);
            tma_load_3d_pair(dst, &p.map_a, bar, kb * kBK, m0, bz);
            tma_load_3d_pair(dst + kUmmaABytes, &p.map_b, bar, kb * kBK, n0, bz);
            if (++s == (uint32_t)stages) s = 0, ph ^= 1;
          }
        }
        // the last release of every slot that was used: none may be in flight when this CTA ends
        const int mine = total > pair ? (total - pair + pairs - 1) / pairs : 0;
        const long long uses = (long long)mine * num_kb;
        if (uses < stages) s = 0, ph = 0;
        for (int i = 0; i < stages && i < uses && ok; ++i) {
          ok = mbar_wait(empty0 + 8 * s, ph, c.status, UMMA_WAIT_EMPTY_TIMEOUT);
          if (++s == (uint32_t)stages) s = 0, ph ^= 1;
        }
      }
      __syncwarp();
    } else if (warp == 5) {
      if (rank == 0 && elect_one()) {
        const uint32_t idesc = (1u << 4) | (1u << 7) | (1u << 10) | ((uint32_t)(BN >> 3) << 17) | ((uint32_t)(kPairRows >> 4) << 24);
        const uint32_t lo0 = ((ring >> 4) & 0x3fffu) | (1u << 16);
        uint32_t s = 0, ph = 0, lo = lo0;
        int i = 0;
        for (int t = pair; t < total && ok; t += pairs, ++i) {
          const uint32_t acc = tmem + (uint32_t)(i & 1) * 256u;
          ok = mbar_wait(acc_empty + 8 * (i & 1), ((i >> 1) & 1) ^ 1, c.status, UMMA_WAIT_ACC_TIMEOUT);
          tc_fence_after();
          for (int kb = 0; kb < num_kb && ok; ++kb) {
            ok = mbar_wait(full0 + 8 * s, ph, c.status, UMMA_WAIT_FULL_TIMEOUT);
            if (!ok) break;
            tc_fence_after();
#pragma unroll
            for (int j = 0; j < 4; ++j) umma_ss_pair(acc, lo + 2 * j, lo + (kUmmaABytes >> 4) + 2 * j, idesc, kb > 0 || j > 0);
            umma_commit_pair(empty0 + 8 * s);
            if (++s == (uint32_t)stages) s = 0, ph ^= 1, lo = lo0;
            else lo += (uint32_t)stage_bytes >> 4;
          }
          umma_commit_pair(acc_full + 8 * (i & 1));
        }
      }
      __syncwarp();
    } else {
      PairWriter w{};
      const int chunks = BN / 64;
      w.map_out = &p.map_out, w.M = p.M, w.N = p.N, w.causal = 0;
      w.buf0 = staging + (uint32_t)(quad * kPairBufs) * 4096u;
      w.nbuf = kPairBufs, w.lane = lane, w.nb_step = 64, w.group = 1;
      w.pa = &p, w.bar0 = full0 + kActBarOffset + 8 * kActBars * quad, w.status = c.status, w.per_half = chunks;
      const uint32_t empty_at[2] = {peer_smem(acc_empty, 0), peer_smem(acc_empty + 8, 0)};
      int i = 0;
      for (int t = pair; t < total; t += pairs, ++i) {   // (to the end after a wait that gave up, too: the four warps meet in every tile)
        int m0, n0, bz;
        place(t, m0, n0, bz);
        m0 += rank * kUmmaBM;
        asm volatile("bar.sync %0, 128;" ::"r"(c.bar_id + 8) : "memory");   // the last tile's bias has been read
        for (int k = c.tid; k < BN; k += 128) bias_tile[k] = (p.bias && n0 + k < p.N) ? __ldg(p.bias + n0 + k) : 0.f;
        asm volatile("bar.sync %0, 128;" ::"r"(c.bar_id + 8) : "memory");
        w.m_base = w.m0 = m0 + quad * 32, w.bz = bz, w.n_tile0 = w.col0 = n0;
        w.base = chunks * i, w.total = chunks * (i + 1);
        if (ok) ok = __all_sync(0xffffffffu, mbar_wait(acc_full + 8 * (i & 1), (i >> 1) & 1, c.status, UMMA_WAIT_ACC_TIMEOUT));
        if (!ok) continue;
        tc_fence_after();
        const uint32_t trow = tmem + (uint32_t)(i & 1) * 256u + ((uint32_t)(quad * 32) << 16);
#pragma unroll 1
        for (int ch = 0; ch < chunks; ++ch) {
          const uint32_t buf = w.begin_chunk();
#pragma unroll
          for (int sub = 0; sub < 4; sub += 2) {
            uint32_t r0[16], r1[16];
            tmem_ld_32x16(trow + (ch * 4 + sub) * 16, r0);
            tmem_ld_32x16(trow + (ch * 4 + sub + 1) * 16, r1);
            tmem_ld_wait();
            float v[16];
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r0[j]);
            w.put16(buf, sub, n0 + ch * 64, v, bias_tile);
#pragma unroll
            for (int j = 0; j < 16; ++j) v[j] = __uint_as_float(r1[j]);
            w.put16(buf, sub + 1, n0 + ch * 64, v, bias_tile);
          }
          w.end_chunk(buf, n0 + ch * 64);
        }
        tc_fence_before();
        mbar_arrive_cluster(empty_at[i & 1]);   // this accumulator may be written again
      }
      w.finish();
      w.drain();
    }
    __syncwarp();
    tc_fence_before();
    cluster_sync_all();   // neither CTA's memory is read, or reported to, any more
    tc_fence_after();
    if (warp == 5) asm volatile("tcgen05.dealloc.cta_group::2.sync.aligned.b32 %0, %1;" ::"r"(tmem), "r"(512) : "memory");
  }
};

}  // namespace bfuse
