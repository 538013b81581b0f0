// pa_prompt.cu -- prompt attention over paged K/V caches for B200 (sm_100a).
//
// Chunks of new tokens attend to their sequences' cached tokens, their own
// among them (causal), under an optional sliding window with visible first
// tokens. For query row r at position p, over the tokens t that it sees
// (t <= p and (t < sinks or t > p - window)):
//
//   o = sum_t 2^(c q.k_t - m) v_t / sum_t 2^(c q.k_t - m),   c = scale log2(e)
//
// with a running m: one pass over the keys. What a chunk costs is 4 D operations
// per (query head, visible token); keys and values are read once per 128 or 256
// query rows, so long chunks are bound by the matrix pipe and the exponentials.
#include <cuda.h>
#include <cuda_runtime.h>
#include <cudaTypedefs.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <stdint.h>
#include <string.h>

#include <algorithm>
#include <climits>
#include <mutex>
#include <numeric>
#include <type_traits>

#include "pa_decode.h"
#include "fastdiv.h"

namespace pp {

using pa::FastDiv;
using pa::fast_div;
using pa::make_fastdiv;

constexpr unsigned kFull = 0xffffffffu;
constexpr float kSentinel = -1e30f;     // LSE of a row that sees nothing
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kNaN = __builtin_nanf("");
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const char* q;
  long long q_st, q_sh;                           // bytes
  const char* kc;
  const char* vc;
  long long k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;   // bytes (Fetch::kPieces)
  const int* bt;
  long long bt_sb;                                // elements
  int max_blocks;
  const int* starts;
  const int* lens;
  int T, B, Hq, Hkv, G, bs, NB;
  int window, sinks;                              // window: INT_MAX stands for none
  float scale_log2;
  char* out;
  long long o_st, o_sh;                           // bytes
  float* lse;
  unsigned* status;
};

__device__ __forceinline__ void flag(const Params& p, unsigned bits) {
  if (p.status) atomicOr(p.status, bits);
}

// Sequence b's queries [start, start + n) and length S. A range outside the
// queries or a length outside the table is cut to what there is and flagged.
struct Seq { int start, n, S; };
__device__ __forceinline__ Seq load_seq(const Params& p, int b, bool& bad) {
  Seq s;
  const int s0 = __ldg(p.starts + b), s1 = __ldg(p.starts + b + 1), len = __ldg(p.lens + b);
  const long long cap = static_cast<long long>(p.max_blocks) * p.bs;
  s.start = min(max(s0, 0), p.T);
  s.n = max(0, min(s1, p.T) - s.start);
  s.S = len < 0 ? 0 : len > cap ? static_cast<int>(cap) : len;
  bad = s0 < 0 || s1 < s0 || s1 > p.T || len < 0 || len > cap;
  return s;
}

// (a, b) rounded to the 16-bit type, a in the low half.
template <typename T>
__device__ __forceinline__ uint32_t pack2(float a, float b);
template <>
__device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
  const __half2 h = __floats2half2_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}
template <>
__device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
  const __nv_bfloat162 h = __floats2bfloat162_rn(a, b);
  return *reinterpret_cast<const uint32_t*>(&h);
}

// The sequence that holds a query row (warp-uniform), -1 for a row of none.
__device__ __forceinline__ int seq_of_row(const Params& p, int row) {
  const int lane = threadIdx.x & 31;
  if (p.B < 32) {                        // one load per lane, no search
    const int s = lane <= p.B ? __ldg(p.starts + lane) : 0;
    const unsigned at = __ballot_sync(kFull, lane < p.B && s <= row);
    const int b = at ? 31 - __clz(at) : 0;
    const int s0 = __shfl_sync(kFull, s, b), s1 = __shfl_sync(kFull, s, b + 1);
    return row >= s0 && row < s1 ? b : -1;
  }
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(p.starts + mid) <= row) lo = mid; else hi = mid - 1;
  }
  return row >= __ldg(p.starts + lo) && row < __ldg(p.starts + lo + 1) ? lo : -1;
}

// ----------------------------------------------------------------------------
// Tile path: tcgen05 over pages copied by TMA
// ----------------------------------------------------------------------------
// One CTA takes 128 * NQ packed query rows of one (sequence, KV head): row R is
// token R / G, head R % G of the group, so that the G query heads that share the
// keys share their tiles. It walks the keys that any of its rows sees, the visible
// first tokens and the window's from its first to the last row's position, in
// tiles of kTN. Per tile and 128 rows:
//
//   S (128 x kTN, TMEM) = Q K^T       one tcgen05.mma per 16 dimensions
//   P = 2^(c S - m), rounded to the 16-bit type, over S in TMEM
//   O (128 x D, TMEM) += P V          one tcgen05.mma per 16 tokens
//
// Roles: producer warps (lane = one copy: a box of a page), a warp that cleans V
// tiles at the edges of what is visible, one issuing warp per 128 rows, and four
// softmax warps per 128 rows, thread = row, so that row maxima and sums need no
// exchange. With NQ = 2 the two row tiles alternate on the matrix pipe: while
// one's S is turned into P, the other's products run. With NQ = 1 (short chunks,
// head_dim 256) S has two buffers and the next tile's S is computed during the
// current softmax.
//
// What bounds it (8192 tokens, Hq32/Hkv8, D 128, window 4096 / none: 368 / 466 us,
// 1.12 / 1.18 PFLOP/s, in runs of 100 calls; 410 / 525 us, 1.0 / 1.05 PFLOP/s, once
// calls follow each other for 0.4 s and the power cap lowers the clock; comparisons
// here and below are of short runs): the chain from a tile's S to its P. 256 rows x 128 keys
// take the matrix pipe 2048 cycles, the special function units as many, and the
// tile's turn ~3000: load of S 250, maximum 300-400, exponentials 1400 (1024 if no
// other warp ran), then the rest of P V and the next S 1000. Tried and slower:
// two threads per row (twice the warps; a meeting for each maximum, registers
// spill: 481 us where one thread took 425), tiles of 64 keys with two S buffers
// (S is no longer waited for, but every tile's fixed costs double and the row
// tile is read twice as often: 418 against 388), P formed against the previous
// maximum while the new one is taken (430 against 388), a grid of one CTA
// per SM that walks its jobs with the next keys already loading (376 against 361;
// the hardware's order of CTAs balances better than any fixed one).
//
// P is rounded to the operand type once (half a step, relative); its sum, the
// maxima and O are kept in 32 bits. The roundings of P are independent of the one of
// the output and for values of random sign add up to as much: the error against 64
// bits is up to sqrt(2) times that of rounding the exact result (measured 1.25-1.4),
// and in each element at most half a step of the largest value more. Keeping P as a
// pair of 16-bit parts, as decode does, would make P V two products (half as much
// again on the matrix pipe). O is rescaled only when a row's maximum has grown by more than 2^8: until then P and the sum are relative to an older
// maximum, which changes neither's relative rounding (P <= 2^8).
//
// Masks: a tile that is not entirely visible to all rows of a warp compares
// each score's token with the row's limits. Tokens that no row sees are cut off
// in steps of 16 by the products' shape (N of the first, K of the second); the V
// rows of such tokens inside the remaining steps are zeroed in shared memory
// first, as 0 * NaN would reach O.
template <int D, int NQ>
struct TC {
  static constexpr int kTN = D == 256 ? 64 : 128;      // keys per tile
  static constexpr int kChunks = D / 64;               // 128-byte chunks of a row
  static constexpr int kQTile = 128 * D * 2;
  static constexpr int kKV = kTN * D * 2;              // one K or V tile
  static constexpr int kSlots = D == 128 && NQ == 1 ? 6 : 5;
  // CTAs per SM. head_dim 64 fits two of one row tile each: one's set-up and output
  // run beside the other's products (8192 tokens, Hq32/Hkv8: 382 us against 410 as
  // one CTA of two row tiles). At 128 the ring would shrink to two tiles.
  static constexpr int kCtas = D == 64 ? 2 : 1;
  static constexpr int kSmem = NQ * kQTile + kSlots * kKV + 1024;
  static constexpr int kSBufs = NQ == 2 || kCtas == 2 ? 1 : 2;   // S buffers per row tile
  static constexpr int kOCol = NQ * kSBufs * kTN;      // first TMEM column of O
  // warps: 4 softmax and one issuing warp per row tile, the producers, the cleaner;
  // full warpgroups split their registers unevenly
  static constexpr int kProducers = NQ == 2 ? 4 : 2;
  static constexpr int kThreads = NQ == 2 ? 512 : 128 + (1 + kProducers + 1) * 32;
  // V tiles handed on by the cleaner, at most one ring of them ahead
  static constexpr int kVBars = 4;
  static_assert(2 * kVBars >= kSlots, "V barriers");
  static constexpr int kBars = 2 * kSlots + kVBars + NQ * (7 + kSBufs);
  static constexpr int kTmemCols = 512 / kCtas;
  // 128 registers a thread at launch, where they are split
  static constexpr bool kSplitRegs = kThreads * kCtas == 512;
  static_assert(kOCol + NQ * D <= kTmemCols, "tensor memory");
  static_assert((kSmem + 2048) * kCtas <= 233472, "shared memory");
};
constexpr unsigned long long kWaitLimitNs = 2000000000ull;   // 2 s per barrier wait
constexpr float kRescaleLog2 = 8.f;
// Registers per thread of a 512-thread CTA: 128 at launch; the two softmax
// warpgroups take kSoftmaxRegs once the two others have gone down to kOtherRegs.
// (At the launch's share the softmax spills, and with shared memory full of tiles
// the spills miss the first-level cache.)
constexpr int kLaunchRegs = 128, kSoftmaxRegs = 200, kOtherRegs = 56;
static_assert(kSoftmaxRegs + kOtherRegs <= 2 * kLaunchRegs, "register split");
template <int N>
__device__ __forceinline__ void regs_up() {
  asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(N));
}
template <int N>
__device__ __forceinline__ void regs_down() {
  asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(N));
}

// How the keys' rows come: boxes of a page's rows (page size a multiple of 8), four
// rows by their numbers in the cache seen as one list of rows (other page sizes), or
// 16 bytes at a time by cp.async (strides that make no such list).
enum class Fetch { kBoxes, kRows, kPieces };
struct TileParams {
  Params p;
  int dh;                   // head_dim: D, or 32 in the kernel for 64
  int R, lR;                // token rows per TMA box, and its log2
  int bs_log2;              // log2 of the page size, or -1
  FastDiv div_g, div_bs;
  int row_b[2], row_s[2], row_h[2];   // kRows: rows from a page, slot, head to the next, of K and V
  int splits;
  float* o_part;            // [splits][T * Hq][D], splits > 1
  float* lse_part;          // [splits][T * Hq]
};

__device__ __forceinline__ uint32_t smem_u32(const void* p) {
  return static_cast<uint32_t>(__cvta_generic_to_shared(p));
}
__device__ __forceinline__ void mbar_init(uint32_t bar, uint32_t count) {
  asm volatile("mbarrier.init.shared::cta.b64 [%0], %1;" ::"r"(bar), "r"(count) : "memory");
}
__device__ __forceinline__ void mbar_arrive(uint32_t bar) {
  asm volatile("mbarrier.arrive.shared::cta.b64 _, [%0];" ::"r"(bar) : "memory");
}
__device__ __forceinline__ void mbar_expect_tx(uint32_t bar, uint32_t bytes) {
  asm volatile("mbarrier.arrive.expect_tx.shared::cta.b64 _, [%0], %1;" ::"r"(bar), "r"(bytes)
               : "memory");
}
__device__ __forceinline__ bool mbar_try_wait(uint32_t bar, uint32_t parity) {
  uint32_t ok;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "mbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(ok)
      : "r"(bar), "r"(parity)
      : "memory");
  return ok != 0;
}
__device__ __forceinline__ unsigned long long global_ns() {
  unsigned long long t;
  asm volatile("mov.u64 %0, %%globaltimer;" : "=l"(t));
  return t;
}
// Waits for the barrier's phase with a wall-clock bound; false on timeout.
__device__ __forceinline__ bool mbar_wait(uint32_t bar, uint32_t parity) {
  if (mbar_try_wait(bar, parity)) return true;
  const unsigned long long t0 = global_ns();
  while (true) {
#pragma unroll 1
    for (int i = 0; i < 32; ++i)
      if (mbar_try_wait(bar, parity)) return true;
    if (global_ns() - t0 > kWaitLimitNs) return false;
  }
}
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* map, int c0, int c1,
                                            int c2, int c3, int c4, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.5d.shared::cluster.global.tile.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c0), "r"(c1), "r"(c2), "r"(c3), "r"(c4), "r"(bar)
      : "memory");
}
// Four rows of 64 dimensions, from column c on.
__device__ __forceinline__ void tma_load_rows(uint32_t dst, const CUtensorMap* map, int c, int r0,
                                              int r1, int r2, int r3, uint32_t bar) {
  asm volatile(
      "cp.async.bulk.tensor.2d.shared::cta.global.tile::gather4.mbarrier::complete_tx::bytes"
      " [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst),
      "l"(reinterpret_cast<uint64_t>(map)), "r"(c), "r"(r0), "r"(r1), "r"(r2), "r"(r3), "r"(bar)
      : "memory");
}
// One lane of a converged warp. (A lane elected this way is known to be alone,
// so that the matrix instructions behind the branch take their operands from
// uniform registers directly.)
__device__ __forceinline__ bool elect_one() {
  uint32_t is;
  asm volatile(
      "{\n\t.reg .pred p;\n\t"
      "elect.sync _|p, 0xffffffff;\n\t"
      "selp.u32 %0, 1, 0, p;\n\t}"
      : "=r"(is));
  return is != 0;
}
__device__ __forceinline__ void fence_async_smem() {
  asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_before() {
  asm volatile("tcgen05.fence::before_thread_sync;" ::: "memory");
}
__device__ __forceinline__ void tc_fence_after() {
  asm volatile("tcgen05.fence::after_thread_sync;" ::: "memory");
}
// Arrival on the barrier once every matrix instruction issued so far is done.
__device__ __forceinline__ void tc_commit(uint32_t bar) {
  asm volatile("tcgen05.commit.cta_group::1.mbarrier::arrive::one.shared::cluster.b64 [%0];" ::"r"(bar)
               : "memory");
}
template <int kCols>
__device__ __forceinline__ void tmem_free(uint32_t tmem) {
  asm volatile("tcgen05.dealloc.cta_group::1.sync.aligned.b32 %0, %1;" ::"r"(tmem), "n"(kCols)
               : "memory");
}
// Shared-memory matrix descriptor, 128-byte swizzle: 8-row groups 1024 bytes
// apart; `lead`: bytes between the 64-element blocks of an operand whose
// contiguous dimension is not the summed one (V), unused otherwise. The high
// word is the same for every operand here; advancing by b bytes adds b / 16 to
// the low one.
constexpr uint32_t kDescHigh = 1024 >> 4 | 1u << 14 | 2u << 29;
__device__ __forceinline__ uint32_t smem_desc(uint32_t addr, uint32_t lead) {
  return (addr & 0x3ffff) >> 4 | (lead >> 4) << 16;
}
// D[tmem] (+)= A[smem] B[smem], and with A in tensor memory.
__device__ __forceinline__ void mma_ss(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 x, y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 x, {%1, %5};\n\tmov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], x, y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "n"(kDescHigh)
      : "memory");
}
__device__ __forceinline__ void mma_ts(uint32_t d, uint32_t a, uint32_t b, uint32_t idesc, bool add) {
  asm volatile(
      "{\n\t.reg .pred p;\n\t.reg .b64 y;\n\tsetp.ne.b32 p, %4, 0;\n\t"
      "mov.b64 y, {%2, %5};\n\t"
      "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], y, %3, p;\n\t}" ::"r"(d),
      "r"(a), "r"(b), "r"(idesc), "r"(static_cast<uint32_t>(add)), "n"(kDescHigh)
      : "memory");
}
// Instruction descriptor: 32-bit accumulator, A and B of type T, M = 128;
// `b_mn`: B's contiguous dimension is N (V), else K.
template <typename T>
__device__ __forceinline__ constexpr uint32_t instr_desc(int n, bool b_mn) {
  const uint32_t ty = sizeof(T) == 2 && std::is_same<T, __nv_bfloat16>::value ? 1u : 0u;
  return 1u << 4 | ty << 7 | ty << 10 | (b_mn ? 1u : 0u) << 16 |
         static_cast<uint32_t>(n >> 3) << 17 | (128u >> 4) << 24;
}
// Pairs of 32-bit floats: one issue slot for two elements.
__device__ __forceinline__ uint64_t f2(float x, float y) {
  uint64_t r;
  asm("mov.b64 %0, {%1, %2};" : "=l"(r) : "f"(x), "f"(y));
  return r;
}
__device__ __forceinline__ void f2_split(uint64_t v, float& x, float& y) {
  asm("mov.b64 {%0, %1}, %2;" : "=f"(x), "=f"(y) : "l"(v));
}
__device__ __forceinline__ uint64_t f2_fma(uint64_t a, uint64_t b, uint64_t c) {
  uint64_t r;
  asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(r) : "l"(a), "l"(b), "l"(c));
  return r;
}
__device__ __forceinline__ uint64_t f2_add(uint64_t a, uint64_t b) {
  uint64_t r;
  asm("add.rn.f32x2 %0, %1, %2;" : "=l"(r) : "l"(a), "l"(b));
  return r;
}
__device__ __forceinline__ float max3(float a, float b, float c) {   // NaN if any is
  float r;
  asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(r) : "f"(a), "f"(b), "f"(c));
  return r;
}
__device__ __forceinline__ float max_nan(float a, float b) {   // NaN if either is
  float r;
  asm("max.NaN.f32 %0, %1, %2;" : "=f"(r) : "f"(a), "f"(b));
  return r;
}
// (2^x, 2^y) on the FMA pipe, for a share of the exponentials (the special
// function unit does 4 a cycle per scheduler: 2048 cycles for 256 rows x 128 keys, as
// long as the two products take): n =
// the integer nearest to x, from the low bits of x + 1.5 * 2^23; 2^(x - n) by a
// polynomial of degree 4 fitted to the least largest relative error on [-1/2,
// 1/2] with its constant term held at 1 (2.9e-6 in 32-bit arithmetic; P is
// rounded to 2^-9 or 2^-12 of it); n added to the exponent. x < 128. Arguments
// up to -127 give 0 exactly, NaN gives infinity or NaN.
__device__ __forceinline__ void ex2_pair_fma(uint64_t v, float& x, float& y) {
  f2_split(v, x, y);
  v = f2(max_nan(x, -127.f), max_nan(y, -127.f));
  const float kRound = 12582912.f;
  const uint64_t t = f2_add(v, f2(kRound, kRound));
  const uint64_t n = f2_add(t, f2(-kRound, -kRound));
  const uint64_t f = f2_fma(n, f2(-1.f, -1.f), v);
  uint64_t r = f2(0.009582852013409138f, 0.009582852013409138f);
  r = f2_fma(r, f, f2(0.055906426161527634f, 0.055906426161527634f));
  r = f2_fma(r, f, f2(0.24024099111557007f, 0.24024099111557007f));
  r = f2_fma(r, f, f2(0.6931241750717163f, 0.6931241750717163f));
  r = f2_fma(r, f, f2(1.f, 1.f));
  float tx, ty;
  f2_split(t, tx, ty);
  f2_split(r, x, y);
  x = __uint_as_float(__float_as_uint(x) + (__float_as_uint(tx) << 23));
  y = __uint_as_float(__float_as_uint(y) + (__float_as_uint(ty) << 23));
}
__device__ __forceinline__ float ex2(float x) {
  float y;
  asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
  return y;
}
// 32 rows (lanes of the warp's quarter) x N columns of tensor memory, thread = row.
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%32];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31])
      : "r"(addr + 0)
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[64]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%64];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%65];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
        "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63])
      : "r"(addr + 0), "r"(addr + 32)
      : "memory");
}
__device__ __forceinline__ void tmem_ld(uint32_t addr, uint32_t (&r)[128]) {
  asm volatile(
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%0, %1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31}, [%128];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%32, %33, %34, %35, %36, %37, %38, %39, %40, %41, %42, %43, %44, %45, %46, %47, %48, %49, %50, %51, %52, %53, %54, %55, %56, %57, %58, %59, %60, %61, %62, %63}, [%129];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%64, %65, %66, %67, %68, %69, %70, %71, %72, %73, %74, %75, %76, %77, %78, %79, %80, %81, %82, %83, %84, %85, %86, %87, %88, %89, %90, %91, %92, %93, %94, %95}, [%130];\n\t"
      "tcgen05.ld.sync.aligned.32x32b.x32.b32 {%96, %97, %98, %99, %100, %101, %102, %103, %104, %105, %106, %107, %108, %109, %110, %111, %112, %113, %114, %115, %116, %117, %118, %119, %120, %121, %122, %123, %124, %125, %126, %127}, [%131];\n\t"
      "tcgen05.wait::ld.sync.aligned;"
      : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),
        "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]),
        "=r"(r[15]), "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]),
        "=r"(r[22]), "=r"(r[23]), "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]),
        "=r"(r[29]), "=r"(r[30]), "=r"(r[31]), "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]),
        "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]), "=r"(r[40]), "=r"(r[41]), "=r"(r[42]),
        "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]), "=r"(r[48]), "=r"(r[49]),
        "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]), "=r"(r[56]),
        "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),
        "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]),
        "=r"(r[71]), "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]),
        "=r"(r[78]), "=r"(r[79]), "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]),
        "=r"(r[85]), "=r"(r[86]), "=r"(r[87]), "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]),
        "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]), "=r"(r[96]), "=r"(r[97]), "=r"(r[98]),
        "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), "=r"(r[104]),
        "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]),
        "=r"(r[111]), "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]),
        "=r"(r[117]), "=r"(r[118]), "=r"(r[119]), "=r"(r[120]), "=r"(r[121]), "=r"(r[122]),
        "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])
      : "r"(addr + 0), "r"(addr + 32), "r"(addr + 64), "r"(addr + 96)
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[16]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16};"
      :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15])
      : "memory");
}
__device__ __forceinline__ void tmem_st(uint32_t addr, const uint32_t (&r)[32]) {
  asm volatile(
      "tcgen05.st.sync.aligned.32x32b.x32.b32 [%0], {%1, %2, %3, %4, %5, %6, %7, %8, %9, %10, %11, %12, %13, %14, %15, %16, %17, %18, %19, %20, %21, %22, %23, %24, %25, %26, %27, %28, %29, %30, %31, %32};"
      :: "r"(addr), "r"(r[0]), "r"(r[1]), "r"(r[2]), "r"(r[3]), "r"(r[4]), "r"(r[5]), "r"(r[6]), "r"(r[7]),
        "r"(r[8]), "r"(r[9]), "r"(r[10]), "r"(r[11]), "r"(r[12]), "r"(r[13]), "r"(r[14]), "r"(r[15]),
        "r"(r[16]), "r"(r[17]), "r"(r[18]), "r"(r[19]), "r"(r[20]), "r"(r[21]), "r"(r[22]), "r"(r[23]),
        "r"(r[24]), "r"(r[25]), "r"(r[26]), "r"(r[27]), "r"(r[28]), "r"(r[29]), "r"(r[30]), "r"(r[31])
      : "memory");
}
// The lowest n bits (none for n <= 0, all for n >= 32).
__device__ __forceinline__ uint32_t ones_below(int n) {
  return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1;
}
// A CTA's work: its rows and the keys they see. The keys are numbered without
// those that no row sees: the sinks, rounded up to whole boxes of R tokens
// (`sink_keys`), then the window from the box of its first token on; key v is
// token v, or v + delta behind the sinks. Tiles are kTN of these keys, so that a
// few sinks cost a few keys and not a tile, and the window starts at a tile's
// first columns whatever its place (ragged batch of 8, window 777: 51 us against
// 61 with separate, aligned tiles).
struct Job {
  int b, kvh, split;
  Seq s;
  int r0, rows;             // first packed row, packed rows of the sequence
  int sink_keys, delta;
  int gap0, gap1;           // keys [gap0, gap1) are seen by no row
  int end;                  // keys
  int sinks;                // visible first tokens (at most the sequence)
  int k0, k1;               // tiles of this CTA
};
// A tile's first key, and the range [from, to) of its keys that some row sees
// (except those in the gap).
struct KeyTile { int base, from, to; };
template <int kTN>
__device__ __forceinline__ KeyTile key_tile(const Job& j, int k) {
  KeyTile t;
  t.base = k * kTN;
  t.from = t.base >= j.gap0 && t.base < j.gap1 ? j.gap1 : t.base;
  t.to = min(t.base + kTN, j.end);
  return t;
}

// The job of block x, or false. Tiles are numbered from the last sequence's last
// rows, which see the most keys under a causal mask, to the first ones.
template <int D, int NQ>
__device__ __forceinline__ bool find_job(const TileParams& a, Job& j, int* sh) {
  constexpr int kRows = 128 * NQ, kTN = TC<D, NQ>::kTN;
  const Params& p = a.p;
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5, nw = blockDim.x >> 5;
  const int per = p.Hkv * a.splits;
  const int x = blockIdx.x / per;
  const int rest = blockIdx.x - x * per;
  bool bad = false;
  int tile = 0;
  if (p.B <= 32) {
    // few sequences: every warp finds the job by itself
    const int b = p.B - 1 - lane;
    Seq s = {0, 0, 0};
    if (b >= 0) s = load_seq(p, b, bad);
    if (bad && blockIdx.x == 0 && warp == 0) flag(p, PA_STATUS_BAD_SEQLEN);
    const int nt = (s.n * p.G + kRows - 1) / kRows;
    int v = nt;
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
      const int u = __shfl_up_sync(kFull, v, o);
      if (lane >= o) v += u;
    }
    const unsigned reach = __ballot_sync(kFull, x < v);
    if (!reach) return false;
    const int src = __ffs(reach) - 1;
    tile = __shfl_sync(kFull, v, src) - 1 - x;
    j.b = p.B - 1 - src;
    j.s.start = __shfl_sync(kFull, s.start, src);
    j.s.n = __shfl_sync(kFull, s.n, src);
    j.s.S = __shfl_sync(kFull, s.S, src);
  } else {
    // running sums over the sequences, from the last to the first
    int before = 0;
    if (threadIdx.x == 0) sh[32] = -1;
    for (int b0 = 0; b0 < p.B; b0 += blockDim.x) {
      const int b = p.B - 1 - (b0 + static_cast<int>(threadIdx.x));
      int nt = 0;
      bad = false;
      if (b >= 0) nt = (load_seq(p, b, bad).n * p.G + kRows - 1) / kRows;
      if (bad && blockIdx.x == 0) flag(p, PA_STATUS_BAD_SEQLEN);
      int v = nt;
#pragma unroll
      for (int o = 1; o < 32; o <<= 1) {
        const int u = __shfl_up_sync(kFull, v, o);
        if (lane >= o) v += u;
      }
      if (lane == 31) sh[warp] = v;
      __syncthreads();
      int base = before, all = 0;
      for (int w = 0; w < nw; ++w) {
        if (w < warp) base += sh[w];
        all += sh[w];
      }
      const int lo = base + v - nt;
      if (x >= lo && x < lo + nt) {
        sh[32] = b;
        sh[33] = lo + nt - 1 - x;
      }
      before += all;
      __syncthreads();
      if (before > x && blockIdx.x) break;   // block 0 checks every sequence
    }
    j.b = sh[32];
    if (j.b < 0) return false;
    j.s = load_seq(p, j.b, bad);
    tile = sh[33];
  }
  j.r0 = tile * kRows;
  j.rows = j.s.n * p.G;
  j.kvh = rest / a.splits;
  j.split = rest - j.kvh * a.splits;
  const int pos0 = j.s.S - j.s.n;
  const int last = min(j.r0 + kRows, j.rows) - 1;
  const int pmin = pos0 + static_cast<int>(fast_div(j.r0, a.div_g));
  // tokens [low, hi) are in the window of some row
  const int hi = max(0, pos0 + static_cast<int>(fast_div(last, a.div_g)) + 1);
  const int low = pmin >= p.window ? pmin - p.window + 1 : 0;
  const int first = low >> a.lR << a.lR;
  j.sinks = min(p.sinks, j.s.S);
  j.sink_keys = (j.sinks + a.R - 1) >> a.lR << a.lR;
  if (first <= j.sink_keys) {          // one range
    j.sink_keys = j.delta = 0;
    j.gap0 = min(j.sinks, low);
    j.gap1 = low;
  } else {
    j.delta = first - j.sink_keys;
    j.gap0 = j.sinks;
    j.gap1 = low - j.delta;
  }
  j.end = hi - j.delta;
  const int tiles = hi > 0 ? (j.end + kTN - 1) / kTN : 0;
  j.k0 = static_cast<int>(static_cast<long long>(tiles) * j.split / a.splits);
  j.k1 = static_cast<int>(static_cast<long long>(tiles) * (j.split + 1) / a.splits);
  return true;
}

template <typename T, int D, int NQ, Fetch kFetch>
__global__ void __launch_bounds__(TC<D, NQ>::kThreads, TC<D, NQ>::kCtas)
    prompt_tile_kernel(const __grid_constant__ CUtensorMap mk, const __grid_constant__ CUtensorMap mv,
                       const TileParams a) {
  using C = TC<D, NQ>;
  constexpr int kTN = C::kTN;
  extern __shared__ unsigned char smem_raw[];
  __shared__ __align__(8) uint64_t bars[C::kBars];
  __shared__ uint32_t s_tmem;
  __shared__ int s_find[34];
  const Params& p = a.p;
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;

  unsigned char* smem = reinterpret_cast<unsigned char*>(
      (reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
  const uint32_t sq = smem_u32(smem);
  const uint32_t skv = sq + NQ * C::kQTile;
  const uint32_t bar0 = smem_u32(bars);
  auto kv_full = [&](int s) { return bar0 + s * 8; };
  auto kv_empty = [&](int s) { return bar0 + (C::kSlots + s) * 8; };
  auto v_ready = [&](int i) { return bar0 + (2 * C::kSlots + i % C::kVBars) * 8; };   // i-th tile's
  const uint32_t bar1 = bar0 + (2 * C::kSlots + C::kVBars) * 8;
  auto q_full = [&](int t) { return bar1 + t * 8; };
  auto o_done = [&](int t) { return bar1 + (NQ + t) * 8; };
  auto drained = [&](int t) { return bar1 + (2 * NQ + t) * 8; };
  auto p_full = [&](int t, int half) { return bar1 + (3 * NQ + 2 * t + half) * 8; };
  auto turn = [&](int t) { return bar1 + (5 * NQ + t) * 8; };
  auto staged = [&](int t) { return bar1 + (6 * NQ + t) * 8; };
  auto s_full = [&](int i) { return bar1 + (7 * NQ + i) * 8; };
  if (threadIdx.x == 0) {
    for (int s = 0; s < C::kSlots; ++s) {
      mbar_init(kv_full(s), kFetch == Fetch::kPieces ? C::kProducers * 32 : C::kProducers);
      mbar_init(kv_empty(s), NQ);
    }
    for (int i = 0; i < C::kVBars; ++i) mbar_init(v_ready(i), 32);
    for (int t = 0; t < NQ; ++t) {
      mbar_init(q_full(t), 128);
      mbar_init(p_full(t, 0), 128);
      mbar_init(p_full(t, 1), 128);
      mbar_init(o_done(t), 1);
      mbar_init(drained(t), 1);
      mbar_init(turn(t), 1);
      mbar_init(staged(t), 128);
    }
    for (int i = 0; i < NQ * C::kSBufs; ++i) mbar_init(s_full(i), 1);
    asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
  }
  if (warp == NQ * 4) {
    asm volatile("tcgen05.alloc.cta_group::1.sync.aligned.shared::cta.b32 [%0], %1;" ::"r"(
                     smem_u32(&s_tmem)),
                 "n"(C::kTmemCols)
                 : "memory");
    asm volatile("tcgen05.relinquish_alloc_permit.cta_group::1.sync.aligned;");
  }
  tc_fence_before();
  // Dependent launch: from here on global memory is read.
  asm volatile("griddepcontrol.wait;" ::: "memory");
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  Job j;
  const bool found = find_job<D, NQ>(a, j, s_find);   // the same answer in every thread
  __syncthreads();
  tc_fence_after();
  const uint32_t tmem = s_tmem;
  if (!found) {
    if (warp == NQ * 4) tmem_free<C::kTmemCols>(tmem);
    return;
  }
  bool ok = true;

  if (warp >= NQ * 4) {
    if constexpr (C::kSplitRegs) regs_down<kOtherRegs>();
    if (warp >= NQ * 4 + NQ && warp < NQ * 4 + NQ + C::kProducers) {
      // ---------------------------------------------------------------- producer
      if constexpr (kFetch == Fetch::kPieces) {
        // Strides that are no whole numbers of rows: 16 bytes a thread and copy, to where a
        // box would put them. Up to kFly tiles' copies stay in flight per thread; a tile
        // is handed over when its own have landed (and the fence has made them visible to
        // the matrix pipe). 8192 tokens, window 4096, Hq32/Hkv8, pages of 1 and 4 tokens:
        // 1049 and 803 us, bound by the copies' address arithmetic beside the softmax
        // warps (as lists of rows both take 463, pages of 16 as boxes 363).
        constexpr int kPer = D / 8, kThr = C::kProducers * 32, kRows = kTN * kPer / kThr;
        constexpr int kFly = 2;
        static_assert(kThr % kPer == 0, "rows per pass");
        const int me = threadIdx.x - (NQ * 4 + NQ) * 32;
        const int c = me % kPer, first = me / kPer;
        const int bytes = c * 8 < a.dh ? 16 : 0;   // behind head_dim: zeros
        int s = 0, out = 0, fills = 0;          // slot to fill, slot to hand over next
        uint32_t phase = 0;
        auto hand_over = [&]() {
          fence_async_smem();
          mbar_arrive(kv_full(out));
          if (++out == C::kSlots) out = 0;
        };
        for (int k = j.k0; k < j.k1 && ok; ++k) {
          int page[kRows];
#pragma unroll
          for (int i = 0; i < kRows; ++i) {
            const int key = k * kTN + first + i * (kThr / kPer);
            page[i] = -1;
            if (key < j.end && !(key >= j.gap0 && key < j.gap1)) {
              const int tok = key < j.sink_keys ? key : key + j.delta;
              page[i] = __ldg(p.bt + j.b * p.bt_sb + static_cast<int>(fast_div(tok, a.div_bs)));
              if (page[i] < 0 || page[i] >= p.NB) {
                flag(p, PA_STATUS_BAD_BLOCK);
                page[i] = -1;
              }
            }
          }
          for (int kv = 0; kv < 2; ++kv) {
            ok = __all_sync(kFull, mbar_wait(kv_empty(s), phase ^ 1));
            if (!ok) break;
            const char* base = (kv ? p.vc + j.kvh * p.v_sh : p.kc + j.kvh * p.k_sh) + c * bytes;
            const long long sb = kv ? p.v_sb : p.k_sb, ss = kv ? p.v_ss : p.k_ss;
#pragma unroll
            for (int i = 0; i < kRows; ++i) {
              const int r = first + i * (kThr / kPer);
              if (page[i] < 0) continue;
              const int key = k * kTN + r;
              const int tok = key < j.sink_keys ? key : key + j.delta;
              const int slot = tok - static_cast<int>(fast_div(tok, a.div_bs)) * p.bs;
              asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                               skv + s * C::kKV + (c >> 3) * kTN * 128 + r * 128 +
                               (((c & 7) ^ (r & 7)) << 4)),
                           "l"(base + page[i] * sb + slot * ss), "r"(bytes)
                           : "memory");
            }
            asm volatile("cp.async.commit_group;" ::: "memory");
            if (++s == C::kSlots) {
              s = 0;
              phase ^= 1;
            }
            if (++fills > kFly) {
              asm volatile("cp.async.wait_group %0;" ::"n"(kFly) : "memory");
              hand_over();
            }
          }
        }
        asm volatile("cp.async.wait_all;" ::: "memory");   // also where a wait gave up
        for (int left = min(fills, kFly); left > 0; --left) hand_over();
      } else if constexpr (kFetch == Fetch::kRows) {
        // A copy is four keys' rows of one 64-dim chunk; the lanes share them out as
        // they do boxes. The four keys' tokens follow each other, their pages do not. A
        // key of them that no row sees brings a visible one's row. 128 copies a tile at
        // 25 to 40 cycles each bound it where boxes of 16 rows wait for S and P (8192
        // tokens, Hq32/Hkv8: window 4096 463 us against 363; head_dim 64, no window 611
        // against 401).
        const int f = lane * C::kProducers + warp - (NQ * 4 + NQ);
        const int group = f / C::kChunks, chunk = f - group * C::kChunks;
        auto visible = [&](int key) {
          return group < kTN / 4 && key < j.end && !(key >= j.gap0 && key < j.gap1);
        };
        auto lookup = [&](int k, int (&page)[4]) {
          const int key = k * kTN + group * 4;
          const int tok = key < j.sink_keys ? key : key + j.delta;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            page[i] = INT_MIN;
            if (visible(key + i))
              page[i] = __ldg(p.bt + j.b * p.bt_sb + static_cast<int>(fast_div(tok + i, a.div_bs)));
          }
        };
        int page[4], next[4], s = 0;
        uint32_t phase = 0;
        if (j.k0 < j.k1) lookup(j.k0, next);
        for (int k = j.k0; k < j.k1 && ok; ++k) {
          const int key = k * kTN + group * 4;
          const int tok = key < j.sink_keys ? key : key + j.delta;
          int slot[4], have = -1;
#pragma unroll
          for (int i = 0; i < 4; ++i) {
            page[i] = next[i];
            slot[i] = tok + i - static_cast<int>(fast_div(tok + i, a.div_bs)) * p.bs;
            if (page[i] != INT_MIN && (page[i] < 0 || page[i] >= p.NB)) {
              flag(p, PA_STATUS_BAD_BLOCK);
              page[i] = INT_MIN;
            }
            if (page[i] != INT_MIN) have = i;
          }
          if (k + 1 < j.k1) lookup(k + 1, next);
          const bool valid = have >= 0;
          const uint32_t bytes = __popc(__ballot_sync(kFull, valid)) * 4 * 128;
          for (int kv = 0; kv < 2; ++kv) {
            ok = __all_sync(kFull, mbar_wait(kv_empty(s), phase ^ 1));
            if (!ok) break;
            if (lane == 0) mbar_expect_tx(kv_full(s), bytes);
            __syncwarp();
            if (valid) {
              int row[4], some = 0;
#pragma unroll
              for (int i = 0; i < 4; ++i) {
                row[i] = page[i] * a.row_b[kv] + slot[i] * a.row_s[kv] + j.kvh * a.row_h[kv];
                if (i == have) some = row[i];
              }
#pragma unroll
              for (int i = 0; i < 4; ++i)
                if (page[i] == INT_MIN) row[i] = some;
              tma_load_rows(skv + s * C::kKV + chunk * kTN * 128 + group * 512, kv ? &mv : &mk,
                            chunk * 64, row[0], row[1], row[2], row[3], kv_full(s));
            }
            if (++s == C::kSlots) {
              s = 0;
              phase ^= 1;
            }
          }
        }
        if (!ok) {
          // leave no copy in flight (as below)
          for (int i = 0; i < C::kSlots; ++i) mbar_wait(kv_full(i), i < s ? phase : phase ^ 1);
        }
      } else {
      // A box is R token rows of one 64-dim chunk; lane l of producer w has box
      // l * kProducers + w. (A box takes ~60 cycles to set off, whichever lane does
      // it: one warp for all 64 boxes of a tile with pages of 16 tokens kept the
      // products waiting, 434 us where pages of 32 took 393.)
      const int f = lane * C::kProducers + warp - (NQ * 4 + NQ);
      const int box = f / C::kChunks, chunk = f - box * C::kChunks;
      auto lookup = [&](int k, int& phys, int& slot) {
        phys = INT_MIN;
        slot = 0;
        const int key = k * kTN + (box << a.lR);
        // a box in which no row sees a token is not read
        if (box < (kTN >> a.lR) && key < j.end && !(key >= j.gap0 && key + a.R <= j.gap1)) {
          const int tok = key < j.sink_keys ? key : key + j.delta;
          const int pg = a.bs_log2 >= 0 ? tok >> a.bs_log2 : static_cast<int>(fast_div(tok, a.div_bs));
          slot = tok - pg * p.bs;
          phys = __ldg(p.bt + j.b * p.bt_sb + pg);
        }
      };
      int phys, slot, nphys = INT_MIN, nslot = 0, s = 0;
      uint32_t phase = 0;
      if (j.k0 < j.k1) lookup(j.k0, nphys, nslot);
      for (int k = j.k0; k < j.k1 && ok; ++k) {
        phys = nphys;
        slot = nslot;
        if (k + 1 < j.k1) lookup(k + 1, nphys, nslot);
        bool valid = phys != INT_MIN;
        if (valid && (phys < 0 || phys >= p.NB)) {
          flag(p, PA_STATUS_BAD_BLOCK);
          valid = false;
        }
        const uint32_t bytes = __popc(__ballot_sync(kFull, valid)) * a.R * 128;
        for (int kv = 0; kv < 2; ++kv) {
          ok = mbar_wait(kv_empty(s), phase ^ 1);
          if (!__all_sync(kFull, ok)) {
            ok = false;
            break;
          }
          if (lane == 0) mbar_expect_tx(kv_full(s), bytes);
          __syncwarp();
          if (valid)
            tma_load_5d(skv + s * C::kKV + chunk * kTN * 128 + (box << a.lR) * 128, kv ? &mv : &mk, 0,
                        slot, chunk, j.kvh, phys, kv_full(s));
          if (++s == C::kSlots) {
            s = 0;
            phase ^= 1;
          }
        }
      }
      if (!ok) {
        // leave no copy in flight: every slot's last fill (a slot that was never
        // filled passes as the phase before its first)
        for (int i = 0; i < C::kSlots; ++i) mbar_wait(kv_full(i), i < s ? phase : phase ^ 1);
      }
      }
    }
    if (warp == NQ * 4 + NQ + C::kProducers) {
      // ----------------------------------------------------------------- cleaner
      // Hands each V tile on to the issuing warps, after zeroing the rows of its
      // multiplied 16-token steps whose tokens no row sees.
      int s = 0;
      uint32_t phase = 0;
      for (int k = j.k0; k < j.k1; ++k) {
        if (++s == C::kSlots) {      // past the K tile
          s = 0;
          phase ^= 1;
        }
        ok = __all_sync(kFull, mbar_wait(kv_full(s), phase));
        if (!ok) break;
        const KeyTile kt = key_tile<kTN>(j, k);
        const int v0 = kt.from - kt.base, v1 = kt.to - kt.base;
        const int c0 = v0 & ~15, c1 = (v1 + 15) & ~15;
        const int g0 = j.gap0 - kt.base, g1 = j.gap1 - kt.base;
        if (v0 != c0 || v1 != c1 || (g0 < c1 && g1 > c0 && g0 < g1)) {
          constexpr int kRowsAtOnce = D / 8 < 32 ? 32 / (D / 8) : 1;
          const int c = lane % (D / 8);
          for (int r = c0 + lane / (D / 8); r < c1; r += kRowsAtOnce) {
            if (r >= v0 && r < v1 && !(r >= g0 && r < g1)) continue;
            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(
                             skv + s * C::kKV + (c >> 3) * kTN * 128 + r * 128 + (c & 7) * 16),
                         "r"(0)
                         : "memory");
          }
          fence_async_smem();
        }
        mbar_arrive(v_ready(k - j.k0));
        if (++s == C::kSlots) {
          s = 0;
          phase ^= 1;
        }
      }
      if (!ok && lane == 0) flag(p, PA_STATUS_TIMEOUT);
    }
    if (warp < NQ * 4 + NQ) {
      // -------------------------------------------------------------- issuing warps
      // One lane per row tile issues its products. What it runs between them
      // bounds the kernel (the softmax warps take most issue slots: a wait on a
      // barrier that is already complete costs ~100-200 cycles, a matrix
      // instruction of 64 cycles' work ~70): with one warp for both row tiles, whole-
      // warp waits and descriptors rebuilt per instruction, 8192 tokens, window
      // 4096, Hq32/Hkv8 took 417 us. So: a warp per row tile, a single lane, the
      // next keys' wait ahead of P's, no wait between the two products.
      if (elect_one()) {
        const int t = warp - NQ * 4;
        const int n = j.k1 - j.k0;
        constexpr uint32_t kDescPV = instr_desc<T>(D, true);
        constexpr uint32_t kStep = C::kKV >> 4;
        const uint32_t q_desc = smem_desc(sq + t * C::kQTile, 16);
        const uint32_t k_desc = smem_desc(skv, 16);
        const uint32_t v_desc = smem_desc(skv, kTN * 128);
        const uint32_t o_col = tmem + C::kOCol + t * D;
        const uint32_t s_col = tmem + t * C::kSBufs * kTN;
        // S from the keys in slot ks
        auto issue_s = [&](int buf, int ks, const KeyTile& kt) {
          const uint32_t idesc = instr_desc<T>((kt.to - kt.base + 15) & ~15, false);
          const uint32_t kb = k_desc + ks * kStep;
#pragma unroll
          for (int i = 0; i < D / 16; ++i)
            mma_ss(s_col + buf * kTN, q_desc + ((i >> 2) * 128 * 128 + (i & 3) * 32) / 16,
                   kb + ((i >> 2) * kTN * 128 + (i & 3) * 32) / 16, idesc, i > 0);
          tc_commit(s_full(t * C::kSBufs + buf));
        };
        // O += P V over one half of the tile's 16-token steps, values in slot vs
        auto issue_o = [&](int buf, int vs, const KeyTile& kt, int half, bool add) {
          constexpr int kHalf = kTN / 32;
          const uint32_t pa = s_col + buf * kTN;
          const uint32_t vb = v_desc + vs * kStep;
          const int i0 = (kt.from - kt.base) >> 4, i1 = (kt.to - kt.base + 15) >> 4;
          if (i0 == 0 && i1 == kTN / 16) {
#pragma unroll
            for (int i = 0; i < kHalf; ++i)
              mma_ts(o_col, pa + (half * kHalf + i) * 8, vb + (half * kHalf + i) * (16 * 128 / 16),
                     kDescPV, i > 0 || half || add);
          } else {
            const int e = min(i1, (half + 1) * kHalf);
            for (int i = max(i0, half * kHalf); i < e; ++i)
              mma_ts(o_col, pa + i * 8, vb + i * (16 * 128 / 16), kDescPV, i > i0 || add);
          }
        };
        auto wait = [&](uint32_t bar, uint32_t parity) {
          if (ok) ok = mbar_wait(bar, parity);
          return ok;
        };
        // Tile i's keys are fill 2 i of the ring, its values fill 2 i + 1.
        int ks = 0, vs = 1;
        uint32_t kph = 0;
        KeyTile cur = key_tile<kTN>(j, j.k0);
        // The two row tiles' (P V, next S) blocks alternate on the pipe: mixed, both
        // would be ready late, and the softmax warps of both would first wait and
        // then run at the same time.
        auto my_turn = [&](int block) {
          return NQ == 1 || (t == 0 && block == 0) || wait(turn(t), (t == 0 ? block - 1 : block) & 1);
        };
        auto pass_turn = [&]() {
          if (NQ == 2) mbar_arrive(turn(1 - t));
        };
        if (n > 0 && wait(q_full(t), 0) && wait(kv_full(0), 0) && my_turn(0)) {
          issue_s(0, 0, cur);
          if (n > 1) tc_commit(kv_empty(0));
          pass_turn();
        }
        for (int i = 0; i < n && ok; ++i) {
          const bool more = i + 1 < n;
          const KeyTile nxt = key_tile<kTN>(j, j.k0 + i + (more ? 1 : 0));
          ks += 2;
          if (ks >= C::kSlots) {
            ks -= C::kSlots;
            kph ^= 1;
          }
          if (more && !wait(kv_full(ks), kph)) break;
          if (C::kSBufs == 2 && more) {
            // the next tile's S, into the other buffer, during this tile's softmax
            issue_s((i + 1) & 1, ks, nxt);
            if (i + 2 < n) tc_commit(kv_empty(ks));
          }
          const int buf = C::kSBufs == 2 ? i & 1 : 0;
          if (!wait(v_ready(i), i / C::kVBars & 1) || !wait(p_full(t, 0), i & 1)) break;
          tc_fence_after();
          issue_o(buf, vs, cur, 0, i > 0);
          if (!my_turn(i + 1) || !wait(p_full(t, 1), i & 1)) break;
          tc_fence_after();
          issue_o(buf, vs, cur, 1, i > 0);
          if (C::kSBufs == 2 || !more) tc_commit(o_done(t));
          if (C::kSBufs == 1 && more) {
            issue_s(0, ks, nxt);
            if (i + 2 < n) tc_commit(kv_empty(ks));
          }
          pass_turn();
          if (more) tc_commit(kv_empty(vs));
          vs += 2;
          if (vs >= C::kSlots) vs -= C::kSlots;
          cur = nxt;
        }
        if (!ok) {
          flag(p, PA_STATUS_TIMEOUT);
          tc_commit(drained(t));
          mbar_wait(drained(t), 0);
        }
      }
      __syncwarp();
    }
  } else {
    // ----------------------------------------------------------------- softmax
    if constexpr (C::kSplitRegs) regs_up<kSoftmaxRegs>();
    const int t = warp >> 2;
    const int tid = threadIdx.x & 127;
    const int r0 = j.r0 + t * 128;
    if (j.k0 < j.k1) {
      // the row tile into shared memory: 16-byte pieces, D/8 threads a row. (Not for rows
      // that see nothing: no product would wait for these copies, and the output takes
      // their place.)
      constexpr int kPer = D / 8;
      const int c = tid % kPer;
#pragma unroll
      for (int i = 0; i < kPer; ++i) {
        const int r = i * (128 / kPer) + tid / kPer;
        const int pr = r0 + r;
        const bool in = pr < j.rows && c * 8 < a.dh;
        const int tok = in ? static_cast<int>(fast_div(pr, a.div_g)) : 0;
        const char* src = in ? p.q + (j.s.start + tok) * p.q_st + (j.kvh * p.G + pr - tok * p.G) * p.q_sh + c * 16
                             : p.q;
        // asynchronous, past the first-level cache (which shared memory leaves
        // smaller than the tile); rows behind the sequence, and dimensions behind
        // head_dim, become zero
        asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(
                         sq + t * C::kQTile + (c >> 3) * 128 * 128 + r * 128 +
                         (((c & 7) ^ (r & 7)) << 4)),
                     "l"(src), "r"(in ? 16 : 0)
                     : "memory");
      }
      asm volatile("cp.async.wait_all;" ::: "memory");
      fence_async_smem();
      mbar_arrive(q_full(t));
    }
    const int pr = r0 + tid;
    const bool live = pr < j.rows;
    const int tok = live ? static_cast<int>(fast_div(pr, a.div_g)) : 0;
    const int pos = j.s.S - j.s.n + tok;
    // the row sees keys v < hi with v >= low or v < sinks (its tokens t <= pos with
    // t > pos - window or t < sinks; behind sinks of their own, delta keys are left out)
    const int hi = live ? max(pos + 1 - j.delta, 0) : 0;
    const int low = (pos >= p.window ? pos - p.window + 1 : 0) - j.delta;
    const float scl = p.scale_log2;
    const uint32_t lanes = static_cast<uint32_t>(warp & 3) << 21;   // TMEM lane 32 * (warp % 4)
    const uint32_t o_at = tmem + lanes + C::kOCol + t * D;
    float m = -INFINITY, l = 0.f;                 // of finite scores
    const int n = j.k1 - j.k0;
    // Two S buffers: waits for the product of tile i - 1, once per tile and before tile i's
    // P is handed over, so that no barrier here gets a phase ahead of its reader.
    int waited = 0;
    auto o_free = [&](int i) {
      if (C::kSBufs == 1 || waited == i) return true;
      ok = mbar_wait(o_done(t), (i - 1) & 1);
      ok = __all_sync(kFull, ok);
      tc_fence_after();
      waited = i;
      return ok;
    };
    for (int i = 0; i < n; ++i) {
      const int buf = C::kSBufs == 2 ? (i & 1) : 0;
      const uint32_t s_at = tmem + lanes + (t * C::kSBufs + buf) * kTN;
      ok = mbar_wait(s_full(t * C::kSBufs + buf), C::kSBufs == 2 ? (i >> 1) & 1 : i & 1);
      if (!__all_sync(kFull, ok)) {
        ok = false;
        break;
      }
      tc_fence_after();
      const int base = key_tile<kTN>(j, j.k0 + i).base;
      uint32_t raw[kTN];
      tmem_ld(s_at, raw);
      float s[kTN];
#pragma unroll
      for (int c = 0; c < kTN; ++c) s[c] = __uint_as_float(raw[c]);
      if (__any_sync(kFull, hi < base + kTN || low > base)) {
        const int h = hi - base, lo = low - base, sk = j.sinks - base;
#pragma unroll
        for (int c0 = 0; c0 < kTN; c0 += 32) {
          // 32 columns' visibility as one word
          const uint32_t seen = ones_below(h - c0) & (~ones_below(lo - c0) | ones_below(sk - c0));
          if (__any_sync(kFull, ~seen)) {
#pragma unroll
            for (int c = 0; c < 32; ++c)
              s[c0 + c] = seen & 1u << c ? s[c0 + c] : -INFINITY;
          }
        }
      }
      float mx[4] = {s[0], s[1], s[2], s[3]};
#pragma unroll
      for (int c = 4; c + 7 < kTN; c += 8) {
#pragma unroll
        for (int e = 0; e < 4; ++e) mx[e] = max3(mx[e], s[c + 2 * e], s[c + 2 * e + 1]);
      }
      const float top = max3(max3(mx[0], mx[1], mx[2]), max3(mx[3], s[kTN - 4], s[kTN - 3]),
                             max_nan(s[kTN - 2], s[kTN - 1]));
      // a score of NaN or infinity leaves no number (the exponentials on the FMA pipe
      // would): the sum carries it
      if (!(top < INFINITY)) l = kNaN;
      if (i == 0) {
        m = top;
      } else if (__any_sync(kFull, (top - m) * scl > kRescaleLog2)) {
        // (the difference is NaN, not greater, while the row has seen nothing)
        const float mn = fmaxf(m, top);
        const float f = mn == -INFINITY ? 1.f : ex2((m - mn) * scl);
        m = mn;
        l *= f;
        // O is free once the previous tile's product is done (with one S buffer the
        // commit behind this tile's S covers it)
        if (!o_free(i)) break;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          tmem_ld(o_at + c, o);
#pragma unroll
          for (int e = 0; e < 32; ++e) o[e] = __float_as_uint(__uint_as_float(o[e]) * f);
          tmem_st(o_at + c, o);
        }
      }
      const float off = m == -INFINITY ? 0.f : -m * scl;
      const uint64_t scl2 = f2(scl, scl), off2 = f2(off, off);
      uint64_t sum[2] = {f2(0.f, 0.f), f2(0.f, 0.f)};
      bool stop = false;
#pragma unroll
      for (int half = 0; half < 2; ++half) {
#pragma unroll
        for (int c0 = half * (kTN / 2); c0 < (half + 1) * (kTN / 2); c0 += 32) {
          uint32_t pk[16];
#pragma unroll
          for (int c = 0; c < 32; c += 2) {
            const uint64_t v = f2_fma(f2(s[c0 + c], s[c0 + c + 1]), scl2, off2);
            float x, y;
            // A quarter on the FMA pipe: 8192 tokens, Hq32/Hkv8, window 4096: 372 us
            // against 388 without and 414 with 3 of 8 (issue slots run out and
            // registers spill); head_dim 64, no window: 411, 445, 453.
            if ((c & 7) == 4) {
              ex2_pair_fma(v, x, y);
            } else {
              f2_split(v, x, y);
              x = ex2(x);
              y = ex2(y);
            }
            sum[(c >> 1) & 1] = f2_add(sum[(c >> 1) & 1], f2(x, y));
            pk[c / 2] = pack2<T>(x, y);
          }
          tmem_st(s_at + c0 / 2, pk);
        }
        asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory");
        if (half == 0 && !o_free(i)) {
          stop = true;
          break;
        }
        // the first half's product may start while the second half is formed
        tc_fence_before();
        mbar_arrive(p_full(t, half));
      }
      if (stop) break;
      float x0, x1, x2, x3;
      f2_split(sum[0], x0, x1);
      f2_split(sum[1], x2, x3);
      l += (x0 + x1) + (x2 + x3);
    }
    if (n > 0 && ok) {
      ok = mbar_wait(o_done(t), C::kSBufs == 2 ? (n - 1) & 1 : 0);
      ok = __all_sync(kFull, ok);
      tc_fence_after();
    }
    if (!ok) {
      if (lane == 0) flag(p, PA_STATUS_TIMEOUT);
    } else {
      const float inv = l == 0.f ? 0.f : 1.f / l;
      const float lse = l == 0.f ? kSentinel : (m * scl + log2f(l)) * kLn2;
      const int hq = j.kvh * p.G + pr - tok * p.G;
      const long long at = static_cast<long long>(j.s.start + tok) * p.Hq + hq;
      if (a.splits == 1) {
        // Through shared memory (the row tile's queries are no longer needed), so that
        // whole rows leave in one piece: 16-byte pieces, XOR-spread over the banks.
        constexpr int kPer = D / 8;
        const uint32_t so = sq + t * C::kQTile;
#pragma unroll 1
        for (int c = 0; c < D; c += 32) {
          uint32_t o[32];
          if (n > 0) {
            tmem_ld(o_at + c, o);
          } else {
#pragma unroll
            for (int e = 0; e < 32; ++e) o[e] = 0;
          }
#pragma unroll
          for (int e = 0; e < 32; e += 8) {
            uint32_t w[4];
#pragma unroll
            for (int x = 0; x < 4; ++x)
              w[x] = pack2<T>(__uint_as_float(o[e + 2 * x]) * inv,
                              __uint_as_float(o[e + 2 * x + 1]) * inv);
            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(
                             so + tid * (D * 2) + ((((c + e) >> 3) ^ (tid & 7)) << 4)),
                         "r"(w[0]), "r"(w[1]), "r"(w[2]), "r"(w[3])
                         : "memory");
          }
        }
        mbar_arrive(staged(t));
        ok = __all_sync(kFull, mbar_wait(staged(t), 0));   // bounded, unlike a named barrier
        if (!ok && lane == 0) flag(p, PA_STATUS_TIMEOUT);
        const int c = tid % kPer;
#pragma unroll 4
        for (int i = 0; i < kPer; ++i) {
          const int r = i * (128 / kPer) + tid / kPer;
          const int q = r0 + r;
          if (ok && q < j.rows && c * 8 < a.dh) {
            const int qt = static_cast<int>(fast_div(q, a.div_g));
            uint4 v;
            asm volatile("ld.shared.v4.b32 {%0, %1, %2, %3}, [%4];"
                         : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w)
                         : "r"(so + r * (D * 2) + ((c ^ (r & 7)) << 4)));
            *(reinterpret_cast<uint4*>(p.out + (j.s.start + qt) * p.o_st +
                                       (j.kvh * p.G + q - qt * p.G) * p.o_sh) + c) = v;
          }
        }
        if (live && p.lse) p.lse[at] = lse;
      } else {
        const long long row = static_cast<long long>(j.split) * p.T * p.Hq + at;
        if (n > 0) {
          float* dst = a.o_part + row * D;
#pragma unroll 1
          for (int c = 0; c < D; c += 32) {
            uint32_t o[32];
            tmem_ld(o_at + c, o);
            if (live) {
#pragma unroll
              for (int e = 0; e < 32; e += 4)
                *reinterpret_cast<float4*>(dst + c + e) =
                    make_float4(__uint_as_float(o[e]) * inv, __uint_as_float(o[e + 1]) * inv,
                                __uint_as_float(o[e + 2]) * inv, __uint_as_float(o[e + 3]) * inv);
            }
          }
        }
        if (live) a.lse_part[row] = n > 0 ? lse : kSentinel;
      }
    }
  }
  tc_fence_before();
  __syncthreads();
  tc_fence_after();
  if (warp == NQ * 4) tmem_free<C::kTmemCols>(tmem);
}

// Joins the splits of a row: one warp per (row, query head), weights
// 2^(lse - max) over the splits that saw a token.
template <typename T, int D>
__global__ void __launch_bounds__(128) prompt_join_kernel(const TileParams a) {
  constexpr int N = D / 32;
  const Params& p = a.p;
  const int lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 4 + (threadIdx.x >> 5);
  const long long rows = static_cast<long long>(p.T) * p.Hq;
  if (w >= rows) return;
  const int row = static_cast<int>(w / p.Hq);
  const int hq = static_cast<int>(w - static_cast<long long>(row) * p.Hq);
  asm volatile("griddepcontrol.wait;" ::: "memory");   // the splits' partials
  asm volatile("griddepcontrol.launch_dependents;" ::: "memory");
  if (seq_of_row(p, row) < 0) return;
  // lane = split: its weight, then all splits' rows in flight together
  float sum = 0.f, acc[N], top = -INFINITY;
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int k0 = 0; k0 < a.splits; k0 += 32) {
    const float l = k0 + lane < a.splits ? __ldcg(a.lse_part + (k0 + lane) * rows + w) : kSentinel;
    if (__all_sync(kFull, l <= -1e29f)) continue;      // these splits saw nothing (NaN is something)
    float t = l;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(kFull, t, o));
    t = fmaxf(t, top);
    const float old = exp2f((top - t) * kLog2e);
    top = t;
    sum *= old;
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= old;
    const float mine = l <= -1e29f ? 0.f : exp2f((l - top) * kLog2e);
    const int cnt = min(32, a.splits - k0);
#pragma unroll 4
    for (int k = 0; k < cnt; ++k) {
      const float f = __shfl_sync(kFull, mine, k);
      if (f != 0.f) {                                  // (an empty split has no row)
        const float* src = a.o_part + ((k0 + k) * rows + w) * D + lane * N;
        sum += f;
#pragma unroll
        for (int i = 0; i < N; ++i) acc[i] = fmaf(f, __ldcg(src + i), acc[i]);
      }
    }
  }
  const float inv = sum == 0.f ? 0.f : 1.f / sum;
  uint32_t* dst = reinterpret_cast<uint32_t*>(p.out + row * p.o_st + hq * p.o_sh + lane * N * 2);
#pragma unroll
  for (int i = 0; i < N / 2; ++i)
    if (lane * N < a.dh) dst[i] = pack2<T>(acc[2 * i] * inv, acc[2 * i + 1] * inv);
  if (lane == 0 && p.lse) p.lse[w] = sum == 0.f ? kSentinel : top + logf(sum);
}

// ----------------------------------------------------------------------------
// Host side
// ----------------------------------------------------------------------------
static bool aligned16(const void* ptr) { return (reinterpret_cast<uintptr_t>(ptr) & 15) == 0; }

static pa_status_t validate(const pa_prompt_params* p) {
  if (!p) return PA_ERR_ARG;
  if (p->num_tokens < 0 || p->batch < 0 || p->num_heads <= 0 || p->num_kv_heads <= 0 ||
      p->block_size <= 0 || p->num_blocks <= 0 || p->max_blocks < 0)
    return PA_ERR_ARG;
  if (p->num_heads % p->num_kv_heads != 0) return PA_ERR_ARG;
  if (p->dtype != PA_F16 && p->dtype != PA_BF16) return PA_ERR_ARG;
  if (!(p->scale > 0.f) || p->scale > 1e30f) return PA_ERR_ARG;
  if (p->window < 0 || p->num_sinks < 0 || (p->window == 0 && p->num_sinks != 0))
    return PA_ERR_ARG;
  if (p->num_splits < 0) return PA_ERR_ARG;
  if (p->head_dim != 32 && p->head_dim != 64 && p->head_dim != 128 && p->head_dim != 256)
    return PA_ERR_UNSUPPORTED;
  if (p->block_size > (1 << 20)) return PA_ERR_UNSUPPORTED;
  // tokens of a table, and packed (token, head) rows of a batch, are counted in int32
  if (static_cast<long long>(p->max_blocks) * p->block_size > 0x7fffff00ll ||
      static_cast<long long>(p->num_tokens) * p->num_heads > 0x3fffffffll)
    return PA_ERR_UNSUPPORTED;
  return PA_OK;
}

static pa_status_t validate_launch(const pa_prompt_params* p) {
  if (!p->q || !p->k_cache || !p->v_cache || !p->block_table || !p->query_starts || !p->seq_lens ||
      !p->out)
    return PA_ERR_ARG;
  if (!aligned16(p->q) || !aligned16(p->k_cache) || !aligned16(p->v_cache) || !aligned16(p->out))
    return PA_ERR_ARG;
  const int64_t strides[10] = {p->q_stride_t,    p->q_stride_h,    p->out_stride_t,
                               p->out_stride_h,  p->k_stride_block, p->k_stride_slot,
                               p->k_stride_head, p->v_stride_block, p->v_stride_slot,
                               p->v_stride_head};
  for (int i = 0; i < 10; ++i)
    if (strides[i] % 8) return PA_ERR_ARG;
  return PA_OK;
}

static Params make_params(const pa_prompt_params* p) {
  Params a;
  memset(&a, 0, sizeof(a));
  a.q = static_cast<const char*>(p->q);
  a.q_st = p->q_stride_t * 2;
  a.q_sh = p->q_stride_h * 2;
  a.kc = static_cast<const char*>(p->k_cache);
  a.vc = static_cast<const char*>(p->v_cache);
  a.k_sb = p->k_stride_block * 2;
  a.k_ss = p->k_stride_slot * 2;
  a.k_sh = p->k_stride_head * 2;
  a.v_sb = p->v_stride_block * 2;
  a.v_ss = p->v_stride_slot * 2;
  a.v_sh = p->v_stride_head * 2;
  a.bt = p->block_table;
  a.bt_sb = p->bt_stride_b;
  a.max_blocks = p->max_blocks;
  a.starts = p->query_starts;
  a.lens = p->seq_lens;
  a.T = p->num_tokens;
  a.B = p->batch;
  a.Hq = p->num_heads;
  a.Hkv = p->num_kv_heads;
  a.G = p->num_heads / p->num_kv_heads;
  a.bs = p->block_size;
  a.NB = p->num_blocks;
  a.window = p->window ? p->window : 0x7fffffff;
  a.sinks = p->num_sinks;
  a.scale_log2 = p->scale * kLog2e;
  a.out = static_cast<char*>(p->out);
  a.o_st = p->out_stride_t * 2;
  a.o_sh = p->out_stride_h * 2;
  a.lse = p->lse;
  a.status = p->status;
  return a;
}

static PFN_cuTensorMapEncodeTiled_v12000 encode_fn() {
  static PFN_cuTensorMapEncodeTiled_v12000 fn = nullptr;
  static std::once_flag once;
  std::call_once(once, [] {
    void* ptr = nullptr;
    cudaDriverEntryPointQueryResult q;
    if (cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &ptr, cudaEnableDefault, &q) ==
            cudaSuccess &&
        q == cudaDriverEntryPointSuccess)
      fn = reinterpret_cast<PFN_cuTensorMapEncodeTiled_v12000>(ptr);
  });
  return fn;
}

// Dimensions of a row in the kernel that takes it: head_dim 32 runs as 64, the upper
// half zero.
static int kernel_dim(const pa_prompt_params* p) { return std::max(64, p->head_dim); }

// A paged cache as (64 dims, slot, 64-dim chunk, head, page); a box is R token
// rows of one chunk, 128-byte swizzled. Of a head_dim of 32 the box's upper half lies
// outside the first extent and is filled with zeros.
static bool encode_map(CUtensorMap* map, const pa_prompt_params* p, const void* base,
                       int64_t s_block, int64_t s_slot, int64_t s_head, int R) {
  auto fn = encode_fn();
  if (!fn) return false;
  const CUtensorMapDataType dt =
      p->dtype == PA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t dims[5] = {static_cast<cuuint64_t>(std::min(64, p->head_dim)),
                              static_cast<cuuint64_t>(p->block_size),
                              static_cast<cuuint64_t>(kernel_dim(p) / 64),
                              static_cast<cuuint64_t>(p->num_kv_heads),
                              static_cast<cuuint64_t>(p->num_blocks)};
  const cuuint64_t strides[4] = {static_cast<cuuint64_t>(s_slot) * 2, 128,
                                 static_cast<cuuint64_t>(s_head) * 2,
                                 static_cast<cuuint64_t>(s_block) * 2};
  const cuuint32_t box[5] = {64, static_cast<cuuint32_t>(R), 1, 1, 1};
  const cuuint32_t step[5] = {1, 1, 1, 1, 1};
  return fn(map, dt, 5, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// A paged cache as rows of D dimensions, `unit` elements from one to the next, for
// caches whose strides are whole numbers of rows; a copy takes four rows of 64.
struct RowList {
  int64_t unit, rows;
  int b, s, h;              // rows from a page, slot, head to the next
};
static bool row_list(const pa_prompt_params* p, int64_t s_block, int64_t s_slot, int64_t s_head,
                     RowList* r) {
  const int64_t sb = p->num_blocks > 1 ? s_block : 0, ss = p->block_size > 1 ? s_slot : 0,
                sh = p->num_kv_heads > 1 ? s_head : 0;
  if (sb < 0 || ss < 0 || sh < 0) return false;
  int64_t u = std::gcd(std::gcd(sb, ss), sh);
  if (u == 0) u = p->head_dim;
  if (p->head_dim < 64 || u < p->head_dim || u >= (1ll << 38)) return false;
  r->unit = u;
  r->rows = (p->num_blocks - 1) * (sb / u) + (p->block_size - 1) * (ss / u) +
            (p->num_kv_heads - 1) * (sh / u) + 1;
  if (r->rows > 0x7fffffffll) return false;
  r->b = static_cast<int>(sb / u);
  r->s = static_cast<int>(ss / u);
  r->h = static_cast<int>(sh / u);
  return true;
}
static bool encode_rows(CUtensorMap* map, const pa_prompt_params* p, const void* base,
                        const RowList& r) {
  auto fn = encode_fn();
  if (!fn) return false;
  const CUtensorMapDataType dt =
      p->dtype == PA_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16;
  const cuuint64_t dims[2] = {static_cast<cuuint64_t>(p->head_dim), static_cast<cuuint64_t>(r.rows)};
  const cuuint64_t strides[1] = {static_cast<cuuint64_t>(r.unit) * 2};
  const cuuint32_t box[2] = {64, 1};
  const cuuint32_t step[2] = {1, 1};
  return fn(map, dt, 2, const_cast<void*>(base), dims, strides, box, step,
            CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B,
            CU_TENSOR_MAP_L2_PROMOTION_L2_128B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE) == CUDA_SUCCESS;
}

// How a call runs: row tiles of 128 * nq, the keys in `splits` parts.
struct Plan {
  int nq, splits;
  long long tiles;          // bound on the row tiles of a KV head
  size_t ws_bytes;
};
static Plan make_plan(const pa_prompt_params* p, int sms) {
  Plan pl = {};
  pl.splits = 1;
  const int g = p->num_heads / p->num_kv_heads;
  const long long packed = static_cast<long long>(p->num_tokens) * g;   // rows of a KV head
  // Two row tiles per CTA keep the matrix pipe busy; a batch whose sequences
  // bring no more than one tile each would leave the second empty.
  pl.nq = p->head_dim == 256 || p->head_dim <= 64 || packed <= 128ll * p->batch ? 1 : 2;
  const long long slots = static_cast<long long>(sms) * (p->head_dim <= 64 ? 2 : 1);   // CTAs at once
  // Sum over the sequences of ceil(rows / tile), whatever their shares are: a bound, one
  // too many for each whose rows are whole tiles (one chunk of 32 tokens at G = 4 gets 9
  // parts of its keys where 18 would fill the SMs).
  pl.tiles = packed / (128 * pl.nq) + std::min<long long>(p->batch, p->num_tokens);
  const long long ctas = pl.tiles * p->num_kv_heads;
  if (p->num_splits > 0) {
    pl.splits = p->num_splits;
  } else {
    // Few row tiles: as many parts as fill the SMs once, each of two or more key
    // tiles (each part's partial costs a write, a read and the joining kernel).
    const int tn = p->head_dim == 256 ? 64 : 128;
    const long long cap = static_cast<long long>(p->max_blocks) * p->block_size;
    const long long span = 128ll * pl.nq / g + 1;
    const long long seen =
        p->window ? std::min(cap, static_cast<long long>(p->window) + span + p->num_sinks + tn) : cap;
    const long long by_keys = (seen + tn - 1) / tn / 2;
    pl.splits = static_cast<int>(std::max(1ll, std::min({slots / ctas, by_keys, 64ll})));
  }
  if (pl.splits > 1)
    pl.ws_bytes = static_cast<size_t>(pl.splits) * p->num_tokens * p->num_heads *
                  (kernel_dim(p) + 1) * sizeof(float);
  return pl;
}

template <typename T, int D, int NQ, Fetch kFetch>
static cudaError_t launch_tiles_as(const CUtensorMap& mk, const CUtensorMap& mv, const TileParams& a,
                                const Plan& pl, cudaStream_t stream) {
  using C = TC<D, NQ>;
  static std::mutex mu;
  static bool set[64] = {false};
  int dev = 0;
  cudaError_t e = cudaGetDevice(&dev);
  if (e != cudaSuccess || dev >= 64) return cudaErrorInvalidDevice;
  {
    std::lock_guard<std::mutex> lk(mu);
    if (!set[dev]) {
      e = cudaFuncSetAttribute(prompt_tile_kernel<T, D, NQ, kFetch>,
                               cudaFuncAttributeMaxDynamicSharedMemorySize, C::kSmem);
      if (e != cudaSuccess) return e;
      set[dev] = true;
    }
  }
  const long long grid = pl.tiles * a.p.Hkv * pl.splits;
  if (grid > 0x7fffffffll) return cudaErrorInvalidConfiguration;
  // Programmatic stream serialisation: the barriers' and tensor memory's set-up
  // runs while the previous kernel in the stream ends; griddepcontrol.wait orders
  // everything else behind it.
  cudaLaunchConfig_t cfg = {};
  cudaLaunchAttribute attr[1];
  attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
  attr[0].val.programmaticStreamSerializationAllowed = 1;
  cfg.gridDim = dim3(static_cast<unsigned>(grid));
  cfg.blockDim = dim3(C::kThreads);
  cfg.dynamicSmemBytes = C::kSmem;
  cfg.stream = stream;
  cfg.attrs = attr;
  cfg.numAttrs = 1;
  e = cudaLaunchKernelEx(&cfg, prompt_tile_kernel<T, D, NQ, kFetch>, mk, mv, a);
  if (e == cudaSuccess && pl.splits > 1) {
    const long long warps = static_cast<long long>(a.p.T) * a.p.Hq;
    cfg.gridDim = dim3(static_cast<unsigned>((warps + 3) / 4));
    cfg.blockDim = dim3(128);
    cfg.dynamicSmemBytes = 0;
    e = cudaLaunchKernelEx(&cfg, prompt_join_kernel<T, D>, a);
  }
  return e;
}

template <typename T, int D, int NQ>
static cudaError_t launch_tiles(const CUtensorMap& mk, const CUtensorMap& mv, const TileParams& a,
                                const Plan& pl, Fetch fetch, cudaStream_t stream) {
  if (fetch == Fetch::kRows) return launch_tiles_as<T, D, NQ, Fetch::kRows>(mk, mv, a, pl, stream);
  if (fetch == Fetch::kPieces) return launch_tiles_as<T, D, NQ, Fetch::kPieces>(mk, mv, a, pl, stream);
  return launch_tiles_as<T, D, NQ, Fetch::kBoxes>(mk, mv, a, pl, stream);
}

template <typename T>
static cudaError_t launch_tiles_d(const CUtensorMap& mk, const CUtensorMap& mv, const TileParams& a,
                                  const Plan& pl, Fetch fetch, int D, cudaStream_t stream) {
  if (D == 256) return launch_tiles<T, 256, 1>(mk, mv, a, pl, fetch, stream);
  if (D == 128)
    return pl.nq == 2 ? launch_tiles<T, 128, 2>(mk, mv, a, pl, fetch, stream)
                      : launch_tiles<T, 128, 1>(mk, mv, a, pl, fetch, stream);
  return launch_tiles<T, 64, 1>(mk, mv, a, pl, fetch, stream);
}

}  // namespace pp

using namespace pp;

extern "C" {

pa_status_t pa_prompt_workspace(const pa_prompt_params* p, size_t* workspace_bytes) {
  const pa_status_t v = validate(p);
  if (v != PA_OK) return v;
  size_t bytes = 0;
  if (p->num_tokens > 0 && p->batch > 0) {
    const int sms = pa_device_sm_count();
    if (sms <= 0) return PA_ERR_LAUNCH;
    bytes = make_plan(p, sms).ws_bytes;
  }
  if (workspace_bytes) *workspace_bytes = bytes;
  return PA_OK;
}

pa_status_t pa_prompt(const pa_prompt_params* p, cudaStream_t stream) {
  pa_status_t v = validate(p);
  if (v != PA_OK) return v;
  if (p->num_tokens == 0 || p->batch == 0) return PA_OK;
  v = validate_launch(p);
  if (v != PA_OK) return v;
  const int sms = pa_device_sm_count();
  if (sms <= 0) return PA_ERR_LAUNCH;
  const Plan pl = make_plan(p, sms);
  if (pl.ws_bytes && (pl.ws_bytes > p->workspace_bytes || !p->workspace)) return PA_ERR_WORKSPACE;
  if (!aligned16(p->workspace)) return PA_ERR_ARG;
  const bool half = p->dtype == PA_F16;
  TileParams a;
  memset(&a, 0, sizeof(a));
  a.p = make_params(p);
  a.dh = p->head_dim;
  // box rows: a power of two in the page size, at most 32 (where a window starts,
  // up to R - 1 hidden keys are read)
  a.R = 8;
  while (a.R < 32 && p->block_size % (2 * a.R) == 0) a.R *= 2;
  a.lR = 0;
  while ((1 << a.lR) < a.R) ++a.lR;
  a.bs_log2 = -1;
  for (int k = 0; k < 31; ++k)
    if ((1 << k) == p->block_size) a.bs_log2 = k;
  a.div_g = make_fastdiv(static_cast<uint32_t>(a.p.G));
  a.div_bs = make_fastdiv(static_cast<uint32_t>(p->block_size));
  a.splits = pl.splits;
  a.o_part = static_cast<float*>(p->workspace);
  a.lse_part = a.o_part + static_cast<size_t>(pl.splits) * p->num_tokens * p->num_heads * kernel_dim(p);
  CUtensorMap mk, mv;
  memset(&mk, 0, sizeof(mk));
  memset(&mv, 0, sizeof(mv));
  Fetch fetch = Fetch::kBoxes;
  RowList rk, rv;
  if (p->block_size % 8 == 0) {
    if (!encode_map(&mk, p, p->k_cache, p->k_stride_block, p->k_stride_slot, p->k_stride_head, a.R) ||
        !encode_map(&mv, p, p->v_cache, p->v_stride_block, p->v_stride_slot, p->v_stride_head, a.R))
      return PA_ERR_ARG;
  } else if (row_list(p, p->k_stride_block, p->k_stride_slot, p->k_stride_head, &rk) &&
             row_list(p, p->v_stride_block, p->v_stride_slot, p->v_stride_head, &rv)) {
    fetch = Fetch::kRows;
    if (!encode_rows(&mk, p, p->k_cache, rk) || !encode_rows(&mv, p, p->v_cache, rv))
      return PA_ERR_ARG;
    a.row_b[0] = rk.b, a.row_s[0] = rk.s, a.row_h[0] = rk.h;
    a.row_b[1] = rv.b, a.row_s[1] = rv.s, a.row_h[1] = rv.h;
  } else {
    fetch = Fetch::kPieces;
  }
  const cudaError_t e =
      half ? launch_tiles_d<__half>(mk, mv, a, pl, fetch, p->head_dim, stream)
               : launch_tiles_d<__nv_bfloat16>(mk, mv, a, pl, fetch, p->head_dim, stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // extern "C"
