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
#include <mutex>

#include "pa_decode.h"
#include "fastdiv.h"

namespace pp {

using pa::FastDiv;
using pa::fast_div;
using pa::make_fastdiv;

constexpr unsigned kFull = 0xffffffffu;
constexpr float kSentinel = -1e30f;     // LSE of a row that sees nothing
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kLn2 = 0.6931471805599453f;

struct Params {
  const char* q;
  long long q_st, q_sh;                           // bytes
  const char* kc;
  const char* vc;
  long long k_sb, k_ss, k_sh, v_sb, v_ss, v_sh;   // bytes (CUDA-core path)
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

template <typename T>
__device__ __forceinline__ float to_float(uint16_t x);
template <>
__device__ __forceinline__ float to_float<__half>(uint16_t x) {
  return __half2float(__ushort_as_half(x));
}
template <>
__device__ __forceinline__ float to_float<__nv_bfloat16>(uint16_t x) {
  return __bfloat162float(__ushort_as_bfloat16(x));
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

// ----------------------------------------------------------------------------
// CUDA-core path: every shape
// ----------------------------------------------------------------------------
// One warp per (query row, query head): lane j scores the j-th token of 32
// against the query (in shared memory), then the lanes, each owning D/32
// dimensions, accumulate p_j v_j. It serves head_dim 32 and pages that are not
// a multiple of 8 tokens, which the tile kernel's copies do not cover.
template <typename T, int D>
__global__ void __launch_bounds__(128) prompt_rows_kernel(const Params p) {
  constexpr int N = D / 32;
  __shared__ float qs[4][D];
  const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
  const long long w = static_cast<long long>(blockIdx.x) * 4 + warp;
  if (w >= static_cast<long long>(p.T) * p.Hq) return;
  const int row = static_cast<int>(w / p.Hq);
  const int hq = static_cast<int>(w - static_cast<long long>(row) * p.Hq);
  // the last sequence that starts at or before the row
  int lo = 0, hi = p.B - 1;
  while (lo < hi) {
    const int mid = (lo + hi + 1) >> 1;
    if (__ldg(p.starts + mid) <= row) lo = mid; else hi = mid - 1;
  }
  bool bad;
  const Seq s = load_seq(p, lo, bad);
  if (bad && lane == 0) flag(p, PA_STATUS_BAD_SEQLEN);
  if (row < s.start || row >= s.start + s.n) return;   // behind the last sequence
  const int b = lo, kvh = hq / p.G;
  const int pos = s.S - s.n + row - s.start;
  const int first = pos >= p.window ? pos - p.window + 1 : 0;   // of the window
  const int a = min(p.sinks, first);                            // visible sinks
  const int count = pos < 0 ? 0 : a + pos + 1 - first;
  const uint16_t* qp = reinterpret_cast<const uint16_t*>(p.q + row * p.q_st + hq * p.q_sh);
  for (int d = lane; d < D; d += 32) qs[warp][d] = to_float<T>(qp[d]);
  __syncwarp();
  float m = -INFINITY, l = 0.f, acc[N];
#pragma unroll
  for (int i = 0; i < N; ++i) acc[i] = 0.f;
  for (int c = 0; c < count; c += 32) {
    int t = c + lane;
    int page = -1, slot = 0;
    if (t < count) {
      t = t < a ? t : t - a + first;
      const int j = t / p.bs;
      page = __ldg(p.bt + b * p.bt_sb + j);
      slot = t - j * p.bs;
      if (page < 0 || page >= p.NB) {
        flag(p, PA_STATUS_BAD_BLOCK);
        page = -1;
      }
    }
    float sc = -INFINITY;
    if (page >= 0) {
      const uint4* kr = reinterpret_cast<const uint4*>(p.kc + page * p.k_sb + slot * p.k_ss + kvh * p.k_sh);
      float dot = 0.f;
#pragma unroll
      for (int i = 0; i < D / 8; ++i) {
        const uint4 x = __ldg(kr + i);
        const uint32_t x4[4] = {x.x, x.y, x.z, x.w};
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          dot = fmaf(to_float<T>(x4[e] & 0xffff), qs[warp][i * 8 + 2 * e], dot);
          dot = fmaf(to_float<T>(x4[e] >> 16), qs[warp][i * 8 + 2 * e + 1], dot);
        }
      }
      sc = dot * p.scale_log2;
    }
    float cm = sc;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) cm = fmaxf(cm, __shfl_xor_sync(kFull, cm, o));
    const float mn = fmaxf(m, cm);
    if (mn == -INFINITY) continue;
    const float alpha = exp2f(m - mn);
    const float pv = sc == -INFINITY ? 0.f : exp2f(sc - mn);
    float ps = pv;
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) ps += __shfl_xor_sync(kFull, ps, o);
    l = fmaf(l, alpha, ps);
#pragma unroll
    for (int i = 0; i < N; ++i) acc[i] *= alpha;
    m = mn;
    const int nj = min(32, count - c);
    for (int j = 0; j < nj; ++j) {
      const float pj = __shfl_sync(kFull, pv, j);
      const int pg = __shfl_sync(kFull, page, j);
      const int sl = __shfl_sync(kFull, slot, j);
      if (pg < 0) continue;
      const uint16_t* vr = reinterpret_cast<const uint16_t*>(p.vc + pg * p.v_sb + sl * p.v_ss + kvh * p.v_sh) + lane * N;
#pragma unroll
      for (int i = 0; i < N; ++i) acc[i] = fmaf(pj, to_float<T>(__ldg(vr + i)), acc[i]);
    }
  }
  const float inv = l > 0.f ? 1.f / l : 0.f;
  uint16_t* dst = reinterpret_cast<uint16_t*>(p.out + row * p.o_st + hq * p.o_sh) + lane * N;
#pragma unroll
  for (int i = 0; i < N; ++i) dst[i] = static_cast<uint16_t>(pack2<T>(acc[i] * inv, 0.f));
  if (lane == 0 && p.lse)
    p.lse[static_cast<long long>(row) * p.Hq + hq] = l > 0.f ? (m + log2f(l)) * kLn2 : kSentinel;
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

template <typename T>
static cudaError_t launch_rows(const Params& a, int D, cudaStream_t stream) {
  const long long warps = static_cast<long long>(a.T) * a.Hq;
  const dim3 grid(static_cast<unsigned>((warps + 3) / 4));
  if (D == 32) prompt_rows_kernel<T, 32><<<grid, 128, 0, stream>>>(a);
  else if (D == 64) prompt_rows_kernel<T, 64><<<grid, 128, 0, stream>>>(a);
  else if (D == 128) prompt_rows_kernel<T, 128><<<grid, 128, 0, stream>>>(a);
  else prompt_rows_kernel<T, 256><<<grid, 128, 0, stream>>>(a);
  return cudaGetLastError();
}

}  // namespace pp

using namespace pp;

extern "C" {

pa_status_t pa_prompt_workspace(const pa_prompt_params* p, size_t* workspace_bytes) {
  const pa_status_t v = validate(p);
  if (v != PA_OK) return v;
  if (workspace_bytes) *workspace_bytes = 0;
  return PA_OK;
}

pa_status_t pa_prompt(const pa_prompt_params* p, cudaStream_t stream) {
  pa_status_t v = validate(p);
  if (v != PA_OK) return v;
  if (p->num_tokens == 0 || p->batch == 0) return PA_OK;
  v = validate_launch(p);
  if (v != PA_OK) return v;
  const Params a = make_params(p);
  const cudaError_t e = p->dtype == PA_F16 ? launch_rows<__half>(a, p->head_dim, stream)
                                           : launch_rows<__nv_bfloat16>(a, p->head_dim, stream);
  return e == cudaSuccess ? PA_OK : PA_ERR_LAUNCH;
}

}  // extern "C"
