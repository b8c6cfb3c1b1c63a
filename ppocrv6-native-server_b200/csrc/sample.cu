// Token sampling: temperature, top-k, top-p, min-p and the draw, one CTA per
// row of logits.
//
// Masses are whole numbers, floor(exp(-(max - x) / T) * 2^32): every sum is
// exact whatever its order, so the result depends on no split of the work.
// What stays of a row is always a prefix of its order (larger logits first,
// equal ones by index), so it is described by one logit value (as an
// order-preserving 32-bit key), and by how many of the logits equal to it
// stay. That value is found digit by digit from the top: a histogram of
// counts and masses over 256 values of one byte of the key, among the logits
// that agree with the digits found so far.
#include "kernels.h"
#include "ptx.cuh"
#include <cuda_bf16.h>

namespace pb2 {
namespace {

constexpr int kThreads = 1024;
using u64 = unsigned long long;

template <int TYPE> __device__ __forceinline__ float logit(const void *row, int i) {
  float x;
  if constexpr (TYPE == LOGIT_F32)
    x = static_cast<const float *>(row)[i];
  else if constexpr (TYPE == LOGIT_BF16)
    x = __bfloat162float(static_cast<const __nv_bfloat16 *>(row)[i]);
  else
    x = __half2float(static_cast<const half *>(row)[i]);
  return x == x ? x + 0.f : -INFINITY; // NaN never wins; -0 equals 0
}
// Larger logits, larger keys.
__device__ __forceinline__ uint32_t key_of(float x) {
  const uint32_t u = __float_as_uint(x);
  return u & 0x80000000u ? ~u : u | 0x80000000u;
}
__device__ __forceinline__ float value_of(uint32_t key) {
  return __uint_as_float(key & 0x80000000u ? key & 0x7FFFFFFFu : ~key);
}
__device__ __forceinline__ float share_of(float x, float top, float t) {
  return x == top ? 1.f : expf(-__fdiv_rn(__fsub_rn(top, x), t));
}
__device__ __forceinline__ u64 mass_of(float e) { return __float2ull_rz(e * 4294967296.f); }
// floor(whole * share / 2^24) for share <= 2^24, whole < 2^57.
__device__ __forceinline__ u64 part_of(u64 whole, u64 share) {
  return share * (whole >> 24) + ((share * (whole & 0xFFFFFFu)) >> 24);
}

// The first `ties` logits equal to the key and every larger one: `count`
// logits of mass `mass`.
struct Prefix {
  uint32_t key;
  int ties, count;
  u64 mass;
};

struct Shared {
  unsigned count[256];
  u64 mass[256];
  u64 warp[32];
  int warp_n[32];
  Prefix found;
};

template <typename T> __device__ __forceinline__ T block_sum(T v, T *slots) {
  const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
  for (int o = 16; o; o /= 2)
    v += __shfl_xor_sync(~0u, v, o);
  __syncthreads();
  if (lane == 0)
    slots[warp] = v;
  __syncthreads();
  v = slots[lane];
#pragma unroll
  for (int o = 16; o; o /= 2)
    v += __shfl_xor_sync(~0u, v, o);
  return v;
}

// The first `want` logits of the row's order (by_mass false), or the fewest
// whose mass reaches `want` > 0 (by_mass true).
template <int TYPE>
__device__ Prefix select(const void *row, int vocab, float top, float t, bool by_mass, u64 want, Shared &sh) {
  uint32_t prefix = 0;
  u64 before = 0; // mass of the logits above the digits found so far
  int above = 0;
  for (int shift = 24; shift >= 0; shift -= 8) {
    __syncthreads();
    for (int i = threadIdx.x; i < 256; i += kThreads) {
      sh.count[i] = 0;
      sh.mass[i] = 0;
    }
    __syncthreads();
    for (int i = threadIdx.x; i < vocab; i += kThreads) {
      const float x = logit<TYPE>(row, i);
      const uint32_t k = key_of(x);
      if (shift == 24 || (k >> (shift + 8)) == prefix) {
        const uint32_t d = (k >> shift) & 255u;
        atomicAdd(&sh.count[d], 1u);
        const u64 m = mass_of(share_of(x, top, t));
        if (m)
          atomicAdd(&sh.mass[d], m);
      }
    }
    __syncthreads();
    // Every thread walks the bins alike.
    int d = 255;
    for (; d > 0; --d) {
      const u64 have = by_mass ? before + sh.mass[d] : static_cast<u64>(above) + sh.count[d];
      if (have >= want)
        break;
      before += sh.mass[d];
      above += sh.count[d];
    }
    prefix = prefix << 8 | static_cast<uint32_t>(d);
  }
  Prefix p;
  p.key = prefix;
  const int equal = static_cast<int>(sh.count[prefix & 255u]);
  const u64 each = mass_of(share_of(value_of(prefix), top, t));
  if (by_mass)
    p.ties = each ? static_cast<int>(min(static_cast<u64>(equal), (want - before + each - 1) / each)) : equal;
  else
    p.ties = min(equal, static_cast<int>(want) - above);
  p.count = above + p.ties;
  p.mass = before + each * p.ties;
  return p;
}

template <int TYPE> __global__ void __launch_bounds__(kThreads) sample_kernel(const __grid_constant__ SampleArgs a) {
  __shared__ Shared sh;
  pdl_begin();
  const int r = blockIdx.x, tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
  const int V = a.vocab;
  const void *row = static_cast<const char *>(a.logits) + static_cast<long long>(r) * a.stride * (TYPE == LOGIT_F32 ? 4 : 2);
  float t = a.temperature ? a.temperature[r] : 1.f;
  int k = a.top_k ? a.top_k[r] : 0;
  k = k <= 0 || k > V ? V : k;
  if (!(t > 0.f)) {
    t = 1.f;
    k = 1;
  }
  const float tp = a.top_p ? a.top_p[r] : 1.f, mp = a.min_p ? a.min_p[r] : 0.f;
  const u64 p24 = __float2ull_rz(fminf(fmaxf(tp, 0.f), 1.f) * 16777216.f);
  const u64 u24 = min(__float2ull_rz(fminf(fmaxf(a.uniform[r], 0.f), 1.f) * 16777216.f), 16777215ull);

  float top = -INFINITY;
  for (int i = tid; i < V; i += kThreads)
    top = fmaxf(top, logit<TYPE>(row, i));
#pragma unroll
  for (int o = 16; o; o /= 2)
    top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  float *slots = reinterpret_cast<float *>(sh.warp);
  if (lane == 0)
    slots[warp] = top;
  __syncthreads();
  top = slots[lane];
#pragma unroll
  for (int o = 16; o; o /= 2)
    top = fmaxf(top, __shfl_xor_sync(~0u, top, o));
  if (top == -INFINITY) {
    if (tid == 0) {
      a.ids[r] = -1;
      a.prob[r] = 0.f;
      a.kept[r] = 0;
    }
    return;
  }
  u64 sum = 0;
  int likely = 0;
  for (int i = tid; i < V; i += kThreads) {
    const float e = share_of(logit<TYPE>(row, i), top, t);
    sum += mass_of(e);
    likely += e >= mp;
  }
  const u64 all = block_sum(sum, sh.warp);
  likely = max(block_sum(likely, sh.warp_n), 1);

  Prefix p{0, V, V, all}; // everything (key 0 is below every logit's)
  if (k < V)
    p = select<TYPE>(row, V, top, t, false, k, sh);
  if (p24 < (1ull << 24)) {
    const u64 limit = max(part_of(p.mass, p24), 1ull);
    p = select<TYPE>(row, V, top, t, true, limit, sh);
  }
  if (likely < p.count)
    p = select<TYPE>(row, V, top, t, false, likely, sh);

  // The draw, in index order: each warp sums a run of the row.
  const u64 target = part_of(p.mass, u24);
  const float edge = value_of(p.key);
  const u64 each = p.key ? mass_of(share_of(edge, top, t)) : 0;
  const int run = ((V + kThreads / 32 - 1) / (kThreads / 32) + 31) / 32 * 32;
  const int i0 = min(warp * run, V), i1 = min(i0 + run, V);
  u64 mass = 0;
  int ties = 0;
  for (int i = i0 + lane; i < i1; i += 32) {
    const float x = logit<TYPE>(row, i);
    const uint32_t key = key_of(x);
    if (key > p.key)
      mass += mass_of(share_of(x, top, t));
    ties += key == p.key;
  }
#pragma unroll
  for (int o = 16; o; o /= 2) {
    mass += __shfl_xor_sync(~0u, mass, o);
    ties += __shfl_xor_sync(~0u, ties, o);
  }
  __syncthreads();
  if (lane == 0) {
    sh.warp[warp] = mass;
    sh.warp_n[warp] = ties;
  }
  __syncthreads();
  u64 before = 0;
  int tied = 0;
  for (int w = 0; w < warp; ++w) {
    before += sh.warp[w] + each * min(sh.warp_n[w], max(p.ties - tied, 0));
    tied += sh.warp_n[w];
  }
  const u64 after = before + mass + each * min(ties, max(p.ties - tied, 0));
  if (!(before <= target && target < after))
    return;
  // This warp's run holds the token.
  for (int i = i0; i < i1; i += 32) {
    const float x = i + lane < i1 ? logit<TYPE>(row, i + lane) : -INFINITY;
    const uint32_t key = i + lane < i1 ? key_of(x) : 0;
    const unsigned tie = __ballot_sync(~0u, i + lane < i1 && key == p.key);
    const bool stays = key > p.key || ((tie >> lane & 1) && tied + __popc(tie & ((1u << lane) - 1)) < p.ties);
    const u64 m = stays && i + lane < i1 ? mass_of(share_of(x, top, t)) : 0;
    u64 cum = m;
#pragma unroll
    for (int o = 1; o < 32; o *= 2) {
      const u64 y = __shfl_up_sync(~0u, cum, o);
      cum += lane >= o ? y : 0;
    }
    const unsigned past = __ballot_sync(~0u, before + cum > target);
    if (past) {
      if (lane == __ffs(past) - 1) {
        a.ids[r] = i + lane;
        a.prob[r] = __fdiv_rn(__ull2float_rn(m), __ull2float_rn(all));
        a.kept[r] = p.count;
      }
      return;
    }
    before += __shfl_sync(~0u, cum, 31);
    tied += __popc(tie);
  }
}

} // namespace

cudaError_t sample_tokens(const SampleArgs &a, int type, cudaStream_t stream) {
  auto *kernel = type == LOGIT_F32    ? sample_kernel<LOGIT_F32>
                 : type == LOGIT_BF16 ? sample_kernel<LOGIT_BF16>
                                      : sample_kernel<LOGIT_F16>;
  return launch_pdl(kernel, a.rows, kThreads, 0, stream, a);
}

} // namespace pb2
