// Writing keys and values into the 4-bit cache, and reading them back.
//
// Both kernels move bytes: 4 per value come in (K and V, 16 bits each) and
// 1.25 go out, or the other way round. A thread owns eight channels of one
// (token, head) of K and of V: one 16-byte and one 4-byte access each, four
// neighbouring lanes making a group of 32 channels, so the group's minimum
// and maximum take two shuffles. Blocks are laid out over (new tokens of a
// sequence) x (sequence): ragged batches leave blocks that only exit.
#include "kv4.cuh"

namespace pb2 {
namespace {

constexpr int kThreads = 256;

struct CacheArgs {
  Kv4Tokens t;
  uint8_t *pool;
  const uint16_t *k, *v; // append: source rows
  uint16_t *ko, *vo;     // read: destination rows
  long long k_stride, v_stride;
  int kv_heads;
  FastDiv heads_div;
};

// Where this thread's eight channels sit.
struct Spot {
  bool live;          // a token of this sequence
  bool held;          // with a position in the cache
  long long row;      // packed row
  int head, chunk;    // eight-channel chunk of the head
  uint8_t *block;     // (page, head) block
  int slot;           // token within the page
};
template <int D> __device__ __forceinline__ Spot spot_of(const CacheArgs &g) {
  constexpr int kChunks = D / 8;
  Spot s;
  const int b = blockIdx.y;
  const Kv4Seq q = kv4_seq(g.t, b);
  const uint32_t idx = blockIdx.x * kThreads + threadIdx.x;
  s.chunk = idx % kChunks;
  const uint32_t rest = idx / kChunks;
  const uint32_t tok = g.heads_div.div(rest);
  s.head = rest - tok * g.kv_heads;
  s.live = tok < static_cast<uint32_t>(q.n);
  const int pos = q.len - q.n + static_cast<int>(tok);
  s.held = s.live && pos >= 0;
  s.row = q.first + static_cast<long long>(tok);
  s.block = nullptr;
  s.slot = 0;
  if (s.held) {
    const long long page = kv4_page(g.t, b, pos);
    s.slot = pos & ((1 << g.t.page_shift) - 1);
    s.block = g.pool + (page * g.kv_heads + s.head) * static_cast<long long>((D + D / 4) << g.t.page_shift);
  }
  return s;
}

// Quantises eight channels (with the three lanes that hold the rest of the
// group): returns the packed codes and the group's (scale, minimum).
template <bool BF16> __device__ __forceinline__ uint32_t quantise8(uint4 w, uint32_t &params) {
  const uint32_t in[4] = {w.x, w.y, w.z, w.w};
  constexpr float kMost = BF16 ? 8.507059173023462e37f : 65000.f; // 2^126
  float x[8];
#pragma unroll
  for (int i = 0; i < 4; ++i) {
    x[2 * i] = kv4_lo<BF16>(in[i]);
    x[2 * i + 1] = kv4_hi<BF16>(in[i]);
  }
#pragma unroll
  for (int i = 0; i < 8; ++i)
    x[i] = x[i] == x[i] ? fminf(fmaxf(x[i], -kMost), kMost) : 0.f;
  float lo = x[0], hi = x[0];
#pragma unroll
  for (int i = 1; i < 8; ++i) {
    lo = fminf(lo, x[i]);
    hi = fmaxf(hi, x[i]);
  }
#pragma unroll
  for (int o = 1; o < 4; o *= 2) {
    lo = fminf(lo, __shfl_xor_sync(~0u, lo, o));
    hi = fmaxf(hi, __shfl_xor_sync(~0u, hi, o));
  }
  params = kv4_pack<BF16>(__fdiv_rn(__fsub_rn(hi, kv4_lo<BF16>(kv4_pack<BF16>(lo, lo))), 15.f), lo);
  const float scale = kv4_lo<BF16>(params);
  lo = kv4_hi<BF16>(params);
  const float inv = scale > 1e-30f ? __fdiv_rn(1.f, scale) : 0.f;
  uint32_t codes = 0;
#pragma unroll
  for (int i = 0; i < 8; ++i) {
    const float c = fminf(fmaxf(__fmul_rn(__fsub_rn(x[i], lo), inv), 0.f), 15.f);
    // Adding 1.5 * 2^23 rounds to the nearest whole number (ties to even)
    // and leaves it in the low bits.
    codes |= (__float_as_uint(__fadd_rn(c, 12582912.f)) & 15u) << (4 * i);
  }
  return codes;
}

template <int D, bool BF16> __global__ void __launch_bounds__(kThreads) append_kernel(const __grid_constant__ CacheArgs g) {
  pdl_begin();
  const Spot s = spot_of<D>(g);
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (s.held) {
    const long long e = s.head * D + s.chunk * 8;
    k = *reinterpret_cast<const uint4 *>(g.k + s.row * g.k_stride + e);
    v = *reinterpret_cast<const uint4 *>(g.v + s.row * g.v_stride + e);
  }
  uint32_t kp, vp;
  const uint32_t kc = quantise8<BF16>(k, kp), vc = quantise8<BF16>(v, vp);
  if (!s.held)
    return;
  const int page = 1 << g.t.page_shift;
  uint32_t *codes = reinterpret_cast<uint32_t *>(s.block) + s.slot * (D / 8) + s.chunk;
  codes[0] = kc;
  codes[page * (D / 8)] = vc;
  if (s.chunk % 4 == 0) {
    uint32_t *params = reinterpret_cast<uint32_t *>(s.block) + page * (D / 4) + s.slot * (D / 32) + s.chunk / 4;
    params[0] = kp;
    params[page * (D / 32)] = vp;
  }
}

template <bool BF16> __device__ __forceinline__ uint4 restore8(uint32_t codes, uint32_t params) {
  const float scale = kv4_lo<BF16>(params), lo = kv4_hi<BF16>(params);
  float x[8];
#pragma unroll
  for (int i = 0; i < 8; ++i) // 2^23 + c, exactly
    x[i] = fmaf(__uint_as_float(0x4B000000u | ((codes >> (4 * i)) & 15u)) - 8388608.f, scale, lo);
  return make_uint4(kv4_pack<BF16>(x[0], x[1]), kv4_pack<BF16>(x[2], x[3]), kv4_pack<BF16>(x[4], x[5]),
                    kv4_pack<BF16>(x[6], x[7]));
}

template <int D, bool BF16> __global__ void __launch_bounds__(kThreads) read_kernel(const __grid_constant__ CacheArgs g) {
  pdl_begin();
  const Spot s = spot_of<D>(g);
  if (!s.live)
    return;
  uint4 k = make_uint4(0, 0, 0, 0), v = k;
  if (s.held) {
    const int page = 1 << g.t.page_shift;
    const uint32_t *codes = reinterpret_cast<const uint32_t *>(s.block) + s.slot * (D / 8) + s.chunk;
    const uint32_t *params =
        reinterpret_cast<const uint32_t *>(s.block) + page * (D / 4) + s.slot * (D / 32) + s.chunk / 4;
    const uint32_t kc = codes[0], vc = codes[page * (D / 8)], kp = params[0], vp = params[page * (D / 32)];
    k = restore8<BF16>(kc, kp);
    v = restore8<BF16>(vc, vp);
  }
  const long long e = (s.row * g.kv_heads + s.head) * D + s.chunk * 8;
  *reinterpret_cast<uint4 *>(g.ko + e) = k;
  *reinterpret_cast<uint4 *>(g.vo + e) = v;
}

template <int D, bool BF16> cudaError_t launch(const CacheArgs &g, bool append, cudaStream_t s) {
  const long long work = static_cast<long long>(g.t.max_new) * g.kv_heads * (D / 8);
  const dim3 grid(static_cast<unsigned>((work + kThreads - 1) / kThreads), g.t.batch);
  return launch_pdl(append ? append_kernel<D, BF16> : read_kernel<D, BF16>, grid, kThreads, 0, s, g);
}

cudaError_t dispatch(const Kv4Cache &c, const CacheArgs &g, bool append, cudaStream_t s) {
  // Chunks of a sequence's new tokens are counted in 32 bits.
  if (static_cast<long long>(g.t.max_new) * c.kv_heads * (c.head_dim / 8) >= (1ll << 31) || g.t.batch > 65535)
    return cudaErrorInvalidValue;
  switch (c.head_dim * 2 + c.bf16) {
  case 64: return launch<32, false>(g, append, s);
  case 65: return launch<32, true>(g, append, s);
  case 128: return launch<64, false>(g, append, s);
  case 129: return launch<64, true>(g, append, s);
  case 256: return launch<128, false>(g, append, s);
  case 257: return launch<128, true>(g, append, s);
  }
  return cudaErrorInvalidValue;
}

} // namespace

cudaError_t kv4_append(const Kv4Cache &c, const Kv4Tokens &t, const void *k, long long k_stride, const void *v,
                       long long v_stride, cudaStream_t stream) {
  CacheArgs g{};
  g.t = t;
  g.pool = c.pool;
  g.k = static_cast<const uint16_t *>(k);
  g.v = static_cast<const uint16_t *>(v);
  g.k_stride = k_stride;
  g.v_stride = v_stride;
  g.kv_heads = c.kv_heads;
  g.heads_div = FastDiv(c.kv_heads);
  return dispatch(c, g, true, stream);
}

cudaError_t kv4_read(const Kv4Cache &c, const Kv4Tokens &t, void *k, void *v, cudaStream_t stream) {
  CacheArgs g{};
  g.t = t;
  g.pool = c.pool;
  g.ko = static_cast<uint16_t *>(k);
  g.vo = static_cast<uint16_t *>(v);
  g.kv_heads = c.kv_heads;
  g.heads_div = FastDiv(c.kv_heads);
  return dispatch(c, g, false, stream);
}

} // namespace pb2
