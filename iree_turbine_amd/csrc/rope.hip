// Rotary positions: the pairs of the first R elements of every head turned by position * frequency,
//   (a, b) -> m (a cos t - b sin t, a sin t + b cos t),   t = pos * f_i,  i < R / 2,
// with pair i made of elements (2i, 2i + 1) (interleaved) or (i, i + R/2) (halves); elements from R on pass through.
// The transpose (sin negated) is the gradient.  Frequencies come from the caller, so every way of stretching them for
// long contexts is a matter of that vector and of m.
//
// Angles are formed in 64 bits: at position 10^6 a product in 32 bits is off by 0.06 rad.  t / 2 pi is reduced to
// [-1/2, 1/2] turns there, and only the remainder goes to 32 bits.  That costs R/2 short 64-bit computations per token,
// shared by all its heads through LDS.  The rotation itself is done in 32 bits and rounded once.
//
// The op reads and writes every element once (HBM bound): 16 bytes per lane where rows allow it.
#include "common.hpp"
#include <math.h>
#include <type_traits>

namespace mi355 {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_PAIRS = 512;  // R / 2

// One operand: where a token's head rows lie, in elements; the D elements of a row are contiguous.
struct RopeRows {
  const void* src;
  void* dst;
  long long src_token, src_head, dst_token, dst_head;
  int heads;
};

template <typename T>
__device__ __forceinline__ float rp_load(T v) {
  return (float)v;
}
template <typename T>
__device__ __forceinline__ T rp_store(float v) {
  return (T)v;
}

// (cos, sin) of pos * freq, both times `mul`
__device__ __forceinline__ floatx2 rp_angle(int pos, double freq, float mul, float sin_mul) {
  const double turns = (double)pos * (freq * 0.15915494309189533577);
  const float rest = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.f * rest, &s, &c);
  return floatx2{c * mul, s * sin_mul};
}

// One work item of a head row: item i < n_pair rotates W pairs, the others copy W elements (halves) or 2 W (interleaved:
// W pairs are 2 W neighbours).  W = 1: no alignment is assumed.
template <typename T, bool INTER, int W>
__device__ __forceinline__ void rp_item(const T* __restrict__ src, T* __restrict__ dst, int item, int n_pair, int half,
                                        const floatx2* cs) {
  constexpr int WI = INTER ? 2 * W : W;  // elements at one place
  struct alignas(W == 1 ? sizeof(T) : WI * sizeof(T)) Pack { T v[WI]; };
  if (item >= n_pair) {
    const int at = 2 * half + (item - n_pair) * W;
    if constexpr (INTER) {
      // the rest of the row is cut into W elements, half a place each
      struct alignas(W == 1 ? sizeof(T) : W * sizeof(T)) Half { T v[W]; };
      *reinterpret_cast<Half*>(dst + at) = *reinterpret_cast<const Half*>(src + at);
    } else {
      *reinterpret_cast<Pack*>(dst + at) = *reinterpret_cast<const Pack*>(src + at);
    }
    return;
  }
  if constexpr (INTER) {
    const int at = item * WI;
    Pack x = *reinterpret_cast<const Pack*>(src + at);
#pragma unroll
    for (int e = 0; e < W; e++) {
      const floatx2 r = cs[item * W + e];
      const float a = rp_load(x.v[2 * e]), b = rp_load(x.v[2 * e + 1]);
      x.v[2 * e] = rp_store<T>(a * r[0] - b * r[1]);
      x.v[2 * e + 1] = rp_store<T>(a * r[1] + b * r[0]);
    }
    *reinterpret_cast<Pack*>(dst + at) = x;
  } else {
    const int at = item * W;
    Pack x = *reinterpret_cast<const Pack*>(src + at), y = *reinterpret_cast<const Pack*>(src + at + half);
#pragma unroll
    for (int e = 0; e < W; e++) {
      const floatx2 r = cs[at + e];
      const float a = rp_load(x.v[e]), b = rp_load(y.v[e]);
      x.v[e] = rp_store<T>(a * r[0] - b * r[1]);
      y.v[e] = rp_store<T>(a * r[1] + b * r[0]);
    }
    *reinterpret_cast<Pack*>(dst + at) = x;
    *reinterpret_cast<Pack*>(dst + at + half) = y;
  }
}

// One token per workgroup: its angles into LDS, then its head rows.
template <typename T, typename F, bool INTER, int W>
__global__ __launch_bounds__(RP_THREADS) void rope_kernel(RopeRows x, const int* __restrict__ positions,
                                                          const F* __restrict__ freq, int half, int D, float mul,
                                                          float sin_mul) {
  __shared__ floatx2 cs[RP_MAX_PAIRS];
  const long long tok = blockIdx.x;
  const int pos = positions[tok];
  for (int i = threadIdx.x; i < half; i += RP_THREADS) cs[i] = rp_angle(pos, (double)freq[i], mul, sin_mul);
  __syncthreads();
  const int n_pair = half / W, per_row = n_pair + (D - 2 * half) / W;
  const T* src = static_cast<const T*>(x.src) + tok * x.src_token;
  T* dst = static_cast<T*>(x.dst) + tok * x.dst_token;
  for (int i = threadIdx.x; i < x.heads * per_row; i += RP_THREADS) {
    const int h = i / per_row;
    rp_item<T, INTER, W>(src + h * x.src_head, dst + h * x.dst_head, i - h * per_row, n_pair, half, cs);
  }
}

// The serving form: queries rotated into q_out, keys rotated and values copied into the cache rows that `slots` names
// (a slot outside [0, num_slots): the token's key and value are dropped).
template <typename T, typename F, bool INTER, int W>
__global__ __launch_bounds__(RP_THREADS) void rope_append_kernel(RopeRows q, RopeRows k, RopeRows v,
                                                                 const int* __restrict__ positions,
                                                                 const F* __restrict__ freq, const long long* __restrict__ slots,
                                                                 long long num_slots, int half, float mul) {
  constexpr int D = 128;
  __shared__ floatx2 cs[D / 2];
  const long long tok = blockIdx.x;
  const int pos = positions[tok];
  const long long slot = slots[tok];
  if ((int)threadIdx.x < half) cs[threadIdx.x] = rp_angle(pos, (double)freq[threadIdx.x], mul, mul);
  __syncthreads();
  const int n_pair = half / W, per_row = n_pair + (D - 2 * half) / W;
  const bool keep = slot >= 0 && slot < num_slots;
  const int rows = q.heads + (keep ? k.heads : 0);
  for (int i = threadIdx.x; i < rows * per_row; i += RP_THREADS) {
    const int h = i / per_row, item = i - h * per_row;
    if (h < q.heads)
      rp_item<T, INTER, W>(static_cast<const T*>(q.src) + tok * q.src_token + h * q.src_head,
                           static_cast<T*>(q.dst) + tok * q.dst_token + h * q.dst_head, item, n_pair, half, cs);
    else
      rp_item<T, INTER, W>(static_cast<const T*>(k.src) + tok * k.src_token + (h - q.heads) * k.src_head,
                           static_cast<T*>(k.dst) + slot * k.dst_token + (h - q.heads) * k.dst_head, item, n_pair, half, cs);
  }
  if (!keep) return;
  const T* vs = static_cast<const T*>(v.src) + tok * v.src_token;
  T* vd = static_cast<T*>(v.dst) + slot * v.dst_token;
  struct alignas(W == 1 ? sizeof(T) : W * sizeof(T)) Pack { T e[W]; };
  for (int i = threadIdx.x; i < v.heads * (D / W); i += RP_THREADS) {
    const int h = i / (D / W), e = (i - h * (D / W)) * W;
    *reinterpret_cast<Pack*>(vd + h * v.dst_head + e) = *reinterpret_cast<const Pack*>(vs + h * v.src_head + e);
  }
}

// whether every row of `x` starts on a 16-byte border
static bool rows16(const RopeRows& x, int elem) {
  const long long unit = 16 / elem;
  return aligned16(x.src) && aligned16(x.dst) && x.src_token % unit == 0 && x.src_head % unit == 0 && x.dst_token % unit == 0 &&
         x.dst_head % unit == 0;
}

template <typename T, typename F, bool INTER>
static int rope_launch(const RopeRows& x, const int* pos, const F* freq, int half, int D, float mul, float sin_mul, int64_t tokens,
                       hipStream_t s) {
  constexpr int V = 16 / sizeof(T);           // elements of 16 bytes
  constexpr int W = INTER ? V / 2 : V;        // pairs (or elements of a half) per item
  dim3 grid((unsigned)tokens), block(RP_THREADS);
  const bool wide = rows16(x, sizeof(T)) && half % W == 0 && (D - 2 * half) % W == 0;
  if (wide)
    hipLaunchKernelGGL((rope_kernel<T, F, INTER, W>), grid, block, 0, s, x, pos, freq, half, D, mul, sin_mul);
  else
    hipLaunchKernelGGL((rope_kernel<T, F, INTER, 1>), grid, block, 0, s, x, pos, freq, half, D, mul, sin_mul);
  return check_launch("rope_kernel", grid, block, 0);
}

template <typename T, typename F, bool INTER>
static int rope_append_launch(const RopeRows& q, const RopeRows& k, const RopeRows& v, const int* pos, const F* freq,
                              const int64_t* slots, long long num_slots, int half, float mul, int64_t tokens, hipStream_t s) {
  constexpr int V = 16 / sizeof(T), W = INTER ? V / 2 : V;
  dim3 grid((unsigned)tokens), block(RP_THREADS);
  const bool wide = rows16(q, sizeof(T)) && rows16(k, sizeof(T)) && rows16(v, sizeof(T)) && half % W == 0;
  const long long* sl = reinterpret_cast<const long long*>(slots);
  if (wide)
    hipLaunchKernelGGL((rope_append_kernel<T, F, INTER, W>), grid, block, 0, s, q, k, v, pos, freq, sl, num_slots, half, mul);
  else
    hipLaunchKernelGGL((rope_append_kernel<T, F, INTER, 1>), grid, block, 0, s, q, k, v, pos, freq, sl, num_slots, half, mul);
  return check_launch("rope_append_kernel", grid, block, 0);
}

}  // namespace mi355

using namespace mi355;

static bool good_stride(int64_t v) { return v >= 0 && v < (1ll << 40); }

template <typename T, typename F>
static int rope_any(const RopeRows& x, const int32_t* pos, const void* freq, int half, int D, int interleaved, float mul,
                    float sin_mul, int64_t tokens, hipStream_t s) {
  const F* f = static_cast<const F*>(freq);
  return interleaved ? rope_launch<T, F, true>(x, pos, f, half, D, mul, sin_mul, tokens, s)
                     : rope_launch<T, F, false>(x, pos, f, half, D, mul, sin_mul, tokens, s);
}

extern "C" int mi355_rope(const void* x, void* out, const int32_t* positions, const void* inv_freq, int freq_is_f64, int64_t tokens,
                          int64_t heads, int64_t D, int64_t rotary_dim, const int64_t* x_strides, const int64_t* out_strides,
                          int interleaved, int inverse, float scale, int dtype, void* stream) {
  const char* fn = "rope";
  if (!x || !out || !positions || !inv_freq || !x_strides || !out_strides) return fail(-MI355_E_NULL, "%s: null pointer", fn);
  if (tokens <= 0 || tokens >= (1ll << 24) || heads <= 0 || heads > 65535 || D <= 0 || D > 65536 || rotary_dim <= 0 || rotary_dim > D ||
      rotary_dim % 2 || rotary_dim > 2 * RP_MAX_PAIRS || heads * D > (1ll << 30))
    return fail(-MI355_E_SHAPE, "%s: bad sizes tokens=%lld heads=%lld D=%lld rotary_dim=%lld (even, at most D and %d)", fn,
                (long long)tokens, (long long)heads, (long long)D, (long long)rotary_dim, 2 * RP_MAX_PAIRS);
  for (int i = 0; i < 2; i++)
    if (!good_stride(x_strides[i]) || !good_stride(out_strides[i])) return fail(-MI355_E_SHAPE, "%s: strides must be in [0, 2^40)", fn);
  if (!isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be finite", fn);
  const RopeRows r{x, out, x_strides[0], x_strides[1], out_strides[0], out_strides[1], (int)heads};
  const float sin_mul = inverse ? -scale : scale;
  const int half = (int)rotary_dim / 2;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MI355_ROPE(T)                                                                                                 \
  (freq_is_f64 ? rope_any<T, double>(r, positions, inv_freq, half, (int)D, interleaved, scale, sin_mul, tokens, s)    \
               : rope_any<T, float>(r, positions, inv_freq, half, (int)D, interleaved, scale, sin_mul, tokens, s))
  if (dtype == MI355_F16) return MI355_ROPE(half_t);
  if (dtype == MI355_BF16) return MI355_ROPE(__bf16);
  if (dtype == MI355_F32) return MI355_ROPE(float);
#undef MI355_ROPE
  return fail(-MI355_E_DTYPE, "%s: dtype %d (MI355_F16, MI355_BF16 or MI355_F32)", fn, dtype);
}

template <typename T, typename F>
static int append_any(const RopeRows& q, const RopeRows& k, const RopeRows& v, const int32_t* pos, const void* freq,
                      const int64_t* slots, long long num_slots, int half, int interleaved, float mul, int64_t tokens, hipStream_t s) {
  const F* f = static_cast<const F*>(freq);
  return interleaved ? rope_append_launch<T, F, true>(q, k, v, pos, f, slots, num_slots, half, mul, tokens, s)
                     : rope_append_launch<T, F, false>(q, k, v, pos, f, slots, num_slots, half, mul, tokens, s);
}

extern "C" int mi355_rope_kv_append(const void* q, const void* k_new, const void* v_new, void* q_out, void* k_cache, void* v_cache,
                                    const int32_t* positions, const void* inv_freq, int freq_is_f64, const int64_t* slots,
                                    int64_t tokens, int64_t num_q_heads, int64_t num_kv_heads, int64_t D, int64_t rotary_dim,
                                    int64_t num_slots, const int64_t* q_strides, const int64_t* k_strides, const int64_t* v_strides,
                                    int interleaved, float scale, int dtype, void* stream) {
  const char* fn = "rope_kv_append";
  if (!q || !k_new || !v_new || !q_out || !k_cache || !v_cache || !positions || !inv_freq || !slots || !q_strides || !k_strides ||
      !v_strides)
    return fail(-MI355_E_NULL, "%s: null pointer", fn);
  if (D != 128) return fail(-MI355_E_SHAPE, "%s: head dim %lld not supported (only 128)", fn, (long long)D);
  if (tokens <= 0 || tokens >= (1ll << 24) || num_q_heads <= 0 || num_kv_heads <= 0 || num_q_heads > 65535 || num_kv_heads > 65535 ||
      rotary_dim <= 0 || rotary_dim > D || rotary_dim % 2 || num_slots <= 0 || num_slots > (1ll << 34))
    return fail(-MI355_E_SHAPE, "%s: bad sizes tokens=%lld hq=%lld hkv=%lld rotary_dim=%lld slots=%lld", fn, (long long)tokens,
                (long long)num_q_heads, (long long)num_kv_heads, (long long)rotary_dim, (long long)num_slots);
  for (int i = 0; i < 2; i++)
    if (!good_stride(q_strides[i]) || !good_stride(k_strides[i]) || !good_stride(v_strides[i]))
      return fail(-MI355_E_SHAPE, "%s: strides must be in [0, 2^40)", fn);
  if (!isfinite(scale)) return fail(-MI355_E_SHAPE, "%s: scale must be finite", fn);
  const long long qr = num_q_heads * 128, kr = num_kv_heads * 128;
  const RopeRows rq{q, q_out, q_strides[0], q_strides[1], qr, 128, (int)num_q_heads};
  const RopeRows rk{k_new, k_cache, k_strides[0], k_strides[1], kr, 128, (int)num_kv_heads};
  const RopeRows rv{v_new, v_cache, v_strides[0], v_strides[1], kr, 128, (int)num_kv_heads};
  const int half = (int)rotary_dim / 2;
  hipStream_t s = reinterpret_cast<hipStream_t>(stream);
#define MI355_APPEND(T)                                                                                                   \
  (freq_is_f64 ? append_any<T, double>(rq, rk, rv, positions, inv_freq, slots, num_slots, half, interleaved, scale, tokens, s) \
               : append_any<T, float>(rq, rk, rv, positions, inv_freq, slots, num_slots, half, interleaved, scale, tokens, s))
  if (dtype == MI355_F16) return MI355_APPEND(half_t);
  if (dtype == MI355_BF16) return MI355_APPEND(__bf16);
#undef MI355_APPEND
  return fail(-MI355_E_DTYPE, "%s: dtype %d (MI355_F16 or MI355_BF16)", fn, dtype);
}
