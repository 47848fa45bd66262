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
// The op reads and writes every element once (HBM bound): 16 bytes per lane where rows allow it, 8 where only those fit
// (16384 tokens x 8 heads of 80 elements, 40 of them turned: 37 us, 59 element by element), else one element.
// Measured: 16384 tokens x 32 x 128 bf16 48 us (5.6 TB/s), 8000 tokens with the append 32 us of which a part comes out of the
// memory-side cache (cold: 43 us, 4.6 TB/s), 64 tokens with the append 4 us (a launch and two trips to memory).
#include "common.hpp"
#include <math.h>
#include <type_traits>

namespace mi355 {

constexpr int RP_THREADS = 256;
constexpr int RP_MAX_PAIRS = 512;  // R / 2
constexpr int RP_ANGLES = 1024;    // angles per workgroup: its tokens times R / 2

// One operand: where a token's head rows lie, in elements; the D elements of a row are contiguous.
struct RopeRows {
  const void* src;
  void* dst;
  long long src_token, src_head, dst_token, dst_head;
  int heads;
};

// (cos, sin) of pos * freq, both times `mul`
__device__ __forceinline__ floatx2 rp_angle(int pos, double freq, float mul, float sin_mul) {
  const double turns = (double)pos * (freq * 0.15915494309189533577);
  const float rest = (float)(turns - rint(turns));
  float s, c;
  sincospif(2.f * rest, &s, &c);
  return floatx2{c * mul, s * sin_mul};
}

// A head row as work items of V elements (16 bytes, 8 bytes, or one element, which assumes no alignment): n_pair items of W
// pairs each (two places of V elements for halves), then items that copy V elements of the rest.
template <typename T, bool INTER, int V>
struct RopeItems {
  static constexpr int W = INTER ? (V + 1) / 2 : V;       // pairs
  static constexpr int P = INTER ? 2 * W : W;             // elements at one place
  struct alignas(V * sizeof(T)) Place { T v[P]; };
  struct alignas(V * sizeof(T)) Rest { T v[V]; };
  int n_pair, per_row, half;

  __device__ __forceinline__ RopeItems(int half_, int D) : n_pair(half_ / W), per_row(half_ / W + (D - 2 * half_) / V), half(half_) {}
  static bool fits(int half, int D) { return half % W == 0 && (D - 2 * half) % V == 0; }

  static __device__ __forceinline__ void copy(const T* src, T* dst, int at) {
    *reinterpret_cast<Rest*>(dst + at) = *reinterpret_cast<const Rest*>(src + at);
  }
  __device__ __forceinline__ void run(const T* __restrict__ src, T* __restrict__ dst, int item, const floatx2* cs) const {
    if (item >= n_pair) {
      copy(src, dst, 2 * half + (item - n_pair) * V);
    } else if constexpr (INTER) {
      Place x = *reinterpret_cast<const Place*>(src + item * P);
#pragma unroll
      for (int e = 0; e < W; e++) {
        const floatx2 r = cs[item * W + e];
        const float a = (float)x.v[2 * e], b = (float)x.v[2 * e + 1];
        x.v[2 * e] = (T)(a * r[0] - b * r[1]);
        x.v[2 * e + 1] = (T)(a * r[1] + b * r[0]);
      }
      *reinterpret_cast<Place*>(dst + item * P) = x;
    } else {
      const int at = item * W;
      Place x = *reinterpret_cast<const Place*>(src + at), y = *reinterpret_cast<const Place*>(src + at + half);
#pragma unroll
      for (int e = 0; e < W; e++) {
        const floatx2 r = cs[at + e];
        const float a = (float)x.v[e], b = (float)y.v[e];
        x.v[e] = (T)(a * r[0] - b * r[1]);
        y.v[e] = (T)(a * r[1] + b * r[0]);
      }
      *reinterpret_cast<Place*>(dst + at) = x;
      *reinterpret_cast<Place*>(dst + at + half) = y;
    }
  }
};

// The angles of a workgroup's tokens, `half` of them each.
template <typename F>
__device__ __forceinline__ void rope_angles(floatx2* cs, const int* __restrict__ positions, const F* __restrict__ freq, long long tok0,
                                            int tokens, int half, float mul, float sin_mul) {
  for (int i = threadIdx.x; i < tokens * half; i += RP_THREADS) {
    const int t = i / half;
    cs[i] = rp_angle(positions[tok0 + t], (double)freq[i - t * half], mul, sin_mul);
  }
  __syncthreads();
}

// `per_wg` neighbouring tokens per workgroup.
template <typename T, typename F, bool INTER, int V>
__global__ __launch_bounds__(RP_THREADS) void rope_kernel(RopeRows x, const int* __restrict__ positions,
                                                          const F* __restrict__ freq, int half, int D, float mul,
                                                          float sin_mul, int num_tokens, int per_wg) {
  __shared__ floatx2 cs[RP_ANGLES];
  const long long tok0 = (long long)blockIdx.x * per_wg;
  const int tokens = num_tokens - tok0 < per_wg ? (int)(num_tokens - tok0) : per_wg;
  rope_angles(cs, positions, freq, tok0, tokens, half, mul, sin_mul);
  const RopeItems<T, INTER, V> items(half, D);
  const int per_token = x.heads * items.per_row;
  for (int i = threadIdx.x; i < tokens * per_token; i += RP_THREADS) {
    const int row = i / items.per_row, t = tokens == 1 ? 0 : row / x.heads, h = row - t * x.heads;
    items.run(static_cast<const T*>(x.src) + (tok0 + t) * x.src_token + h * x.src_head,
              static_cast<T*>(x.dst) + (tok0 + t) * x.dst_token + h * x.dst_head, i - row * items.per_row, cs + t * half);
  }
}

// The serving form: queries rotated into q_out, keys rotated and values copied into the cache rows that `slots` names
// (a slot outside [0, num_slots): the token's key and value are dropped).
template <typename T, typename F, bool INTER, int V>
__global__ __launch_bounds__(RP_THREADS) void rope_append_kernel(RopeRows q, RopeRows k, RopeRows v,
                                                                 const int* __restrict__ positions,
                                                                 const F* __restrict__ freq, const long long* __restrict__ slots,
                                                                 long long num_slots, int half, float mul, int num_tokens, int per_wg) {
  constexpr int D = 128;
  __shared__ floatx2 cs[RP_ANGLES];
  const long long tok0 = (long long)blockIdx.x * per_wg;
  const int tokens = num_tokens - tok0 < per_wg ? (int)(num_tokens - tok0) : per_wg;
  rope_angles(cs, positions, freq, tok0, tokens, half, mul, mul);
  typedef RopeItems<T, INTER, V> Items;
  const Items items(half, D);
  const int turned = q.heads + k.heads;
  for (int i = threadIdx.x; i < tokens * turned * items.per_row; i += RP_THREADS) {
    const int row = i / items.per_row, item = i - row * items.per_row, t = tokens == 1 ? 0 : row / turned, h = row - t * turned;
    const long long tok = tok0 + t;
    if (h < q.heads) {
      items.run(static_cast<const T*>(q.src) + tok * q.src_token + h * q.src_head,
                static_cast<T*>(q.dst) + tok * q.dst_token + h * q.dst_head, item, cs + t * half);
    } else {
      const long long slot = slots[tok];
      if (slot >= 0 && slot < num_slots)
        items.run(static_cast<const T*>(k.src) + tok * k.src_token + (h - q.heads) * k.src_head,
                  static_cast<T*>(k.dst) + slot * k.dst_token + (h - q.heads) * k.dst_head, item, cs + t * half);
    }
  }
  constexpr int pieces = D / V;
  for (int i = threadIdx.x; i < tokens * v.heads * pieces; i += RP_THREADS) {
    const int row = i / pieces, t = tokens == 1 ? 0 : row / v.heads, h = row - t * v.heads;
    const long long tok = tok0 + t, slot = slots[tok];
    if (slot >= 0 && slot < num_slots)
      Items::copy(static_cast<const T*>(v.src) + tok * v.src_token + h * v.src_head,
                  static_cast<T*>(v.dst) + slot * v.dst_token + h * v.dst_head, (i - row * pieces) * V);
  }
}

// whether every row of `x` starts on a border of `unit` elements
static bool rows_on(const RopeRows& x, int unit, int elem) {
  const uintptr_t bytes = (uintptr_t)unit * elem;
  return reinterpret_cast<uintptr_t>(x.src) % bytes == 0 && reinterpret_cast<uintptr_t>(x.dst) % bytes == 0 && x.src_token % unit == 0 &&
         x.src_head % unit == 0 && x.dst_token % unit == 0 && x.dst_head % unit == 0;
}

// Tokens per workgroup: one, unless a token has less than an item per thread (16384 tokens of one head of 128: 14 us with
// four tokens, 23 with one; of 32 heads 102 with four, 96 with one), as long as that leaves the chip full of workgroups.
static int rope_per_wg(int64_t tokens, int64_t items_per_token, int half) {
  int64_t n = RP_THREADS / items_per_token;
  n = n < tokens / 2048 ? n : tokens / 2048;
  n = n < RP_ANGLES / half ? n : RP_ANGLES / half;
  return n < 1 ? 1 : (int)n;
}

template <typename T, typename F, bool INTER, int V>
static int rope_launch_as(const RopeRows& x, const int* pos, const F* freq, int half, int D, float mul, float sin_mul, int64_t tokens,
                          hipStream_t s) {
  const int per_wg = rope_per_wg(tokens, (int64_t)x.heads * D / RopeItems<T, INTER, V>::P, half);
  dim3 grid((unsigned)((tokens + per_wg - 1) / per_wg)), block(RP_THREADS);
  hipLaunchKernelGGL((rope_kernel<T, F, INTER, V>), grid, block, 0, s, x, pos, freq, half, D, mul, sin_mul, (int)tokens, per_wg);
  return check_launch("rope_kernel", grid, block, 0);
}

// The widest accesses that the rows, the rotated part and the rest allow.  A head of 80 with 40 rotated elements has 8-byte ones.
template <typename T, typename F, bool INTER>
static int rope_launch(const RopeRows& x, const int* pos, const F* freq, int half, int D, float mul, float sin_mul, int64_t tokens,
                       hipStream_t s) {
  constexpr int V16 = 16 / sizeof(T), V8 = V16 / 2;
  if (rows_on(x, V16, sizeof(T)) && RopeItems<T, INTER, V16>::fits(half, D))
    return rope_launch_as<T, F, INTER, V16>(x, pos, freq, half, D, mul, sin_mul, tokens, s);
  if (rows_on(x, V8, sizeof(T)) && RopeItems<T, INTER, V8>::fits(half, D))
    return rope_launch_as<T, F, INTER, V8>(x, pos, freq, half, D, mul, sin_mul, tokens, s);
  return rope_launch_as<T, F, INTER, 1>(x, pos, freq, half, D, mul, sin_mul, tokens, s);
}

template <typename T, typename F, bool INTER, int V>
static int rope_append_as(const RopeRows& q, const RopeRows& k, const RopeRows& v, const int* pos, const F* freq, const int64_t* slots,
                          long long num_slots, int half, float mul, int64_t tokens, hipStream_t s) {
  const int per_wg = rope_per_wg(tokens, (int64_t)(q.heads + 2 * k.heads) * 128 / RopeItems<T, INTER, V>::P, half);
  dim3 grid((unsigned)((tokens + per_wg - 1) / per_wg)), block(RP_THREADS);
  hipLaunchKernelGGL((rope_append_kernel<T, F, INTER, V>), grid, block, 0, s, q, k, v, pos, freq, reinterpret_cast<const long long*>(slots),
                     num_slots, half, mul, (int)tokens, per_wg);
  return check_launch("rope_append_kernel", grid, block, 0);
}

template <typename T, typename F, bool INTER>
static int rope_append_launch(const RopeRows& q, const RopeRows& k, const RopeRows& v, const int* pos, const F* freq,
                              const int64_t* slots, long long num_slots, int half, float mul, int64_t tokens, hipStream_t s) {
  constexpr int V16 = 16 / sizeof(T), V8 = V16 / 2;
  auto on = [&](int unit) { return rows_on(q, unit, sizeof(T)) && rows_on(k, unit, sizeof(T)) && rows_on(v, unit, sizeof(T)); };
  if (on(V16) && RopeItems<T, INTER, V16>::fits(half, 128))
    return rope_append_as<T, F, INTER, V16>(q, k, v, pos, freq, slots, num_slots, half, mul, tokens, s);
  if (on(V8) && RopeItems<T, INTER, V8>::fits(half, 128))
    return rope_append_as<T, F, INTER, V8>(q, k, v, pos, freq, slots, num_slots, half, mul, tokens, s);
  return rope_append_as<T, F, INTER, 1>(q, k, v, pos, freq, slots, num_slots, half, mul, tokens, s);
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
