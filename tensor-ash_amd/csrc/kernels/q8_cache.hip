// The 8-bit K/V cache for gfx950: quantising rows as they are written, and
// reading positions back into dense caches.
//
// Mathematics.  A row x of dh values (one kv head, one position; K and V
// apart) is held as a scale s and codes c_d in -127 .. 127, and stands for
// s * c_d:
//   s = the smallest number of 8 significant bits >= max(max|x| / 127, 2^-100)
//   c_d = x_d / s to nearest, ties to even.
// s having 8 bits, s * 127 (15 bits) and s * (c + 1/2) (16 bits) are exact
// in f32, so both decisions are made exactly: s from the f32 quotient cut to
// 8 bits and one comparison, c from the f32 quotient (q8_code).  s * c is exact
// in f32 as well.  A row that holds an infinity or a NaN gets a NaN scale: all
// of it reads back as NaN.  Half a step is at most 1/254 * (1 + 2^-7) of the
// row's largest value.
//
// Both kernels are bound by HBM on long runs of positions (16384 of 8 heads of
// 128, f16: written in 17.9 us, 101 MB at 5.6 TB/s, the vector units busy in 90%
// of it; read back in 16.6 us, the codes still in the caches) and by their
// launch on short ones (one token: 3.0 us).  A workgroup writes one block of 32
// positions of one head, so that its bytes are its own: V's codes lie across
// positions, and no two workgroups write one 16-byte piece.
#include "common.h"

namespace {

constexpr uint32_t kThreads = 256;
constexpr uint32_t kRow = 36; // bytes of a head dimension's 32 codes in LDS, padded against bank conflicts
constexpr float kLeastScale = 7.888609052210118e-31f; // 2^-100

typedef f32x4 f32x4u __attribute__((aligned(4)));
typedef f16x8 f16x8u __attribute__((aligned(2)));
typedef f16x4 f16x4u __attribute__((aligned(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

// N consecutive values (N a multiple of 8) from any element offset.
template <int N, bool F16> TA_DEVICE void load_row(const void *src, uint64_t at, float (&x)[N]) {
  if constexpr (F16) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const f16x8 t = *reinterpret_cast<const f16x8u *>(static_cast<const _Float16 *>(src) + at + 8 * i);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        x[8 * i + c] = (float)t[c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4 t = *reinterpret_cast<const f32x4u *>(static_cast<const float *>(src) + at + 4 * i);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x[4 * i + c] = t[c];
    }
  }
}

// The scale of a row whose largest magnitude is `top` (NaN where the row is
// not finite).
TA_DEVICE float q8_scale(float top) {
  const float least = fmaxf(top / 127.0f, kLeastScale);
  const uint32_t cut = __float_as_uint(least) & 0xFFFF0000u;
  // cut <= least rounded; the next 8-bit number where 127 * cut is short
  const uint32_t s = __uint_as_float(cut) * 127.0f < top ? cut + 0x10000u : cut;
  return top < __builtin_inff() ? __uint_as_float(s) : __builtin_nanf("");
}

// x / s to nearest, ties to even, as kMagic + c, whose low byte is c.  The
// quotient is taken to f32's nearest (rest = x - s q has ten bits at most and is
// exact, so the second fma sees the true quotient but for 2^-46 of it), and then
// rounded to a whole number.  The two roundings are one: a tie t = c + 1/2 has 8
// bits, s t has 16, so x differs from s t by at least a unit of its own, x / s
// from t by more than 2^-24 of it, and that is more than half a unit of t.
// Four steps a value: the correction of a single product by its remainder's
// sign took eleven, and the kernel 23.5 us for 17.7 (sizes at the top).
constexpr float kMagic = 12582912.0f; // 1.5 * 2^23
TA_DEVICE uint32_t q8_code(float x, float s, float inv) {
  const float q = x * inv;
  return __float_as_uint(fmaf(fmaf(-s, q, x), inv, q) + kMagic);
}

// One block of 32 positions of a kv head: 8 threads to a row, DH / 8 values
// each, K then V.
template <int DH, bool F16> TA_DEVICE void q8_write(const Q8WriteArgs &p) {
  constexpr int N = DH / 8, WORDS = N / 4;
  const uint32_t tid = threadIdx.x, key = tid >> 3, part = tid & 7u, head = blockIdx.y;
  const uint64_t pos0 = (uint64_t)p.pos_base + (p.pos_addr ? *p.pos_addr : 0u);
  const uint64_t block = pos0 / TA_Q8_BLOCK + blockIdx.x;
  if (block >= p.blocks) // also a start past the cache
    return;
  const uint64_t first = block * TA_Q8_BLOCK, at = first + key;
  const bool mine = at >= pos0 && at < pos0 + p.tokens && at < p.t_max;
  if (first >= pos0 + p.tokens)
    return;
  const uint64_t t = mine ? at - pos0 : 0u; // a row that exists
  uint8_t *rec = p.cache + ((uint64_t)head * p.blocks + block) * ta_q8_record(DH);
  const uint32_t slot = ta_q8_slot(key);
  float x[2][N];
  load_row<N, F16>(p.k, p.k_offset + t * p.k_stride + (uint64_t)head * DH + part * N, x[0]);
  load_row<N, F16>(p.v, p.v_offset + t * p.v_stride + (uint64_t)head * DH + part * N, x[1]);
  uint32_t code[2][WORDS];
  float scale[2];
#pragma unroll
  for (int kv = 0; kv < 2; ++kv) {
    float top = 0.0f, sum = 0.0f;
#pragma unroll
    for (int i = 0; i < N; ++i) {
      top = fmaxf(top, fabsf(x[kv][i]));
      sum = fmaf(x[kv][i], 0.0f, sum); // NaN where a value is not finite
    }
    top += sum;
#pragma unroll
    for (int o = 1; o < 8; o <<= 1) {
      const float other = __shfl_xor(top, o);
      top = top == top && other == other ? fmaxf(top, other) : __builtin_nanf("");
    }
    const float s = q8_scale(top);
    scale[kv] = s;
    const bool finite = s == s;
    const float inv = 1.0f / s;
    uint32_t c[N];
#pragma unroll
    for (int i = 0; i < N; ++i)
      c[i] = q8_code(x[kv][i], s, inv);
#pragma unroll
    for (int w = 0; w < WORDS; ++w) {
      const uint32_t lo = __builtin_amdgcn_perm(c[4 * w + 1], c[4 * w], 0x0c0c0400u);
      const uint32_t hi = __builtin_amdgcn_perm(c[4 * w + 3], c[4 * w + 2], 0x04000c0cu);
      code[kv][w] = finite ? lo | hi : 0u;
    }
  }
  if (mine) {
    if constexpr (N == 16)
      *reinterpret_cast<u32x4 *>(rec + (part * 32u + key) * 16u) =
          u32x4{code[0][0], code[0][1], code[0][2], code[0][3]};
    else
      *reinterpret_cast<u32x2 *>(rec + ((part / 2u) * 32u + key) * 16u + (part & 1u) * 8u) =
          u32x2{code[0][0], code[0][1]};
    if (part < 2u) {
      const float s = part == 0 ? scale[0] : scale[1];
      reinterpret_cast<uint16_t *>(rec + 64u * DH + part * 64u)[slot] = (uint16_t)(__float_as_uint(s) >> 16);
    }
  }
  // V codes lie by head dimension.  A whole block is turned in LDS and
  // leaves in 16-byte pieces; of a block in part only its own bytes may be
  // written.
  uint8_t *vcodes = rec + 32u * DH;
  const bool whole = first >= pos0 && first + TA_Q8_BLOCK <= pos0 + p.tokens && first + TA_Q8_BLOCK <= p.t_max;
  if (whole) {
    __shared__ __attribute__((aligned(16))) uint8_t turn[kRow * DH];
#pragma unroll
    for (int i = 0; i < N; ++i)
      turn[(part * N + i) * kRow + slot] = (uint8_t)(code[1][i / 4] >> (8 * (i & 3)));
    __syncthreads();
    for (uint32_t i = tid; i < 2u * DH; i += kThreads) {
      const uint32_t *src = reinterpret_cast<const uint32_t *>(turn + i / 2u * kRow + (i & 1u) * 16u);
      reinterpret_cast<u32x4 *>(vcodes)[i] = u32x4{src[0], src[1], src[2], src[3]};
    }
  } else if (mine) {
#pragma unroll
    for (int i = 0; i < N; ++i)
      vcodes[(part * N + i) * 32u + slot] = (uint8_t)(code[1][i / 4] >> (8 * (i & 3)));
  }
}

TA_DEVICE float code_value(uint32_t word, int byte, float s) { return (float)(int8_t)(word >> (8 * byte)) * s; }
TA_DEVICE float scale_value(uint32_t half) { return __uint_as_float(half << 16); }

// Rows whose largest magnitude is one of f16's top eight have the scale 516,
// and the code 127 then stands for 65532, which f16 would round to infinity:
// as f16 it is f16's largest, 65504.  (No other scale and code give 65532.)
constexpr float kF16TopScale = 516.0f, kF16Top = 65504.0f;
TA_DEVICE bool f16_top(const float (&s)[4]) {
  return s[0] == kF16TopScale || s[1] == kF16TopScale || s[2] == kF16TopScale || s[3] == kF16TopScale;
}
TA_DEVICE float f16_within(float v) { return fabsf(v) == 127.0f * kF16TopScale ? copysignf(kF16Top, v) : v; }

// 128 positions (four blocks) of a kv head.
template <int DH, bool F16> TA_DEVICE void q8_read(const Q8ReadArgs &p) {
  __shared__ __attribute__((aligned(16))) uint8_t turn[4 * DH * kRow];
  const uint32_t tid = threadIdx.x, head = blockIdx.y;
  const uint32_t group = p.first / TA_Q8_READ_KEYS + blockIdx.x;
  const uint64_t end = (uint64_t)p.first + p.n;
  const uint8_t *base = p.cache + (uint64_t)head * p.blocks * ta_q8_record(DH);
  // V codes of the blocks that exist, one 16-byte piece per thread and step
  for (uint32_t i = tid; i < 4u * 2u * DH; i += kThreads) {
    const uint32_t b = i / (2u * DH), at = i % (2u * DH);
    if (group * 4u + b < p.blocks) {
      const u32x4 c = *reinterpret_cast<const u32x4 *>(base + (uint64_t)(group * 4u + b) * ta_q8_record(DH) +
                                                       32u * DH + at * 16u);
      uint32_t *dst = reinterpret_cast<uint32_t *>(turn + (b * DH + at / 2u) * kRow + (at & 1u) * 16u);
#pragma unroll
      for (int w = 0; w < 4; ++w)
        dst[w] = c[w];
    }
  }
  // K: four keys (their 16-byte pieces lie together) x 16 head dimensions a
  // thread; consecutive threads take consecutive keys of one row of kt.
#pragma unroll
  for (uint32_t part = tid >> 5; part < DH / 16u; part += kThreads / 32u) {
    const uint32_t quad = tid & 31u, block = group * 4u + quad / 8u, a = quad & 7u;
    const uint64_t pos = (uint64_t)group * TA_Q8_READ_KEYS + 4u * quad;
    if (pos + 4u <= p.first || pos >= end || block >= p.blocks)
      continue;
    const uint8_t *rec = base + (uint64_t)block * ta_q8_record(DH);
    u32x4 c[4];
#pragma unroll
    for (int r = 0; r < 4; ++r)
      c[r] = *reinterpret_cast<const u32x4 *>(rec + (part * 32u + 4u * a + r) * 16u);
    const u32x2 raw = *reinterpret_cast<const u32x2 *>(rec + 64u * DH + ta_q8_slot(4u * a) * 2u);
    const float s[4] = {scale_value(raw[0] & 0xFFFFu), scale_value(raw[0] >> 16), scale_value(raw[1] & 0xFFFFu),
                        scale_value(raw[1] >> 16)};
    const bool all = pos >= p.first && pos + 4u <= end, top = F16 && f16_top(s);
    const uint64_t row0 = ((uint64_t)head * DH + part * 16u) * p.t_dst + pos;
#pragma unroll
    for (int d = 0; d < 16; ++d) {
      f32x4 v;
#pragma unroll
      for (int r = 0; r < 4; ++r)
        v[r] = code_value(c[r][d / 4], d & 3, s[r]);
      if (top) {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = f16_within(v[r]);
      }
      const uint64_t at = row0 + (uint64_t)d * p.t_dst;
      if (all) {
        if constexpr (F16)
          *reinterpret_cast<f16x4u *>(static_cast<_Float16 *>(p.kt) + at) = __builtin_convertvector(v, f16x4);
        else
          *reinterpret_cast<f32x4u *>(static_cast<float *>(p.kt) + at) = v;
      } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
          if (pos + r >= p.first && pos + r < end) {
            if constexpr (F16)
              static_cast<_Float16 *>(p.kt)[at + r] = (_Float16)v[r];
            else
              static_cast<float *>(p.kt)[at + r] = v[r];
          }
      }
    }
  }
  __syncthreads();
  // V: four keys x eight head dimensions a thread.
  constexpr uint32_t PARTS = DH / 8u; // threads to a row of v
#pragma unroll 2
  for (uint32_t i = tid; i < 32u * PARTS; i += kThreads) {
    const uint32_t part = i % PARTS, quad = i / PARTS, b = quad / 8u, block = group * 4u + b, a = quad & 7u;
    const uint64_t pos = (uint64_t)group * TA_Q8_READ_KEYS + 4u * quad;
    if (pos + 4u <= p.first || pos >= end || block >= p.blocks)
      continue;
    const uint32_t slot = ta_q8_slot(4u * a);
    uint32_t c[8];
#pragma unroll
    for (int d = 0; d < 8; ++d)
      c[d] = *reinterpret_cast<const uint32_t *>(turn + (b * DH + part * 8u + d) * kRow + slot);
    const u32x2 raw = *reinterpret_cast<const u32x2 *>(base + (uint64_t)block * ta_q8_record(DH) + 64u * DH + 64u +
                                                       slot * 2u);
    const float s[4] = {scale_value(raw[0] & 0xFFFFu), scale_value(raw[0] >> 16), scale_value(raw[1] & 0xFFFFu),
                        scale_value(raw[1] >> 16)};
    const bool top = F16 && f16_top(s);
#pragma unroll
    for (int r = 0; r < 4; ++r) {
      if (pos + r < p.first || pos + r >= end)
        continue;
      const uint64_t at = ((uint64_t)head * p.t_dst + pos + r) * DH + part * 8u;
      f32x4 lo, hi;
#pragma unroll
      for (int d = 0; d < 4; ++d) {
        lo[d] = code_value(c[d], r, s[r]);
        hi[d] = code_value(c[4 + d], r, s[r]);
      }
      if (top) {
#pragma unroll
        for (int d = 0; d < 4; ++d) {
          lo[d] = f16_within(lo[d]);
          hi[d] = f16_within(hi[d]);
        }
      }
      if constexpr (F16) {
        const f16x4 l = __builtin_convertvector(lo, f16x4), u = __builtin_convertvector(hi, f16x4);
        *reinterpret_cast<f16x8 *>(static_cast<_Float16 *>(p.v) + at) =
            __builtin_shufflevector(l, u, 0, 1, 2, 3, 4, 5, 6, 7);
      } else {
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p.v) + at) = lo;
        *reinterpret_cast<f32x4 *>(static_cast<float *>(p.v) + at + 4) = hi;
      }
    }
  }
}

} // namespace

#define TA_Q8(DH, SUFFIX, F16)                                                                         \
  extern "C" __global__ __launch_bounds__(kThreads) void ta_q8_write_##SUFFIX##_dh##DH(Q8WriteArgs p) { \
    q8_write<DH, F16>(p);                                                                              \
  }                                                                                                    \
  extern "C" __global__ __launch_bounds__(kThreads) void ta_q8_read_##SUFFIX##_dh##DH(Q8ReadArgs p) {   \
    q8_read<DH, F16>(p);                                                                               \
  }
TA_Q8(64, f32, false)
TA_Q8(64, f16, true)
TA_Q8(128, f32, false)
TA_Q8(128, f16, true)
