// Attention of a tree of drafted tokens over a cache for gfx950: `tokens`
// (1 .. 64) query rows per head see the L committed positions and those
// drafts, at positions L + j, that their masks name.  One token is a decode
// step.  Caches: dense f32 or f16 (kt [H_kv, dh, t_max], v [H_kv, t_max,
// dh]), or the 8-bit one of q8_cache.hip.
//
// Mathematics.  Row (t, head) over its set S of positions, in one pass with
// a running maximum m and sum l (base 2, scale2 = scale * log2 e):
//   s_p = scale2 * q . k_p,  out = sum_S 2^(s_p - m) v_p / sum_S 2^(s_p - m),
// zeros where S is empty.  The 8-bit cache's scales factor out of both
// products: s_p = (q . code_p) * ks_p, and the weight of row p is 2^(s_p - m)
// * vs_p.
//
// Work split.  The rows of a kv head, (token, head of its group), are taken
// 32 at a time, an MFMA's columns (16 for at most 16 rows of the 8-bit cache).
// A workgroup is one, two or four such row tiles over one chunk of the
// positions (64 chunks at most), no more workgroups than CUs where the row
// tiles alone are fewer.  The waves of a row tile share the
// chunk's keys, each with its own m, l and output, and meet in LDS at the end.
// With several chunks, workgroups leave their rows' {o, m, l} in scratch and
// ta_tree_combine joins them in chunk order.  No atomics: results do not
// depend on scheduling.
//
// Operands.  Scores are computed transposed, S^T = K Q^T (m = key, n = row):
// a lane owns one row, the row maximum is a register reduction and one
// exchange between the wave's halves, and O^T += V^T P^T takes P straight
// from the score registers.
//  * f32 and 8-bit caches go to the matrix cores through registers: a lane
//    loads what its operands hold (the 8-bit layout is made for that), the next
//    block as its registers become free, while q's operands lie in LDS.
//  * f16 caches go through LDS tiles that the row tiles share, loaded directly
//    and read transposed, while q's operands stay in registers.
//
// Precision (f32 activations: all within a few of f32's own roundings, but
// for the floor of small weights over f16 caches):
//  * f32 caches: v_mfma_f32_32x32x2_f32, whole values;
//  * f16 caches: f16 matrix cores.  f32 q, scaled by a power of two per row,
//    in three f16 pieces, weights in two, the pieces after the first scaled up
//    and summed apart: a weight within 2^-22 of itself, and within 2^-47 of its
//    row's largest where it is below 2^-25 of that.  f16 q as it is, weights in
//    two pieces: within 2^-22, or 2^-36 of the row's largest;
//  * 8-bit cache: codes are exact in bf16, and so are f32 q and weights in
//    three bf16 pieces of 8 bits.  f16 q meets the codes as f16, with weights
//    in two bf16 pieces (2^-16 of a weight, below the result's own 2^-11).
// An infinity or NaN in a dense cache would meet zero weights and zero pieces
// (0 * inf), and where a mask hides it nothing may come of it: a wave whose
// rows come out non-finite takes its keys again, whole values on the vector
// units, masked ones skipped (64 drafts, 32704 positions, 32 / 8 heads, dh
// 128, f16, an infinity in every head: 1.7 ms; 0.07 without).
//
// Bound and measured (kernel and join, us; copy 5.1 TB/s, f16 matrix product
// 1030 TFLOP/s):
//   f16, 64 drafts, 32704 positions, 32 / 8 heads, dh 128: 60.3 + 4.8, 570
//     TFLOP/s and 2.2 TB/s (47.6 with weights in one piece, 2^-11 off); matrix
//     cores (46% busy) and vector units (43%), one after the other in a wave;
//   8-bit, 1 token, 32767 positions, 32 / 8 heads, dh 128, f32: 15.6 + 5.4,
//     4.4 TB/s; HBM;
//   8-bit, 26 drafts, 8191 positions, 32 / 4 heads, dh 64, f16: 11.8 + 4.0;
//     exponentials and conversions (4.6 MB);
//   f16 cache of odd length, f32, 25 drafts, 4999 positions, 32 / 8 heads, dh
//     128: 19.5 + 4.1; five tiles to a chunk, latency of start, tiles and end;
//   f32, 8 drafts, 1016 positions, 32 / 4 heads, dh 64: 7.0 + 4.0; latency.
#include "common.h"

namespace {

constexpr uint32_t kThreads = 256;
constexpr float kNegMax = -3.402823466e38f;
constexpr float kMinScale = 1.17549435e-38f;  // 2^-126
// A row's reference point m moves only when its maximum has outgrown it by
// 2^kSlack (weights stay below that): with 32 rows in a wave some row finds a
// new maximum in nearly every tile.
constexpr float kSlack = 4.0f;
constexpr float kF16Shift = 11.0f;            // f16 weights, and their sum, times 2^11: at most 2^15
constexpr float kLowScale = 2048.0f;          // f16 pieces after the first

typedef __bf16 bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 f16x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x2 __attribute__((ext_vector_type(2)));
typedef uint32_t u32x4 __attribute__((ext_vector_type(4)));

constexpr int kF32 = 0, kF16 = 1, kQ8 = 2;

// Keeps q's operands in LDS: read once before the loop they would take all
// of its registers.
TA_DEVICE void reread_lds() { asm volatile("" ::: "memory"); }
// Keeps what comes before from what comes after in the instruction order: left
// to itself the compiler turns all of a block's operands first, which takes
// more registers than there are.
TA_DEVICE void in_order() { __builtin_amdgcn_sched_barrier(0); }
// A loaded word is turned from here on, not where it was loaded (turned, a
// block takes four times its registers).
template <class T> TA_DEVICE void from_here(T &x) { asm volatile("" : "+v"(x)); }

// scale * log2 e as a positive number, its sign for q.  A scale of zero becomes
// zeros of q, so that every finite score is 0 and a masked one stays -inf.
// Below f32's smallest normal the product is off by 2^-150, so an exponent by
// 2^-22 at most, where q . k is near f32's largest.
TA_DEVICE float split_scale(float scale, float &sign) {
  const float s2 = scale * 1.44269504088896340736f;
  sign = s2 < 0.0f ? -1.0f : s2 > 0.0f ? 1.0f : 0.0f;
  return s2 != 0.0f ? s2 * sign : kMinScale;
}

TA_DEVICE float exp2_fast(float x) { return __builtin_amdgcn_exp2f(x); }
// Maximum / sum over the two lanes (halves of the wave) of a row.
TA_DEVICE float other_half(float x) {
  const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
  return __uint_as_float((threadIdx.x & 32u) ? r[0] : r[1]);
}
TA_DEVICE uint32_t high_halves(uint32_t b, uint32_t a) { return __builtin_amdgcn_perm(b, a, 0x07060302u); }

// This workgroup's place, and the row of this lane.
struct Place {
  uint32_t kvh, chunk, tile;
  uint32_t lane, j, h;
  uint32_t rows, row, token, head;
  bool live;
  uint32_t committed, total; // L, L + tokens

  // Row tile qb of a workgroup's QB.
  TA_DEVICE Place(const TreeArgs &p, uint32_t QB, uint32_t qb) {
    const uint32_t id = blockIdx.x;
    kvh = id % p.kv_heads;
    chunk = id / p.kv_heads % p.chunks;
    tile = id / p.kv_heads / p.chunks * QB + qb;
    lane = threadIdx.x & 63u;
    j = lane & 31u;
    h = lane >> 5;
    rows = p.tokens * p.group;
    set_row(p, tile * 32u + j);
    const uint64_t len = (uint64_t)p.kv_len + (p.pos_addr ? *p.pos_addr : 0u);
    committed = __builtin_amdgcn_readfirstlane((uint32_t)(len < p.t_max - p.tokens ? len : p.t_max - p.tokens));
    total = committed + p.tokens;
  }
  TA_DEVICE void set_row(const TreeArgs &p, uint32_t r) {
    row = r;
    live = r < rows;
    const uint32_t at = live ? r : rows - 1u;
    token = at / p.group;
    head = kvh * p.group + at % p.group;
  }
  TA_DEVICE uint64_t q_at(const TreeArgs &p, uint32_t dh) const {
    return p.q_offset + (uint64_t)token * p.q_stride + (uint64_t)head * dh;
  }
  // The drafts this lane's row sees.
  TA_DEVICE uint64_t drafts(const TreeArgs &p) const {
    if (!p.mask)
      return (2ull << token) - 1ull; // token 63: all ones
    return (uint64_t)p.mask[2u * token] | (uint64_t)p.mask[2u * token + 1u] << 32;
  }
  TA_DEVICE bool sees(uint32_t pos, uint64_t bits) const {
    return pos < committed || (pos < total && (bits >> (pos - committed) & 1ull));
  }
};

// Running state of a lane's row: the output registers of DB 32-wide blocks
// of the head dimension, maximum (scaled, log2 units; both halves alike) and
// this half's part of the sum.
template <int DH> struct State {
  static constexpr int DB = DH / 32;
  f32x16 o[DB];
  float m, l;
  TA_DEVICE void clear() {
#pragma unroll
    for (int b = 0; b < DB; ++b)
      o[b] = f32x16{};
    m = kNegMax;
    l = 0.0f;
  }
  // Raises the maximum to that of NT tiles of scores t * scale2.
  template <int NT> TA_DEVICE void raise(const f32x16 (&t)[NT], float scale2) {
    float top = t[0][0];
#pragma unroll
    for (int c = 0; c < NT; ++c)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        top = fmaxf(top, t[c][e]);
    top = fmaxf(top, other_half(top)) * scale2;
    if (__any(top > m + kSlack)) {
      const float next = fmaxf(m, top);
      const float corr = exp2_fast(m - next);
      l *= corr;
#pragma unroll
      for (int b = 0; b < DB; ++b)
#pragma unroll
        for (int e = 0; e < 16; ++e)
          o[b][e] *= corr;
      m = next;
    }
  }
  TA_DEVICE bool finite() const {
    float x = l * 0.0f;
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int e = 0; e < 16; ++e)
        x = fmaf(o[b][e], 0.0f, x);
    return x == x;
  }
};

// The head dimension that output register (b, 4 q + r) of half h holds.  f32
// caches: a lane loads dh / 32 neighbouring columns of V, one for each b.
template <int DH, int KIND> TA_DEVICE uint32_t out_dim(int b, int q, int r, uint32_t h) {
  const uint32_t m = 8u * q + 4u * h + r;
  return KIND == kF32 ? (uint32_t)(DH / 32) * m + b : 32u * b + m;
}

// The states of the KP waves of a row tile become one; with one chunk the
// result goes to `out`, else {o, m, l} to the row tile's scratch.  Wave `part`
// of the KP sums every KP-th register quad.
template <int DH, int KP> constexpr int merge_floats() { return KP * (DH / 2) * 64 + 2 * KP * 64; }

template <int DH, int KIND, bool IO16, int KP>
TA_DEVICE void finish(const TreeArgs &p, const Place &w, State<DH> &st, uint32_t part, float *smem) {
  constexpr int DB = DH / 32, QUADS = DB * 4, OWN = KP < 4 ? 4 / KP : 1; // quads q = part + KP i < 4
  static_assert(KP == 2 || KP == 4 || KP == 8, "quads split evenly");
  float l = st.l + other_half(st.l);
  f32x4 *mo = reinterpret_cast<f32x4 *>(smem);
  float *mm = smem + KP * (DH / 2) * 64, *ml = mm + KP * 64;
  __syncthreads(); // the operands in this memory are done with
#pragma unroll
  for (int b = 0; b < DB; ++b)
#pragma unroll
    for (int q = 0; q < 4; ++q)
      mo[(part * QUADS + b * 4 + q) * 64u + w.lane] =
          f32x4{st.o[b][4 * q], st.o[b][4 * q + 1], st.o[b][4 * q + 2], st.o[b][4 * q + 3]};
  mm[part * 64u + w.lane] = st.m;
  ml[part * 64u + w.lane] = l;
  __syncthreads();
  float a[KP], top = mm[w.lane];
#pragma unroll
  for (uint32_t i = 1; i < KP; ++i)
    top = fmaxf(top, mm[i * 64u + w.lane]);
  l = 0.0f;
#pragma unroll
  for (uint32_t i = 0; i < KP; ++i) {
    a[i] = exp2_fast(mm[i * 64u + w.lane] - top);
    l = fmaf(ml[i * 64u + w.lane], a[i], l);
  }
  if (KP > 4 && part >= 4u)
    return;
  f32x4 v[OWN][DB];
#pragma unroll
  for (int o = 0; o < OWN; ++o)
#pragma unroll
    for (int b = 0; b < DB; ++b) {
      const uint32_t at = b * 4u + part + KP * o;
      v[o][b] = mo[at * 64u + w.lane] * a[0];
#pragma unroll
      for (uint32_t i = 1; i < KP; ++i) {
        const f32x4 x = mo[(i * QUADS + at) * 64u + w.lane];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[o][b][r] = fmaf(x[r], a[i], v[o][b][r]);
      }
    }
  if (!w.live)
    return;
  if (p.chunks > 1) {
    float *out = p.partial + (((uint64_t)w.tile * p.chunks + w.chunk) * p.kv_heads + w.kvh) * ta_tree_partial(DH);
#pragma unroll
    for (int o = 0; o < OWN; ++o)
#pragma unroll
      for (int b = 0; b < DB; ++b)
        reinterpret_cast<f32x4 *>(out)[(b * 4u + part + KP * o) * 64u + w.lane] = v[o][b];
    if (part == 0 && w.h == 0) {
      out[DH / 2 * 64 + w.j] = top;
      out[DH / 2 * 64 + 32 + w.j] = l;
    }
    return;
  }
  const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
  const uint64_t at = ((uint64_t)w.token * p.kv_heads * p.group + w.head) * DH;
#pragma unroll
  for (int o = 0; o < OWN; ++o)
#pragma unroll
    for (int r = 0; r < 4; ++r)
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const uint64_t d = at + out_dim<DH, KIND>(b, part + KP * o, r, w.h);
        if constexpr (IO16)
          static_cast<_Float16 *>(p.out)[d] = (_Float16)(v[o][b][r] * inv);
        else
          static_cast<float *>(p.out)[d] = v[o][b][r] * inv;
      }
}

template <int KIND> TA_DEVICE float dense(const void *base, uint64_t at) {
  return KIND == kF16 ? (float)static_cast<const _Float16 *>(base)[at] : static_cast<const float *>(base)[at];
}

// A wave's keys (`width` from every `step`-th on, first .. last - 1) once more,
// eight at a time, whole values on the vector units (see the top): half h
// takes half of q . k and its own output registers.
template <int DH, int KIND, bool IO16>
TA_DEVICE void whole_values(const TreeArgs &p, const Place &w, State<DH> &st, uint32_t first, uint32_t last,
                            uint32_t step, uint32_t width) {
  constexpr int HALF = DH / 2, DB = DH / 32, KEYS = 8;
  typedef std::conditional_t<KIND == kF16, _Float16, float> T;
  typedef T keys_v __attribute__((ext_vector_type(KEYS), aligned(sizeof(T))));
  typedef T cols_v __attribute__((ext_vector_type(KIND == kF16 ? 4 : DB)));
  const T *kt = static_cast<const T *>(p.kt) + (uint64_t)w.kvh * DH * p.t_max;
  const T *vv = static_cast<const T *>(p.v) + (uint64_t)w.kvh * p.t_max * DH;
  const float scale2 = p.scale * 1.44269504088896340736f;
  const uint64_t bits = w.drafts(p), q0 = w.q_at(p, DH) + w.h * HALF;
  const float shift = KIND == kF16 ? kF16Shift : 0.0f; // as the other waves' weights
  st.clear();
  last = min(last, w.total);
  for (uint32_t k0 = first; k0 < last; k0 += step) {
    const uint32_t end = min(k0 + width, last);
    for (uint32_t pos = k0; pos < end; pos += KEYS) {
      bool valid[KEYS], any = false;
      float s[KEYS];
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        valid[i] = w.live && pos + i < end && w.sees(pos + i, bits);
        any = any || valid[i];
        s[i] = 0.0f;
      }
      if (!__any(any))
        continue;
      const bool inside = pos + KEYS <= p.t_max;
#pragma unroll 4
      for (uint32_t d = 0; d < HALF; ++d) {
        const float q = dense<IO16 ? kF16 : kF32>(p.q, q0 + d);
        const T *row = kt + (uint64_t)(w.h * HALF + d) * p.t_max;
        keys_v k;
        if (inside) {
          k = *reinterpret_cast<const keys_v *>(row + pos);
        } else {
#pragma unroll
          for (int i = 0; i < KEYS; ++i)
            k[i] = row[min(pos + i, p.t_max - 1u)];
        }
#pragma unroll
        for (int i = 0; i < KEYS; ++i)
          s[i] = fmaf(q, (float)k[i], s[i]);
      }
      float next = st.m, sum = 0.0f;
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        s[i] = (s[i] + other_half(s[i])) * scale2;
        next = valid[i] ? fmaxf(next, s[i]) : next;
      }
      const float corr = any ? exp2_fast(st.m - next) : 1.0f;
#pragma unroll
      for (int i = 0; i < KEYS; ++i) {
        s[i] = valid[i] ? exp2_fast(s[i] - next + shift) : 0.0f;
        sum += s[i];
      }
      st.m = next;
      st.l = fmaf(st.l, corr, w.h == 0 ? sum : 0.0f);
      // 16 groups of output registers whose columns lie together: (b, 4 q ..)
      // for f16 caches, (all b, 4 q + r) for f32 ones
#pragma unroll
      for (int group = 0; group < (KIND == kF16 ? DB * 4 : 16); ++group) {
        reread_lds(); // no more than these loads at a time
        constexpr int N = KIND == kF16 ? 4 : DB;
        const uint32_t col = KIND == kF16 ? out_dim<DH, KIND>(group / 4, group % 4, 0, w.h)
                                          : out_dim<DH, KIND>(0, group / 4, group % 4, w.h);
        cols_v v[KEYS];
#pragma unroll
        for (uint32_t i = 0; i < KEYS; ++i)
          v[i] = *reinterpret_cast<const cols_v *>(vv + (uint64_t)min(pos + i, end - 1u) * DH + col);
#pragma unroll
        for (int c = 0; c < N; ++c) {
          const int b = KIND == kF16 ? group / 4 : c, e = KIND == kF16 ? 4 * (group % 4) + c : group;
          float x = st.o[b][e] * corr;
#pragma unroll
          for (int i = 0; i < KEYS; ++i)
            x = valid[i] ? fmaf(s[i], (float)v[i][c], x) : x;
          st.o[b][e] = x;
        }
      }
    }
  }
}

// The block range of a chunk.
TA_DEVICE void chunk_blocks(const TreeArgs &p, const Place &w, uint32_t block_keys, uint32_t &b0, uint32_t &b1) {
  const uint32_t blocks = (w.total + block_keys - 1u) / block_keys, each = (blocks + p.chunks - 1u) / p.chunks;
  b0 = min(w.chunk * each, blocks);
  b1 = min(b0 + each, blocks);
}

// q's operands for LDS: 8 threads to a row r, DH / 8 values each, to put(part,
// r, values).
template <int DH, bool IO16, class Put> TA_DEVICE void load_q(const TreeArgs &p, const Place &w, Put &&put) {
  constexpr int N = DH / 8;
  typedef f32x4 f32x4u __attribute__((aligned(4)));
  typedef f16x8 f16x8u __attribute__((aligned(2)));
  if (threadIdx.x >= 256u)
    return;
  const uint32_t r = threadIdx.x >> 3, part = threadIdx.x & 7u;
  Place row = w;
  row.set_row(p, w.tile * 32u + r);
  const uint64_t at = row.q_at(p, DH) + part * N;
  float x[N];
  if constexpr (IO16) {
#pragma unroll
    for (int i = 0; i < N / 8; ++i) {
      const f16x8 v = *reinterpret_cast<const f16x8u *>(static_cast<const _Float16 *>(p.q) + at + 8 * i);
#pragma unroll
      for (int c = 0; c < 8; ++c)
        x[8 * i + c] = (float)v[c];
    }
  } else {
#pragma unroll
    for (int i = 0; i < N / 4; ++i) {
      const f32x4 v = *reinterpret_cast<const f32x4u *>(static_cast<const float *>(p.q) + at + 4 * i);
#pragma unroll
      for (int c = 0; c < 4; ++c)
        x[4 * i + c] = v[c];
    }
  }
#pragma unroll
  for (int i = 0; i < N; ++i)
    x[i] = row.live ? x[i] : 0.0f;
  put(part, r, x);
}

// ------------------------------------------------------------- 8-bit cache

// A word's four codes as bf16 (exact) / as f16 (exact: 1024 + byte, less
// 1152, of the codes with their sign bits turned).
TA_DEVICE u32x2 codes_bf16(uint32_t w) {
  float f[4];
#pragma unroll
  for (int i = 0; i < 4; ++i)
    f[i] = (float)(int8_t)(w >> (8 * i));
  return u32x2{high_halves(__float_as_uint(f[1]), __float_as_uint(f[0])),
               high_halves(__float_as_uint(f[3]), __float_as_uint(f[2]))};
}
TA_DEVICE u32x2 codes_f16(uint32_t w) {
  const uint32_t u = w ^ 0x80808080u;
  const f16x2 bias = {(_Float16)1152.0f, (_Float16)1152.0f};
  const f16x2 a = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04010400u)) - bias;
  const f16x2 b = __builtin_bit_cast(f16x2, __builtin_amdgcn_perm(0x64646464u, u, 0x04030402u)) - bias;
  return u32x2{__builtin_bit_cast(uint32_t, a), __builtin_bit_cast(uint32_t, b)};
}

template <int DH, bool IO16, int KP> struct TreeQ8 {
  static constexpr int KS = DH / 16, DB = DH / 32;
  static constexpr int NQ = IO16 ? 1 : 3, NP = IO16 ? 2 : 3;
  static constexpr int Q_FLOATS = NQ * KS * 64 * 4;
  static constexpr int MERGE = merge_floats<DH, KP>();
  static constexpr int SMEM = Q_FLOATS > MERGE ? Q_FLOATS : MERGE;

  struct Raw { // a block as this lane's operands hold it
    u32x4 k[DB], v[DB], ks[2], vs[2];
  };
  static TA_DEVICE void load_k(const uint8_t *rec, const Place &w, Raw &r) {
#pragma unroll
    for (int u = 0; u < DB; ++u)
      r.k[u] = *reinterpret_cast<const u32x4 *>(rec + u * 1024u + w.lane * 16u);
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.ks[i] = *reinterpret_cast<const u32x4 *>(rec + 64u * DH + w.h * 32u + i * 16u);
  }
  static TA_DEVICE void load_v(const uint8_t *rec, const Place &w, Raw &r) {
#pragma unroll
    for (int i = 0; i < 2; ++i)
      r.vs[i] = *reinterpret_cast<const u32x4 *>(rec + 64u * DH + 64u + w.h * 32u + i * 16u);
#pragma unroll
    for (int u = 0; u < DB; ++u)
      r.v[u] = *reinterpret_cast<const u32x4 *>(rec + 32u * DH + u * 1024u + w.j * 32u + w.h * 16u);
  }
  static TA_DEVICE float scale_of(const u32x4 (&s)[2], int e) {
    const uint32_t x = s[e / 8][e % 8 / 2];
    return __uint_as_float(e & 1 ? x & 0xFFFF0000u : x << 16);
  }

  // One block, whose drafts a row may not see (MASKED) or all committed;
  // `next` (null: none) is fetched into the registers as they become free.
  template <bool MASKED>
  static TA_DEVICE void block(Raw &r, const uint8_t *next, const u32x4 *qs, const Place &w, uint32_t k0,
                              uint64_t bits, float scale2, State<DH> &st) {
    reread_lds();
    f32x16 t[1] = {f32x16{}};
    u32x4 q_next[NQ];
#pragma unroll
    for (int n = 0; n < NQ; ++n)
      q_next[n] = qs[n * KS * 64 + w.lane];
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      in_order();
      u32x4 q_now[NQ];
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        q_now[n] = q_next[n];
        if (s + 1 < KS)
          q_next[n] = qs[(n * KS + s + 1) * 64 + w.lane];
      }
      if (s % 2 == 0)
        from_here(r.k[s / 2]);
      const uint32_t w0 = r.k[s / 2][2 * (s % 2)], w1 = r.k[s / 2][2 * (s % 2) + 1];
      const u32x2 a = IO16 ? codes_f16(w0) : codes_bf16(w0), b = IO16 ? codes_f16(w1) : codes_bf16(w1);
      const u32x4 k = {a[0], a[1], b[0], b[1]};
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 q = q_now[n];
        if constexpr (IO16)
          t[0] = __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, k), __builtin_bit_cast(f16x8, q),
                                                        t[0], 0, 0, 0);
        else
          t[0] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, k),
                                                         __builtin_bit_cast(bf16x8, q), t[0], 0, 0, 0);
      }
    }
    from_here(r.ks[0]);
    from_here(r.ks[1]);
    uint32_t seen = 0u;
    if constexpr (MASKED) {
#pragma unroll
      for (int e = 0; e < 16; ++e)
        seen |= (w.sees(k0 + 8u * (e / 4) + 4u * w.h + e % 4, bits) ? 1u : 0u) << e;
    }
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      t[0][e] *= scale_of(r.ks, e);
      if constexpr (MASKED)
        t[0][e] = seen >> e & 1u ? t[0][e] : -__builtin_inff();
    }
    in_order();
    if (next)
      load_k(next, w, r);
    st.raise(t, scale2);
    from_here(r.vs[0]);
    from_here(r.vs[1]);
    u32x4 pp[NP][2];
#pragma unroll
    for (int e = 0; e < 16; e += 2) {
      float x[2];
#pragma unroll
      for (int i = 0; i < 2; ++i) {
        x[i] = exp2_fast(fmaf(t[0][e + i], scale2, -st.m));
        st.l += x[i];
        x[i] *= scale_of(r.vs, e + i);
        if constexpr (MASKED)
          x[i] = seen >> (e + i) & 1u ? x[i] : 0.0f;
      }
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        pp[n][e / 8][e % 8 / 2] = high_halves(__float_as_uint(x[1]), __float_as_uint(x[0]));
        if (n + 1 < NP) {
#pragma unroll
          for (int i = 0; i < 2; ++i)
            x[i] -= __uint_as_float(__float_as_uint(x[i]) & 0xFFFF0000u);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < DB; ++b)
#pragma unroll
      for (int s = 0; s < 2; ++s) {
        in_order();
        if (s == 0)
          from_here(r.v[b]);
        const u32x2 lo = codes_bf16(r.v[b][2 * s]), hi = codes_bf16(r.v[b][2 * s + 1]);
        const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
        for (int n = 0; n < NP; ++n)
          st.o[b] = __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, v),
                                                            __builtin_bit_cast(bf16x8, pp[n][s]), st.o[b], 0, 0, 0);
      }
    if (next)
      load_v(next, w, r);
    in_order();
  }

  static TA_DEVICE void run(const TreeArgs &p) {
    __shared__ __attribute__((aligned(16))) float smem[SMEM];
    const uint32_t kp = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place w(p, 1, 0);
    uint32_t b0, b1;
    chunk_blocks(p, w, TA_Q8_BLOCK, b0, b1);
    float sign;
    const float scale2 = split_scale(p.scale, sign);
    // The first block before q, and the mask (in host memory) after both: a
    // load is waited for with all before it.
    const uint8_t *base = p.cache + (uint64_t)w.kvh * p.blocks * ta_q8_record(DH);
    auto rec = [&](uint32_t b) { return base + (uint64_t)b * ta_q8_record(DH); };
    Raw r;
    uint32_t b = b0 + kp;
    if (b < b1) {
      load_k(rec(b), w, r);
      load_v(rec(b), w, r);
    }
    u32x4 *qs = reinterpret_cast<u32x4 *>(smem);
    // group g of 8 values: step s = 2 (g / 4) + g % 2, half g / 2 % 2
    load_q<DH, IO16>(p, w, [&](uint32_t part, uint32_t r, const float(&x)[DH / 8]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < DH / 64; ++i) {
        const uint32_t g = part * (DH / 64) + i, s = 2u * (g / 4u) + g % 2u, lane = 32u * (g / 2u % 2u) + r;
        if constexpr (IO16) {
          f16x8 v;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            v[c] = (_Float16)(x[8 * i + c] * sign);
          qs[s * 64u + lane] = __builtin_bit_cast(u32x4, v);
        } else {
          float y[8];
#pragma unroll
          for (int c = 0; c < 8; ++c)
            y[c] = x[8 * i + c] * sign;
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            u32x4 v;
#pragma unroll
            for (int c = 0; c < 4; ++c)
              v[c] = high_halves(__float_as_uint(y[2 * c + 1]), __float_as_uint(y[2 * c]));
            qs[(n * KS + s) * 64u + lane] = v;
#pragma unroll
            for (int c = 0; c < 8; ++c)
              y[c] -= __uint_as_float(__float_as_uint(y[c]) & 0xFFFF0000u);
          }
        }
      }
    });
    State<DH> st;
    st.clear();
    const uint64_t bits = b1 * TA_Q8_BLOCK > w.committed ? w.drafts(p) : 0ull;
    __syncthreads();
    const uint32_t whole = min(b1, w.committed / TA_Q8_BLOCK);
    for (; b < whole; b += KP)
      block<false>(r, b + KP < b1 ? rec(b + KP) : nullptr, qs, w, b * TA_Q8_BLOCK, bits, scale2, st);
    for (; b < b1; b += KP)
      block<true>(r, b + KP < b1 ? rec(b + KP) : nullptr, qs, w, b * TA_Q8_BLOCK, bits, scale2, st);
    finish<DH, kQ8, IO16, KP>(p, w, st, kp, smem);
  }
};

// At most 16 rows over the 8-bit cache (decode steps, small trees): the same on
// the 16 x 16 x 32 matrix instructions, half the products and half the
// exponentials of a 32-row tile, which bound the kernel there (one token,
// 32767 positions, 32 / 8 heads, dh 128, f32: 19.8 us on 32-row tiles).
// Lane (row or key m = lane % 16, g = lane / 16).  Score tile c holds in
// register r of group g the key in slot 8 g + 4 c + r: a lane's 8 weights are
// then 8 neighbouring slots of V's codes, and of the scales.
template <int DH, bool IO16, int KP> struct TreeQ8Few {
  static constexpr int KS = DH / 32, DT = DH / 16; // score k-steps, 16-wide output tiles
  static constexpr int NQ = IO16 ? 1 : 3, NP = IO16 ? 2 : 3;
  static constexpr int Q_FLOATS = NQ * KS * 64 * 4, MERGE = KP * (DT * 64 * 4 + 2 * 16);
  static constexpr int SMEM = Q_FLOATS > MERGE ? Q_FLOATS : MERGE;

  struct Raw {
    u32x4 k[2][DH / 64], ks, vs;
    u32x2 v[DT];
  };
  // Maximum / sum over the four lanes of a row.
  static TA_DEVICE float row_max(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return fmaxf(__uint_as_float(r[0]), __uint_as_float(r[1]));
  }
  static TA_DEVICE float row_sum(float x) {
    auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    x = __uint_as_float(r[0]) + __uint_as_float(r[1]);
    r = __builtin_amdgcn_permlane32_swap(__float_as_uint(x), __float_as_uint(x), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
  }
  // The key in slot s.
  static TA_DEVICE uint32_t key_in(uint32_t s) { return 8u * (s / 4u % 4u) + 4u * (s / 16u) + s % 4u; }
  static TA_DEVICE void load_k(const uint8_t *rec, uint32_t lane, Raw &r) {
    const uint32_t m = lane & 15u, g = lane >> 4;
#pragma unroll
    for (uint32_t c = 0; c < 2; ++c) {
      const uint32_t key = key_in(8u * (m / 4u) + 4u * c + m % 4u);
#pragma unroll
      for (int u = 0; u < DH / 64; ++u)
        r.k[c][u] = *reinterpret_cast<const u32x4 *>(rec + ((4u * u + g) * 32u + key) * 16u);
    }
    r.ks = *reinterpret_cast<const u32x4 *>(rec + 64u * DH + g * 16u);
  }
  static TA_DEVICE void load_v(const uint8_t *rec, uint32_t lane, Raw &r) {
    const uint32_t m = lane & 15u, g = lane >> 4;
    r.vs = *reinterpret_cast<const u32x4 *>(rec + 64u * DH + 64u + g * 16u);
#pragma unroll
    for (int b = 0; b < DT; ++b)
      r.v[b] = *reinterpret_cast<const u32x2 *>(rec + 32u * DH + (16u * b + m) * 32u + g * 8u);
  }
  static TA_DEVICE float scale_of(const u32x4 &s, int i) { // of slot 8 g + i
    return __uint_as_float(i & 1 ? s[i / 2] & 0xFFFF0000u : s[i / 2] << 16);
  }

  template <bool MASKED>
  static TA_DEVICE void block(Raw &r, const uint8_t *next, const u32x4 *qs, const Place &w, uint32_t k0,
                              uint64_t bits, float scale2, f32x4 (&o)[DT], float &m, float &l) {
    reread_lds();
    const uint32_t g = w.lane >> 4;
    f32x4 t[2] = {f32x4{0.0f, 0.0f, 0.0f, 0.0f}, f32x4{0.0f, 0.0f, 0.0f, 0.0f}};
#pragma unroll
    for (int s = 0; s < KS; ++s) {
      in_order();
      u32x4 k[2];
#pragma unroll
      for (int c = 0; c < 2; ++c) {
        if (s % 2 == 0)
          from_here(r.k[c][s / 2]);
        const uint32_t w0 = r.k[c][s / 2][2 * (s % 2)], w1 = r.k[c][s / 2][2 * (s % 2) + 1];
        const u32x2 a = IO16 ? codes_f16(w0) : codes_bf16(w0), b = IO16 ? codes_f16(w1) : codes_bf16(w1);
        k[c] = u32x4{a[0], a[1], b[0], b[1]};
      }
#pragma unroll
      for (int n = 0; n < NQ; ++n) {
        const u32x4 q = qs[(n * KS + s) * 64 + w.lane];
#pragma unroll
        for (int c = 0; c < 2; ++c) {
          if constexpr (IO16)
            t[c] = __builtin_amdgcn_mfma_f32_16x16x32_f16(__builtin_bit_cast(f16x8, k[c]),
                                                          __builtin_bit_cast(f16x8, q), t[c], 0, 0, 0);
          else
            t[c] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, k[c]),
                                                           __builtin_bit_cast(bf16x8, q), t[c], 0, 0, 0);
        }
      }
    }
    from_here(r.ks);
    float x[8], top = -__builtin_inff();
    bool seen[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) {
      x[i] = t[i / 4][i % 4] * scale_of(r.ks, i);
      if constexpr (MASKED) {
        seen[i] = w.sees(k0 + key_in(8u * g + i), bits);
        x[i] = seen[i] ? x[i] : -__builtin_inff();
      }
      top = fmaxf(top, x[i]);
    }
    in_order();
    if (next)
      load_k(next, w.lane, r);
    top = row_max(top) * scale2;
    if (__any(top > m + kSlack)) {
      const float higher = fmaxf(m, top), corr = exp2_fast(m - higher);
      l *= corr;
#pragma unroll
      for (int b = 0; b < DT; ++b)
        o[b] *= corr;
      m = higher;
    }
    from_here(r.vs);
    u32x4 pp[NP];
#pragma unroll
    for (int i = 0; i < 8; i += 2) {
      float y[2];
#pragma unroll
      for (int e = 0; e < 2; ++e) {
        y[e] = exp2_fast(fmaf(x[i + e], scale2, -m));
        l += y[e];
        y[e] *= scale_of(r.vs, i + e);
        if constexpr (MASKED)
          y[e] = seen[i + e] ? y[e] : 0.0f;
      }
#pragma unroll
      for (int n = 0; n < NP; ++n) {
        pp[n][i / 2] = high_halves(__float_as_uint(y[1]), __float_as_uint(y[0]));
        if (n + 1 < NP) {
#pragma unroll
          for (int e = 0; e < 2; ++e)
            y[e] -= __uint_as_float(__float_as_uint(y[e]) & 0xFFFF0000u);
        }
      }
    }
#pragma unroll
    for (int b = 0; b < DT; ++b) {
      in_order();
      from_here(r.v[b]);
      const u32x2 lo = codes_bf16(r.v[b][0]), hi = codes_bf16(r.v[b][1]);
      const u32x4 v = {lo[0], lo[1], hi[0], hi[1]};
#pragma unroll
      for (int n = 0; n < NP; ++n)
        o[b] = __builtin_amdgcn_mfma_f32_16x16x32_bf16(__builtin_bit_cast(bf16x8, v),
                                                       __builtin_bit_cast(bf16x8, pp[n]), o[b], 0, 0, 0);
    }
    if (next)
      load_v(next, w.lane, r);
    in_order();
  }

  static TA_DEVICE void run(const TreeArgs &p) {
    __shared__ __attribute__((aligned(16))) float smem[SMEM];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    Place w(p, 1, 0);
    const uint32_t lane = w.lane, m16 = lane & 15u, g = lane >> 4;
    w.set_row(p, m16);
    uint32_t b0, b1;
    chunk_blocks(p, w, TA_Q8_BLOCK, b0, b1);
    const uint8_t *base = p.cache + (uint64_t)w.kvh * p.blocks * ta_q8_record(DH);
    auto rec = [&](uint32_t b) { return base + (uint64_t)b * ta_q8_record(DH); };
    Raw r;
    uint32_t b = b0 + wave;
    if (b < b1) {
      load_k(rec(b), lane, r);
      load_v(rec(b), lane, r);
    }
    float sign;
    const float scale2 = split_scale(p.scale, sign);
    u32x4 *qs = reinterpret_cast<u32x4 *>(smem);
    // q's operands: 8 values from d = 8 i on of row r are step 2 (i / 8) + i %
    // 2 of lane 16 (i / 2 % 4) + r
    for (uint32_t at = tid; at < 16u * (DH / 8); at += 64 * KP) {
      const uint32_t i = at % (DH / 8), row = at / (DH / 8);
      const uint32_t to = (2u * (i / 8u) + i % 2u) * 64u + 16u * (i / 2u % 4u) + row;
      Place q = w;
      q.set_row(p, row);
      const uint64_t from = q.q_at(p, DH) + 8u * i;
      const float keep = q.live ? sign : 0.0f;
      if constexpr (IO16) {
        typedef f16x8 f16x8u __attribute__((aligned(2)));
        const f16x8 v = *reinterpret_cast<const f16x8u *>(static_cast<const _Float16 *>(p.q) + from);
        qs[to] = q.live ? __builtin_bit_cast(u32x4, v * (_Float16)sign) : u32x4{0u, 0u, 0u, 0u};
      } else {
        typedef f32x4 f32x4u __attribute__((aligned(4)));
        float y[8];
#pragma unroll
        for (int h = 0; h < 2; ++h) {
          const f32x4 v = *reinterpret_cast<const f32x4u *>(static_cast<const float *>(p.q) + from + 4 * h);
#pragma unroll
          for (int c = 0; c < 4; ++c)
            y[4 * h + c] = q.live ? v[c] * keep : 0.0f;
        }
#pragma unroll
        for (int n = 0; n < NQ; ++n) {
          u32x4 v;
#pragma unroll
          for (int c = 0; c < 4; ++c)
            v[c] = high_halves(__float_as_uint(y[2 * c + 1]), __float_as_uint(y[2 * c]));
          qs[n * KS * 64u + to] = v;
#pragma unroll
          for (int c = 0; c < 8; ++c)
            y[c] -= __uint_as_float(__float_as_uint(y[c]) & 0xFFFF0000u);
        }
      }
    }
    const uint64_t bits = b1 * TA_Q8_BLOCK > w.committed ? w.drafts(p) : 0ull;
    f32x4 o[DT];
#pragma unroll
    for (int t = 0; t < DT; ++t)
      o[t] = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
    float m = kNegMax, l = 0.0f;
    __syncthreads();
    const uint32_t whole = min(b1, w.committed / TA_Q8_BLOCK);
    for (; b < whole; b += KP)
      block<false>(r, b + KP < b1 ? rec(b + KP) : nullptr, qs, w, b * TA_Q8_BLOCK, bits, scale2, o, m, l);
    for (; b < b1; b += KP)
      block<true>(r, b + KP < b1 ? rec(b + KP) : nullptr, qs, w, b * TA_Q8_BLOCK, bits, scale2, o, m, l);

    // The waves' states become one; wave i sums every KP-th output tile.
    l = row_sum(l);
    f32x4 *mo = reinterpret_cast<f32x4 *>(smem);
    float *mm = smem + KP * DT * 64 * 4, *ml = mm + KP * 16;
    __syncthreads(); // q's operands are done with
#pragma unroll
    for (int t = 0; t < DT; ++t)
      mo[(wave * DT + t) * 64u + lane] = o[t];
    if (g == 0) {
      mm[wave * 16u + m16] = m;
      ml[wave * 16u + m16] = l;
    }
    __syncthreads();
    float a[KP], top = kNegMax;
    l = 0.0f;
#pragma unroll
    for (int i = 0; i < KP; ++i)
      top = fmaxf(top, mm[i * 16 + m16]);
#pragma unroll
    for (int i = 0; i < KP; ++i) {
      a[i] = exp2_fast(mm[i * 16 + m16] - top);
      l = fmaf(ml[i * 16 + m16], a[i], l);
    }
    if (!w.live)
      return;
    float *part = p.partial + ((uint64_t)w.chunk * p.kv_heads + w.kvh) * ta_tree_partial(DH);
    const float inv = l > 0.0f ? 1.0f / l : l == l ? 0.0f : l;
    const uint64_t at = ((uint64_t)w.token * p.kv_heads * p.group + w.head) * DH;
    for (uint32_t t = wave; t < DT; t += KP) {
      f32x4 v = mo[t * 64u + lane] * a[0];
#pragma unroll
      for (int i = 1; i < KP; ++i) {
        const f32x4 x = mo[(i * DT + t) * 64u + lane];
#pragma unroll
        for (int e = 0; e < 4; ++e)
          v[e] = fmaf(x[e], a[i], v[e]);
      }
      // columns 16 t + 4 g .. + 3: quad 2 (t % 2) + g / 2 of block t / 2, half g % 2
      if (p.chunks > 1) {
        reinterpret_cast<f32x4 *>(part)[(t / 2u * 4u + 2u * (t % 2u) + g / 2u) * 64u + 32u * (g % 2u) + m16] = v;
      } else {
#pragma unroll
        for (int e = 0; e < 4; ++e) {
          const uint64_t d = at + 16u * t + 4u * g + e;
          if constexpr (IO16)
            static_cast<_Float16 *>(p.out)[d] = (_Float16)(v[e] * inv);
          else
            static_cast<float *>(p.out)[d] = v[e] * inv;
        }
      }
    }
    if (p.chunks > 1 && tid < 16u) {
      part[DH / 2 * 64 + m16] = top;
      part[DH / 2 * 64 + 32 + m16] = l;
    }
  }
};

// -------------------------------------------------------------- f16 caches

// K and V tiles lie in LDS as in the caches ([d][key], [key][d]; 16-byte
// pieces swizzled within a row), fetched by direct global -> LDS loads with
// one barrier per tile, and reach the matrix cores through
// ds_read_b64_tr_b16.  A workgroup is QB row tiles x KP key parts of BKW keys;
// q's operands stay in registers.  Tried on 64 drafts, 32704 positions, 32 / 8
// heads, dh 128: 128-key tiles gained nothing, and two row tiles to a wave took
// 71 us where four waves with one each took 62.
template <int DH, bool IO16, bool DIRECT, int QB, int KP, int BKW> struct TreeF16 {
  static constexpr int T = 64 * QB * KP;
  static constexpr int BK = KP * BKW;        // keys per tile
  static constexpr int KB = BKW / 32;        // 32-key score blocks per wave
  static constexpr int KS = DH / 16, DB = DH / 32;
  static constexpr int NQ = IO16 ? 1 : 3;    // f16 pieces of q
  static constexpr int AHEAD = IO16 ? 4 : 2; // LDS reads before their use
  static constexpr int K_BYTES = DH * BK * 2, STAGE = 2 * K_BYTES;
  static constexpr int CK = BK / 8, CV = DH / 8; // 16-byte pieces per K / V row
  static constexpr int LD = K_BYTES / 16 / T;    // direct loads per thread, per operand
  static constexpr int MERGE = QB * merge_floats<DH, KP>() * 4;
  // The waves of the second key part run their output product one tile late (a
  // third buffer keeps its V).  That keeps the two waves of a SIMD in different
  // phases, which on its own was no gain (64 drafts, 32704 positions, 32 / 8
  // heads, f16, weights in one piece: 58 us against 55), but where K goes through registers beside
  // f32 q's three pieces the later use of V's operands is what keeps the loop
  // within its registers (64 drafts, 16000 positions: 61 us, 93 without).
  static constexpr bool LATE = T == 512 && !DIRECT && !IO16 && DH == 128;
  // Tiles in flight.  Two hide more of HBM's latency where a CU holds one
  // workgroup anyway (64 drafts, 32704 positions, 32 / 8 heads, dh 128, f16: 72
  // us behind other work, 76 with one; 69 and 68 when called again).  Four waves lose by them (16 drafts, 32000 positions, dh 64: 26.4
  // us, 23.5 with one).
  static constexpr int FLIGHT = DIRECT && T == 512 ? 2 : 1;
  static constexpr int BUFS = LATE || FLIGHT == 2 ? 3 : 2;
  static constexpr int SMEM = BUFS * STAGE > MERGE ? BUFS * STAGE : MERGE;
  static_assert(LD * T * 16 == K_BYTES && CK >= 8 && CV >= 8, "stages split evenly");
  static_assert(SMEM <= 160 * 1024, "LDS");

  static TA_DEVICE void run(const TreeArgs &p) {
    __shared__ __attribute__((aligned(1024))) char smem[SMEM];
    const uint32_t tid = threadIdx.x, wave = __builtin_amdgcn_readfirstlane(tid >> 6);
    const uint32_t qb = wave % QB, kh = wave / QB;
    const Place w(p, QB, qb);
    const uint32_t lane = w.lane, j = w.j, h = w.h;
    const uint32_t lds0 = (uint32_t)(uintptr_t)(__attribute__((address_space(3))) char *)smem;
    uint32_t t0, t1;
    chunk_blocks(p, w, BK, t0, t1);

    // This lane's q operand: columns 16 s + 8 h .. + 7 of its row.
    f16x8 qf[NQ][KS];
    const float s2 = p.scale * 1.44269504088896340736f, sign = s2 < 0.0f ? -1.0f : 1.0f;
    float scale2 = s2 * sign; // the sign goes to q
    {
      const uint64_t at = w.q_at(p, DH) + h * 8u;
      if constexpr (IO16) {
        typedef f16x8 f16x8u __attribute__((aligned(2)));
#pragma unroll
        for (int s = 0; s < KS; ++s)
          qf[0][s] = *reinterpret_cast<const f16x8u *>(static_cast<const _Float16 *>(p.q) + at + 16 * s) *
                     (_Float16)sign;
      } else {
        typedef f32x4 f32x4u __attribute__((aligned(4)));
        const float *src = static_cast<const float *>(p.q) + at;
        float top = 0.0f;
        f32x4 raw[KS][2];
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 2; ++i) {
            raw[s][i] = *reinterpret_cast<const f32x4u *>(src + 16 * s + 4 * i);
#pragma unroll
            for (int c = 0; c < 4; ++c)
              top = fmaxf(top, fabsf(raw[s][i][c]));
          }
        top = fmaxf(top, other_half(top));
        // the row's largest |q| into [2^14, 2^15); the factor ends at 2^127,
        // which leaves rows below 2^-112 as exact (f32's denormals end there)
        int e = 15 - __builtin_amdgcn_frexp_expf(top);
        e = top > 0.0f ? min(e, 127) : 0;
        const float up = ldexpf(sign, e);
        scale2 = scale2 * ldexpf(1.0f, -e);
#pragma unroll
        for (int s = 0; s < KS; ++s)
#pragma unroll
          for (int i = 0; i < 8; ++i) {
            float x = raw[s][i / 4][i % 4] * up;
#pragma unroll
            for (int n = 0; n < NQ; ++n) {
              qf[n][s][i] = (_Float16)x;
              x = (x - (float)qf[n][s][i]) * (n == 0 ? kLowScale : 1.0f);
            }
          }
      }
    }
    // A scale that underflows (or 0) keeps every finite score at 0 and a
    // masked one (-inf) at -inf.
    scale2 = scale2 < kMinScale ? kMinScale : scale2;
    // The loads of q end here: the compiler places its waits before the first
    // use, and one inside the loop would also wait for the tile in flight.
#pragma unroll
    for (int n = 0; n < NQ; ++n)
#pragma unroll
      for (int s = 0; s < KS; ++s)
        asm volatile("" : "+v"(qf[n][s]));

    State<DH> st;
    st.clear();
    const uint64_t bits = t1 * BK > w.committed ? w.drafts(p) : 0ull;
    const _Float16 *kt = static_cast<const _Float16 *>(p.kt) + (uint64_t)w.kvh * DH * p.t_max;
    const _Float16 *vv = static_cast<const _Float16 *>(p.v) + (uint64_t)w.kvh * p.t_max * DH;
    // Whole tiles go through a uniform base and fixed lane offsets; a tile
    // that runs past the cache clamps every address (keys past t_max are
    // masked, their V rows zeroed below).
    uint32_t koff[LD], voff[LD];
#pragma unroll
    for (int i = 0; i < LD; ++i) {
      const uint32_t q = i * T + tid;
      uint32_t row = q / CK, c = (q % CK) ^ ta_swizzle16(row, CK);
      koff[i] = row * p.t_max + 8u * c;
      row = q / CV, c = (q % CV) ^ ta_swizzle16(row, CV);
      voff[i] = row * DH + 8u * c;
    }
    // K rows that are not whole 16-byte pieces go through registers: fetched
    // before a tile's compute, written to LDS after it.
    f16x8 kreg[DIRECT ? 1 : LD];
    const uint64_t k_left = (uint64_t)(p.kv_heads - w.kvh) * DH * p.t_max;
    auto issue = [&](uint32_t t, uint32_t buf) __attribute__((always_inline)) {
      const uint32_t k0 = t * BK;
      const uint32_t base = __builtin_amdgcn_readfirstlane(lds0 + buf * STAGE + wave * 1024u);
      const _Float16 *ks = kt + k0, *vs = vv + (uint64_t)k0 * DH;
      const bool whole = k0 + BK <= p.t_max;
      if constexpr (DIRECT) {
        if (whole) {
#pragma unroll
          for (int i = 0; i < LD; ++i)
            ta_load_lds16_uniform(ks, koff[i] * 2u, base + i * T * 16u);
        } else {
#pragma unroll
          for (int i = 0; i < LD; ++i) {
            const uint32_t row = (i * T + tid) / CK, key = k0 + koff[i] - row * p.t_max;
            ta_load_lds16_uniform(kt, (row * p.t_max + min(key, p.t_max - 8u)) * 2u, base + i * T * 16u);
          }
        }
      } else {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
          typedef f16x8 f16x8u __attribute__((aligned(2)));
          const uint64_t at = (uint64_t)koff[i] + k0;
          if (at + 8u <= k_left) {
            kreg[i] = *reinterpret_cast<const f16x8u *>(kt + at);
          } else {
#pragma unroll
            for (int x = 0; x < 8; ++x)
              kreg[i][x] = at + x < k_left ? kt[at + x] : (_Float16)0.0f;
          }
        }
      }
      if (whole) {
#pragma unroll
        for (int i = 0; i < LD; ++i)
          ta_load_lds16_uniform(vs, voff[i] * 2u, base + K_BYTES + i * T * 16u);
      } else {
#pragma unroll
        for (int i = 0; i < LD; ++i) {
          const uint32_t row = (i * T + tid) / CV;
          ta_load_lds16_uniform(vs, (voff[i] + (min(k0 + row, p.t_max - 1u) - k0 - row) * DH) * 2u,
                  base + K_BYTES + i * T * 16u);
        }
      }
    };
    auto commit = [&](uint32_t buf) __attribute__((always_inline)) {
      if constexpr (!DIRECT) {
#pragma unroll
        for (int i = 0; i < LD; ++i)
          *reinterpret_cast<f16x8 *>(smem + buf * STAGE + (i * T + tid) * 16u) = kreg[i];
      }
    };

    // Per-lane LDS read offsets (transpose reads: group g of 16 lanes, t).
    const uint32_t g = lane >> 4, t16 = lane & 15u;
    uint32_t k_off[KB], v_off[DB];
    {
      const uint32_t row = 8u * (g >> 1) + (t16 >> 2);
#pragma unroll
      for (int kb = 0; kb < KB; ++kb) {
        const uint32_t col = kh * BKW + kb * 32u + 16u * (g & 1u) + 4u * (t16 & 3u);
        k_off[kb] = row * (BK * 2) + 16u * ((col >> 3) ^ ta_swizzle16(row, CK)) + (col & 7u) * 2u;
      }
      const uint32_t vrow = kh * BKW + 4u * (g >> 1) + (t16 >> 2);
#pragma unroll
      for (int b = 0; b < DB; ++b) {
        const uint32_t col = b * 32u + 16u * (g & 1u) + 4u * (t16 & 3u);
        v_off[b] = K_BYTES + vrow * (DH * 2) + 16u * ((col >> 3) ^ ta_swizzle16(vrow, CV)) + (col & 7u) * 2u;
      }
    }

    // O^T += V^T P^T: step u of a 32-key block pairs P registers 8u..8u+7 (keys
    // 16u + 4h + 0..3 and 16u + 8 + 4h + 0..3) with the same V rows.
    // Operands are read `AHEAD` steps before their use: one by one, every
    // step waited for the LDS.
    // A weight x (2^11 .. 2^15 where it is its row's largest) goes in two f16
    // pieces, hi and the rest of it: within 2^-22 of itself, and below 2^-14 of
    // the row's largest within 2^-36 of that (half of f16's smallest step).  For
    // f16 activations both go into one sum; for f32 ones the second is scaled up
    // and summed apart, which takes the floor to 2^-47.  hi alone would be off by
    // 2^-11 of each weight, all of them to one side where weights coincide.
    f16x8 hi[KB][2], lo[KB][2];
    auto product = [&](uint32_t from) __attribute__((always_inline)) {
      const uint32_t at0 = lds0 + from * STAGE;
      constexpr int STEPS = DB * KB * 2; // (b, kb, u), u fastest
      auto read = [&](int i) __attribute__((always_inline)) {
        const uint32_t at = at0 + v_off[i / (KB * 2)] + (i % (KB * 2)) * 16 * (DH * 2);
        return ta_read_tr16(at, at + 8 * (DH * 2));
      };
      f16x8 v[STEPS];
#pragma unroll
      for (int i = 0; i < AHEAD; ++i)
        v[i] = read(i);
      f32x16 rest;
#pragma unroll
      for (int i = 0; i < STEPS; ++i) {
        if (i + AHEAD < STEPS)
          v[i + AHEAD] = read(i + AHEAD);
        in_order();
        const int b = i / (KB * 2), kb = i / 2 % KB, u = i % 2;
        if (i % (KB * 2) == 0)
          rest = f32x16{};
        st.o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], hi[kb][u], st.o[b], 0, 0, 0);
        if constexpr (IO16)
          st.o[b] = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], lo[kb][u], st.o[b], 0, 0, 0);
        else
          rest = __builtin_amdgcn_mfma_f32_32x32x16_f16(v[i], lo[kb][u], rest, 0, 0, 0);
        in_order();
        if constexpr (!IO16) {
          if (i % (KB * 2) == KB * 2 - 1) {
#pragma unroll
            for (int e = 0; e < 16; ++e)
              st.o[b][e] = fmaf(rest[e], 1.0f / kLowScale, st.o[b][e]);
          }
        }
      }
    };

    if (t0 < t1) {
      issue(t0, 0);
      commit(0);
    }
    if (FLIGHT == 2 && t0 + 1 < t1)
      issue(t0 + 1, 1);
    static_assert(!LATE || KP == 2, "one part is late");
    const bool late = LATE && kh != 0u;
    uint32_t buf = 0, before = BUFS - 1;
    for (uint32_t t = t0; t < t1; ++t) {
      const uint32_t k0 = t * BK, next = buf + 1u == BUFS ? 0u : buf + 1u;
      // tile t landed: all loads but those of the tile after it
      if (FLIGHT == 2 && t + 1 < t1)
        asm volatile("s_waitcnt vmcnt(%0)" ::"n"(2 * LD) : "memory");
      else
        asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
      __syncthreads(); // and every wave is done with the buffer that is filled next
      if (t + FLIGHT < t1)
        issue(t + FLIGHT, FLIGHT == 1 ? next : before);
      if (k0 + BK > w.total) {
        // rows of V past the drafts become zeros (that memory may hold
        // anything, and 0 * inf is not 0)
        const uint32_t first = w.total - min(w.total, k0);
        char *vs = smem + buf * STAGE + K_BYTES;
        for (uint32_t i = first * (DH * 2 / 16) + tid; i < (uint32_t)(BK * DH * 2 / 16); i += T)
          *reinterpret_cast<f32x4 *>(vs + i * 16u) = f32x4{0.0f, 0.0f, 0.0f, 0.0f};
        __syncthreads();
      }
      if (late && t > t0)
        product(before);
      const uint32_t kw0 = k0 + kh * BKW, at0 = lds0 + buf * STAGE;
      f32x16 s[KB], low[KB]; // low: the smaller pieces of q
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
        s[kb] = low[kb] = f32x16{};
      {
        constexpr int STEPS = KS * KB; // (ks, kb), kb fastest
        auto read = [&](int i) __attribute__((always_inline)) {
          const uint32_t at = at0 + k_off[i % KB] + (i / KB) * 16 * (BK * 2);
          return ta_read_tr16(at, at + 4 * (BK * 2));
        };
        f16x8 k[STEPS];
#pragma unroll
        for (int i = 0; i < AHEAD; ++i)
          k[i] = read(i);
#pragma unroll
        for (int i = 0; i < STEPS; ++i) {
          if (i + AHEAD < STEPS)
            k[i + AHEAD] = read(i + AHEAD);
          in_order();
#pragma unroll
          for (int n = 0; n < NQ; ++n) {
            f32x16 &c = n ? low[i % KB] : s[i % KB];
            c = __builtin_amdgcn_mfma_f32_32x32x16_f16(k[i], qf[n][i / KB], c, 0, 0, 0);
          }
          in_order();
        }
      }
      if constexpr (NQ > 1) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[kb][e] = fmaf(low[kb][e], 1.0f / kLowScale, s[kb][e]);
      }
      if (kw0 + BKW > w.committed) {
#pragma unroll
        for (int kb = 0; kb < KB; ++kb)
#pragma unroll
          for (int e = 0; e < 16; ++e)
            s[kb][e] = w.sees(kw0 + kb * 32u + 8u * (e / 4) + 4u * h + e % 4, bits) ? s[kb][e] : -__builtin_inff();
      }
      st.raise(s, scale2);
      const float shift = kF16Shift - st.m;
#pragma unroll
      for (int kb = 0; kb < KB; ++kb)
#pragma unroll
        for (int u = 0; u < 2; ++u)
#pragma unroll
          for (int e = 0; e < 8; e += 2) {
            float x[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              x[i] = exp2_fast(fmaf(s[kb][8 * u + e + i], scale2, shift));
              st.l += x[i];
            }
            f16x2 a = {(_Float16)x[0], (_Float16)x[1]};
            asm("" : "+v"(a)); // widen from the packed pair
#pragma unroll
            for (int i = 0; i < 2; ++i) {
              hi[kb][u][e + i] = a[i];
              lo[kb][u][e + i] = IO16 ? (_Float16)(x[i] - (float)a[i])
                                      : (_Float16)fmaf((float)a[i], -kLowScale, x[i] * kLowScale);
            }
          }
      if (!late)
        product(buf);
      if (t + 1 < t1)
        commit(next);
      before = buf;
      buf = next;
    }
    if (late && t0 < t1)
      product(before);
    if (__any(w.live && !st.finite()))
      whole_values<DH, kF16, IO16>(p, w, st, t0 * BK + kh * BKW, t1 * BK, BK, BKW);
    finish<DH, kF16, IO16, KP>(p, w, st, kh, reinterpret_cast<float *>(smem) + qb * merge_floats<DH, KP>());
  }
};

// -------------------------------------------------------------- f32 caches

// One row tile, KP waves that take 32-key blocks in turn, K and V through
// registers.  Four waves (eight: 46.3 us against 38.5, 16000 positions, 8 kv
// heads, dh 128): a block is 64 loads deep, and eight waves have half the
// registers for them.
template <int DH, int KP> struct TreeF32 {
  static constexpr int HALF = DH / 2, DB = DH / 32, BK = 32;
  static constexpr int Q_FLOATS = HALF * 64, MERGE = merge_floats<DH, KP>();
  static constexpr int SMEM = Q_FLOATS > MERGE ? Q_FLOATS : MERGE;
  typedef float vrow __attribute__((ext_vector_type(DB)));

  // K row s + h dh / 2 of step s, key k0 + j.
  static TA_DEVICE void load_k(const float *kt, const TreeArgs &p, const Place &w, uint32_t k0, float (&r)[HALF]) {
    const float *base = kt + (k0 + BK <= p.t_max ? k0 : 0u);
    const uint32_t lane = w.h * HALF * p.t_max + (k0 + BK <= p.t_max ? w.j : min(k0 + w.j, p.t_max - 1u));
#pragma unroll
    for (int s = 0; s < HALF; ++s)
      r[s] = base[(uint32_t)s * p.t_max + lane];
  }
  // Memory past the drafts may hold anything (0 * inf is not 0): for its keys,
  // whose weights are zeros, the last draft's row.
  static TA_DEVICE void load_v(const float *v, const Place &w, uint32_t k0, vrow (&r)[16]) {
    const float *base = v + (uint64_t)k0 * DH;
    const bool whole = k0 + BK <= w.total;
#pragma unroll
    for (int e = 0; e < 16; ++e) {
      uint32_t key = 8u * (e / 4) + 4u * w.h + e % 4;
      if (!whole)
        key = min(key, w.total - 1u - k0);
      r[e] = *reinterpret_cast<const vrow *>(base + key * DH + w.j * DB);
    }
  }

  static TA_DEVICE void run(const TreeArgs &p) {
    __shared__ __attribute__((aligned(16))) float smem[SMEM];
    const uint32_t wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const Place w(p, 1, 0);
    uint32_t b0, b1;
    chunk_blocks(p, w, BK, b0, b1);
    float sign;
    const float scale2 = split_scale(p.scale, sign);
    const float *kt = static_cast<const float *>(p.kt) + (uint64_t)w.kvh * DH * p.t_max;
    const float *vv = static_cast<const float *>(p.v) + (uint64_t)w.kvh * p.t_max * DH;
    float rk[HALF];
    vrow rv[16];
    uint32_t b = b0 + wave;
    if (b < b1) {
      load_k(kt, p, w, b * BK, rk);
      load_v(vv, w, b * BK, rv);
    }
    // value d = s + h dh / 2 of row r: [s / 4][lane][s % 4]
    load_q<DH, false>(p, w, [&](uint32_t part, uint32_t r, const float(&x)[DH / 8]) __attribute__((always_inline)) {
#pragma unroll
      for (int i = 0; i < DH / 8; i += 4) {
        const uint32_t d = part * (DH / 8) + i, s = d % HALF, lane = 32u * (d / HALF) + r;
        reinterpret_cast<f32x4 *>(smem)[s / 4u * 64u + lane] =
            f32x4{x[i] * sign, x[i + 1] * sign, x[i + 2] * sign, x[i + 3] * sign};
      }
    });
    State<DH> st;
    st.clear();
    const uint64_t bits = b1 * BK > w.committed ? w.drafts(p) : 0ull;
    __syncthreads();
    for (; b < b1; b += KP) {
      const uint32_t k0 = b * BK;
      reread_lds();
      f32x16 t[1] = {f32x16{}};
#pragma unroll
      for (int s = 0; s < HALF; s += 4) {
        const f32x4 q = reinterpret_cast<const f32x4 *>(smem)[s / 4 * 64 + w.lane];
#pragma unroll
        for (int i = 0; i < 4; ++i)
          t[0] = __builtin_amdgcn_mfma_f32_32x32x2f32(rk[s + i], q[i], t[0], 0, 0, 0);
      }
      if (b + KP < b1)
        load_k(kt, p, w, (b + KP) * BK, rk);
      if (k0 + BK > w.committed) {
#pragma unroll
        for (int e = 0; e < 16; ++e)
          t[0][e] = w.sees(k0 + 8u * (e / 4) + 4u * w.h + e % 4, bits) ? t[0][e] : -__builtin_inff();
      }
      st.raise(t, scale2);
#pragma unroll
      for (int e = 0; e < 16; ++e) {
        const float x = exp2_fast(fmaf(t[0][e], scale2, -st.m));
        st.l += x;
#pragma unroll
        for (int d = 0; d < DB; ++d)
          st.o[d] = __builtin_amdgcn_mfma_f32_32x32x2f32(rv[e][d], x, st.o[d], 0, 0, 0);
      }
      if (b + KP < b1)
        load_v(vv, w, (b + KP) * BK, rv);
    }
    if (__any(w.live && !st.finite()))
      whole_values<DH, kF32, false>(p, w, st, (b0 + wave) * BK, b1 * BK, KP * BK, BK);
    finish<DH, kF32, false, KP>(p, w, st, wave, smem);
  }
};

// The chunks of a row tile: a workgroup per (row tile, block b of 32 head
// dimensions, kv head); wave q sums register quad q of that block over the
// chunks, in their order.  What bounds it is latency, so everything is in
// flight at once: the first chunks' outputs before the weights are known.
template <int DH, int KIND, bool IO16> TA_DEVICE void combine(const TreeArgs &p) {
  constexpr int AHEAD = 16;
  __shared__ float weight[TA_TREE_MAX_CHUNKS][32], red[8][32], red_l[8][32];
  const uint32_t kvh = blockIdx.x % p.kv_heads, b = blockIdx.x / p.kv_heads % (DH / 32);
  const uint32_t tile = blockIdx.x / p.kv_heads / (DH / 32);
  const uint32_t lane = threadIdx.x & 63u, j = lane & 31u, h = lane >> 5, q = threadIdx.x >> 6;
  const uint32_t rows = p.tokens * p.group, row = tile * 32u + j;
  const bool live = row < rows;
  const float *part = p.partial + ((uint64_t)tile * p.chunks * p.kv_heads + kvh) * ta_tree_partial(DH);
  const uint64_t step = (uint64_t)p.kv_heads * ta_tree_partial(DH);
  const uint32_t g = threadIdx.x >> 5, last = p.chunks - 1u, at = (b * 4u + q) * 64u + lane;
  f32x4 x[AHEAD];
  if (live) {
#pragma unroll
    for (int c = 0; c < AHEAD; ++c)
      x[c] = reinterpret_cast<const f32x4 *>(part + min((uint32_t)c, last) * step)[at];
  }
  constexpr int PER = TA_TREE_MAX_CHUNKS / 8;
  float m[PER], l[PER], top = kNegMax;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const uint32_t c = g + 8u * i;
    const bool there = live && c < p.chunks;
    m[i] = there ? part[c * step + DH / 2 * 64 + j] : kNegMax;
    l[i] = there ? part[c * step + DH / 2 * 64 + 32 + j] : 0.0f;
  }
#pragma unroll
  for (int i = 0; i < PER; ++i)
    top = fmaxf(top, m[i]);
  red[g][j] = top;
  __syncthreads();
#pragma unroll
  for (int i = 0; i < 8; ++i)
    top = fmaxf(top, red[i][j]);
  float sum = 0.0f;
#pragma unroll
  for (int i = 0; i < PER; ++i) {
    const float a = exp2_fast(m[i] - top);
    weight[g + 8 * i][j] = a;
    sum = fmaf(l[i], a, sum);
  }
  red_l[g][j] = sum;
  __syncthreads();
  if (!live)
    return;
  sum = 0.0f;
#pragma unroll
  for (int i = 0; i < 8; ++i)
    sum += red_l[i][j];
  f32x4 v = {0.0f, 0.0f, 0.0f, 0.0f};
  for (uint32_t c0 = 0; c0 < p.chunks; c0 += AHEAD) {
    f32x4 y[AHEAD];
#pragma unroll
    for (int c = 0; c < AHEAD; ++c)
      y[c] = x[c];
    if (c0 + AHEAD < p.chunks) {
#pragma unroll
      for (int c = 0; c < AHEAD; ++c)
        x[c] = reinterpret_cast<const f32x4 *>(part + min(c0 + AHEAD + c, last) * step)[at];
    }
#pragma unroll
    for (int c = 0; c < AHEAD; ++c) {
      if (c0 + c < p.chunks) {
        const float a = weight[c0 + c][j];
#pragma unroll
        for (int r = 0; r < 4; ++r)
          v[r] = fmaf(y[c][r], a, v[r]);
      }
    }
  }
  const float inv = sum > 0.0f ? 1.0f / sum : sum == sum ? 0.0f : sum;
  const uint32_t token = row / p.group, head = kvh * p.group + row % p.group;
  const uint64_t to = ((uint64_t)token * p.kv_heads * p.group + head) * DH;
#pragma unroll
  for (int r = 0; r < 4; ++r) {
    const uint64_t d = to + out_dim<DH, KIND>(b, q, r, h);
    if constexpr (IO16)
      static_cast<_Float16 *>(p.out)[d] = (_Float16)(v[r] * inv);
    else
      static_cast<float *>(p.out)[d] = v[r] * inv;
  }
}

} // namespace

#define TA_TREE(NAME, THREADS, WAVES, ...)                                                         \
  extern "C" __global__ __launch_bounds__(THREADS, WAVES) void ta_tree_##NAME(TreeArgs p) { __VA_ARGS__::run(p); }
#define TA_TREE_COMBINE(NAME, DH, KIND, IO16)                                                        \
  extern "C" __global__ __launch_bounds__(kThreads) void ta_tree_combine_##NAME##_dh##DH(TreeArgs p) { \
    combine<DH, KIND, IO16>(p);                                                                    \
  }
// f16 caches: 32, 64 (dh 128) and 128 rows to a workgroup, and `_any` forms for
// caches whose K rows are not whole 16-byte pieces.  Those hold a tile's share
// of K in registers.  A CU runs one of these workgroups, so four waves may have
// a SIMD's registers to themselves where half of them would spill: f32 q at dh
// 128 (64 rows, 16000 positions, 8 kv heads: 33.2 us, 55.1 spilling).  Where
// nothing spills half is faster (f32 q, dh 64: 21.3 us against 23.3).
#define TA_TREE_F16(NAME, DH, IO16)                                                                \
  TA_TREE(NAME##_dh##DH##_r32, 256, 2, TreeF16<DH, IO16, true, 1, 4, 32>)                          \
  TA_TREE(NAME##_dh##DH##_r128, 512, 2, TreeF16<DH, IO16, true, 4, 2, 32>)                         \
  TA_TREE(NAME##_dh##DH##_r32_any, 256, DH == 128 && !IO16 ? 1 : 2,                                \
          TreeF16<DH, IO16, false, 1, 4, 32>)                                                      \
  TA_TREE(NAME##_dh##DH##_r128_any, 512, 2, TreeF16<DH, IO16, false, 4, 2, 32>)                    \
  TA_TREE_COMBINE(NAME, DH, kF16, IO16)
#define TA_TREE_F16_R64(NAME, IO16)                                                                \
  TA_TREE(NAME##_dh128_r64, 256, 2, TreeF16<128, IO16, true, 2, 2, 32>)                            \
  TA_TREE(NAME##_dh128_r64_any, 256, IO16 ? 2 : 1, TreeF16<128, IO16, false, 2, 2, 32>)
#define TA_TREE_Q8(NAME, DH, IO16)                                                                 \
  TA_TREE(NAME##_dh##DH##_r16, 512, 2, TreeQ8Few<DH, IO16, 8>)                                     \
  TA_TREE(NAME##_dh##DH##_r32, 512, 2, TreeQ8<DH, IO16, 8>)                                        \
  TA_TREE_COMBINE(NAME, DH, kQ8, IO16)
#define TA_TREE_DH(DH)                                                                             \
  TA_TREE(f32_dh##DH##_r32, 256, 2, TreeF32<DH, 4>)                                                \
  TA_TREE_COMBINE(f32, DH, kF32, false)                                                            \
  TA_TREE_F16(kv16, DH, false)                                                                     \
  TA_TREE_F16(f16, DH, true)                                                                       \
  TA_TREE_Q8(q8, DH, false)                                                                        \
  TA_TREE_Q8(q8_f16, DH, true)
TA_TREE_DH(64)
TA_TREE_DH(128)
TA_TREE_F16_R64(kv16, false)
TA_TREE_F16_R64(f16, true)
