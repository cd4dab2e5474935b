// Drafted tokens over a cache: checks and launch geometry of the 8-bit K/V
// cache, tree attention and RoPE on several axes, from shapes alone (no
// device call, so they run without a GPU).
#include <algorithm>
#include <cmath>

#include "internal.hpp"

namespace tensor_ash {

namespace {

std::string str(uint64_t v) { return std::to_string(v); }

uint64_t ceil_div(uint64_t a, uint64_t b) { return (a + b - 1) / b; }

// Elements [offset, offset + (rows - 1) * stride + width) lie within len.
void check_span(const std::string &op, const char *role, uint64_t offset, uint64_t rows, uint64_t stride,
                uint64_t width, uint64_t len) {
  const unsigned __int128 end = (unsigned __int128)offset + (unsigned __int128)(rows - 1) * stride + width;
  if (end > len)
    fail(op + ": " + role + " rows (offset " + str(offset) + ", stride " + str(stride) + ", " + str(rows) + " of " +
         str(width) + ") reach past its " + str(len) + " elements");
}

void check_head_dim(const std::string &op, uint32_t dh) {
  if (dh != 64 && dh != 128)
    fail(op + ": head dimension " + str(dh) + " unsupported (compiled variants: 64, 128)");
}

void check_grid(const std::string &op, uint32_t kv_heads) {
  if (kv_heads > 65535)
    fail(op + ": " + str(kv_heads) + " kv heads exceed the launch grid (65535)");
}

} // namespace

uint64_t Operand::len() const {
  uint64_t n = 1;
  for (uint32_t d : shape)
    n *= d;
  return n;
}

uint32_t q8_blocks(uint32_t t_max) { return (uint32_t)ceil_div(t_max, TA_Q8_BLOCK); }

uint64_t q8_cache_bytes(const CacheShape &c) {
  const std::string op = "q8_cache_create";
  if (c.kv_heads == 0 || c.t_max == 0)
    fail(op + ": kv_heads (" + str(c.kv_heads) + ") and t_max (" + str(c.t_max) + ") must be nonzero");
  check_head_dim(op, c.dh);
  check_grid(op, c.kv_heads);
  if (c.t_max > (1u << 31))
    fail(op + ": t_max " + str(c.t_max) + " exceeds 2^31");
  return (uint64_t)c.kv_heads * q8_blocks(c.t_max) * ta_q8_record(c.dh);
}

CacheShape dense_cache(const std::string &op, const Operand &kt, const Operand &v) {
  if (kt.dtype != v.dtype)
    fail(op + ": kt (" + dtype_name(kt.dtype) + ") and v (" + dtype_name(v.dtype) + ") must share a storage type");
  if (kt.shape.size() != 3)
    fail(op + ": kt must be [H_kv, dh, T_max], got " + fmt_shape(kt.shape));
  if (v.shape.size() != 3)
    fail(op + ": v must be [H_kv, T_max, dh], got " + fmt_shape(v.shape));
  const CacheShape c{kt.shape[0], kt.shape[1], kt.shape[2]};
  if (v.shape[0] != c.kv_heads || v.shape[1] != c.t_max || v.shape[2] != c.dh)
    fail(op + ": inconsistent caches kt " + fmt_shape(kt.shape) + ", v " + fmt_shape(v.shape));
  check_head_dim(op, c.dh);
  check_grid(op, c.kv_heads);
  return c;
}

Q8WritePlan q8_write_plan(const CacheShape &c, const Operand &k, const Operand &v, const Q8WriteDesc &d) {
  const std::string op = "run_q8_cache_write";
  if (k.dtype != v.dtype)
    fail(op + ": k (" + dtype_name(k.dtype) + ") and v (" + dtype_name(v.dtype) + ") must share a storage type");
  if (d.tokens == 0)
    fail(op + ": tokens must be nonzero");
  if ((uint64_t)d.pos_base + d.tokens > c.t_max)
    fail(op + ": pos_base " + str(d.pos_base) + " + tokens " + str(d.tokens) + " exceeds t_max " + str(c.t_max));
  const uint64_t width = (uint64_t)c.kv_heads * c.dh;
  Q8WritePlan p;
  p.args.k_stride = d.k_stride ? d.k_stride : width;
  p.args.v_stride = d.v_stride ? d.v_stride : width;
  check_span(op, "k", d.k_offset, d.tokens, p.args.k_stride, width, k.len());
  check_span(op, "v", d.v_offset, d.tokens, p.args.v_stride, width, v.len());
  p.args.k_offset = d.k_offset;
  p.args.v_offset = d.v_offset;
  p.args.tokens = d.tokens;
  p.args.pos_base = d.pos_base;
  p.args.blocks = q8_blocks(c.t_max);
  p.args.t_max = c.t_max;
  // blocks that the rows touch; a start read on the device may lie anywhere
  // in its block
  const uint32_t start = d.pos_addr ? TA_Q8_BLOCK - 1 : d.pos_base % TA_Q8_BLOCK;
  p.launch.symbol = std::string("ta_q8_write_") + (k.dtype == DType::F16 ? "f16" : "f32") + "_dh" + str(c.dh);
  p.launch.gx = (uint32_t)ceil_div((uint64_t)start + d.tokens, TA_Q8_BLOCK);
  p.launch.gy = c.kv_heads;
  return p;
}

Q8ReadPlan q8_read_plan(const CacheShape &c, const Operand &kt, const Operand &v, const Q8ReadDesc &d) {
  const std::string op = "run_q8_cache_read";
  const CacheShape dst = dense_cache(op, kt, v);
  if (dst.kv_heads != c.kv_heads || dst.dh != c.dh)
    fail(op + ": kt " + fmt_shape(kt.shape) + " does not fit a cache of " + str(c.kv_heads) + " kv heads of " +
         str(c.dh));
  if (d.positions == 0)
    fail(op + ": positions must be nonzero");
  const uint64_t end = (uint64_t)d.first + d.positions;
  if (end > c.t_max || end > dst.t_max)
    fail(op + ": first " + str(d.first) + " + positions " + str(d.positions) + " exceeds the cache's " +
         str(c.t_max) + " or kt's " + str(dst.t_max));
  Q8ReadPlan p;
  p.args.first = d.first;
  p.args.n = d.positions;
  p.args.blocks = q8_blocks(c.t_max);
  p.args.t_dst = dst.t_max;
  p.launch.symbol = std::string("ta_q8_read_") + (kt.dtype == DType::F16 ? "f16" : "f32") + "_dh" + str(c.dh);
  p.launch.gx = (uint32_t)(ceil_div(end, TA_Q8_READ_KEYS) - d.first / TA_Q8_READ_KEYS);
  p.launch.gy = c.kv_heads;
  return p;
}

namespace {
// Row tiles of a workgroup, its threads and the fewest keys worth a chunk (a
// round of its waves; two for the larger workgroups of the f16 cache).
struct TreeShape {
  uint32_t tiles, threads, keys;
  std::string suffix;
};
// Measured on 8 kv heads of group 4 (us, f16 / f32 q).
//  * 8-bit cache: a workgroup of two row tiles was not worth its sharing of K
//    and V (64 rows of dh 128 at 16000 positions: 21.2 / 24.8 with one tile,
//    23.4 / 27.0 with two; 256 rows at 65000: 147.0 / 208.9, 148.4 / 209.5).
//    16 rows or fewer: 16.3 / 16.9, on a 32-row tile 18.1 / 19.4.
//  * f16 cache, rows x positions below 2^20: few positions to a chunk, so that
//    the larger workgroups' start weighs more than what they share (128 rows
//    of dh 128 at 4000 positions: two tiles 17.3 / 20.7, four 21.9 / 25.6; of
//    dh 64, one tile 14.0 / 15.8, four 16.7 / 18.6).  Beyond, four tiles at
//    once: 128 rows of dh 128 at 65000 100.5 / 104.1 -> 75.5 / 92.8, 256 rows of
//    it at 32768 77.5 / 101.7 -> 65.1 / 88.8, 256 rows of dh 64 at 8000 22.6 /
//    26.4 -> 20.6 / 24.2.  At the border itself dh 64 is level (16.4 / 19.2,
//    16.6 / 19.0) and two tiles of dh 128 are still ahead (20.8 / 26.2, four
//    23.3 / 27.7 at 128 rows and 8192).
//  * f16 cache, two tiles to a workgroup: dh 128 only (64 rows at 16000:
//    22.8 / 28.3, one tile 25.0 / 32.2; dh 64 18.3 / 20.5, one tile 16.9 / 19.3).
TreeShape tree_shape(TreeCache kind, const CacheShape &c, uint64_t rows, uint64_t tiles, uint64_t keys) {
  if (kind == TreeCache::F32)
    return {1, 256, 128, "_r32"};
  if (kind == TreeCache::Q8)
    return {1, 512, 256, rows <= 16 ? "_r16" : "_r32"};
  // K rows of whole 16-byte pieces are loaded straight into LDS
  const std::string any = c.t_max % 8 == 0 ? "" : "_any";
  if (tiles > 2 && rows * keys >= 1u << 20)
    return {4, 512, 128, "_r128" + any};
  if (tiles > 1 && c.dh == 128)
    return {2, 256, 128, "_r64" + any};
  return {1, 256, 128, "_r32" + any};
}
} // namespace

TreePlan tree_plan(const std::string &op, uint32_t cus, TreeCache kind, const CacheShape &c, const Operand &q,
                   const Operand &out, std::optional<uint32_t> mask_cap, const TreeDesc &d) {
  if (q.dtype != out.dtype)
    fail(op + ": q (" + dtype_name(q.dtype) + ") and out (" + dtype_name(out.dtype) + ") must share a storage type");
  const bool io16 = q.dtype == DType::F16;
  if (io16 && kind == TreeCache::F32)
    fail(op + ": f16 q over an f32 cache is unsupported");
  if (d.tokens == 0 || d.tokens > TA_TREE_MAX_TOKENS)
    fail(op + ": tokens " + str(d.tokens) + " out of range 1..=" + str(TA_TREE_MAX_TOKENS));
  if ((uint64_t)d.kv_len + d.tokens > c.t_max)
    fail(op + ": kv_len " + str(d.kv_len) + " + tokens " + str(d.tokens) + " exceeds T_max " + str(c.t_max));
  if (!std::isfinite(d.scale))
    fail(op + ": scale must be finite");
  if (!std::isfinite(d.scale * 1.44269504088896340736f)) // the kernels' exponents are in base 2
    fail(op + ": scale " + std::to_string(d.scale) + " times log2(e) is past f32");
  const uint64_t per_head = (uint64_t)d.tokens * c.kv_heads * c.dh;
  if (out.len() == 0 || out.len() % per_head != 0)
    fail(op + ": out " + fmt_shape(out.shape) + " must hold tokens*H*dh elements (tokens " + str(d.tokens) + ", dh " +
         str(c.dh) + ", H a multiple of " + str(c.kv_heads) + ")");
  const uint64_t group = out.len() / per_head, width = group * c.kv_heads * c.dh;
  if (mask_cap && *mask_cap < 2 * d.tokens)
    fail(op + ": mask holds " + str(*mask_cap) + " words < " + str(2 * d.tokens) + " for " + str(d.tokens) +
         " tokens");
  TreePlan p;
  TreeArgs &a = p.args;
  a.q_offset = d.q_offset;
  a.q_stride = d.q_stride ? d.q_stride : width;
  check_span(op, "q", d.q_offset, d.tokens, a.q_stride, width, q.len());
  const uint32_t item = kind == TreeCache::F32 ? 4 : 2;
  // the kernels reach K's rows of a head by 32-bit offsets
  if (kind != TreeCache::Q8 && (uint64_t)c.dh * c.t_max * item >= (1ull << 32))
    fail(op + ": T_max " + str(c.t_max) + " is past the 4 GiB that a head's cache may take");
  const uint64_t tiles = ceil_div(d.tokens * group, 32);
  const uint64_t keys = d.pos_addr ? c.t_max : (uint64_t)d.kv_len + d.tokens;
  const TreeShape shape = tree_shape(kind, c, d.tokens * group, tiles, keys);
  const uint64_t groups = ceil_div(tiles, shape.tiles);
  // Chunks: at most a workgroup for every CU (280 for 256 took 16.4 us where
  // 252 took 11.5), each with shape.keys keys at least where the length is
  // known.  With a cell it is the capacity's: 500 positions in a cache of 32768
  // (8 kv heads of 4, dh 128) take 15.5 us for 10.3 by number with one token
  // over 8 bits, 18.8 for 15.0 with 64 over f16.  More chunks cost more than they hide (us at 24 / 32 / 48 / 64 chunks, 8 kv heads of dh
  // 128, 32000 positions: f16, 32 rows 30.4 / 30.2 / 37.7 / 36.2, 64 rows 33.9 /
  // 30.8 / 33.8 / 35.3; f32 q on f16, 128 rows 63.8 / 57.2 / 75.1 / 69.8; 8-bit,
  // 32 rows 31.7 / 28.0 / 31.0 / 29.4), and so do chunks of less (f16, 64 rows,
  // 2000 positions: 31 chunks of 64 keys 15.8, 16 of 128 14.0).
  const uint64_t want = std::max<uint64_t>(1, cus / (groups * c.kv_heads));
  const uint64_t most = std::max<uint64_t>(1, keys / shape.keys);
  a.chunks = (uint32_t)std::min<uint64_t>({want, most, TA_TREE_MAX_CHUNKS});
  if (tiles * std::max(a.chunks, c.dh / 32) * c.kv_heads > 0x7FFFFFFFull)
    fail(op + ": " + str(d.tokens * group) + " rows of " + str(c.kv_heads) + " kv heads exceed the launch grid");
  a.kv_len = d.kv_len;
  a.tokens = d.tokens;
  a.kv_heads = c.kv_heads;
  a.group = (uint32_t)group;
  a.t_max = c.t_max;
  a.blocks = q8_blocks(c.t_max);
  a.row_tiles = (uint32_t)tiles;
  a.scale = d.scale;
  const std::string name = std::string(kind == TreeCache::F32   ? "f32"
                                       : kind == TreeCache::F16 ? (io16 ? "f16" : "kv16")
                                                                : (io16 ? "q8_f16" : "q8")) +
                           "_dh" + str(c.dh);
  p.stage.symbol = "ta_tree_" + name + shape.suffix;
  p.stage.gx = (uint32_t)(groups * a.chunks * c.kv_heads);
  p.stage.threads = shape.threads;
  if (a.chunks > 1) {
    p.combine.symbol = "ta_tree_combine_" + name;
    p.combine.gx = a.row_tiles * (c.dh / 32) * c.kv_heads;
    p.partial_bytes = (uint64_t)a.row_tiles * a.chunks * c.kv_heads * ta_tree_partial(c.dh) * 4;
  }
  return p;
}

RopeAxesPlan rope_axes_plan(uint32_t cus, const Operand &input, const Operand &table, uint32_t cell_cap,
                            const Operand &output, const RopeAxesDesc &d) {
  const std::string op = "run_rope_axes";
  if (input.dtype != output.dtype)
    fail(op + ": input (" + dtype_name(input.dtype) + ") and output (" + dtype_name(output.dtype) +
         ") must share a storage type");
  if (table.dtype != DType::F32)
    fail(op + ": table must be f32 storage (got " + dtype_name(table.dtype) + ")");
  if (input.shape != output.shape)
    fail(op + ": output shape " + fmt_shape(output.shape) + " must equal input shape " + fmt_shape(input.shape));
  if (d.rot_dim < 2 || d.rot_dim % 2 != 0 || d.rot_dim > d.head_dim)
    fail(op + ": rot_dim " + str(d.rot_dim) + " must be even, >= 2, and <= head_dim " + str(d.head_dim));
  const uint64_t vec = (uint64_t)d.heads * d.head_dim;
  if (vec == 0 || input.len() % vec != 0)
    fail(op + ": input length " + str(input.len()) + " is not a multiple of heads*head_dim " + str(vec));
  const uint64_t tokens = input.len() / vec;
  if (tokens > UINT32_MAX)
    fail(op + ": token count exceeds u32");
  if (d.sections.empty() || d.sections.size() > TA_ROPE_MAX_AXES)
    fail(op + ": " + str(d.sections.size()) + " axes out of range 1..=" + str(TA_ROPE_MAX_AXES));
  RopeAxesPlan p;
  RopeAxesArgs &a = p.args;
  uint64_t sum = 0;
  for (size_t i = 0; i < d.sections.size(); ++i) {
    if (d.sections[i] == 0)
      fail(op + ": sections[" + str(i) + "] must be nonzero");
    sum += d.sections[i];
    a.ends[i] = (uint32_t)std::min<uint64_t>(sum, UINT32_MAX);
  }
  if (sum != d.rot_dim / 2)
    fail(op + ": sections hold " + str(sum) + " pairs, rot_dim/2 is " + str(d.rot_dim / 2));
  const uint64_t rows = table.len() / d.rot_dim;
  if (rows == 0 || table.len() % d.rot_dim != 0)
    fail(op + ": table length " + str(table.len()) + " is not a multiple of rot_dim " + str(d.rot_dim));
  if ((uint64_t)cell_cap < tokens * d.sections.size())
    fail(op + ": positions hold " + str(cell_cap) + " values < " + str(tokens * d.sections.size()) + " for " +
         str(tokens) + " tokens on " + str(d.sections.size()) + " axes");
  a.tokens = (uint32_t)tokens;
  a.heads = d.heads;
  a.head_dim = d.head_dim;
  a.rot_dim = d.rot_dim;
  a.pos_base = d.pos_base;
  a.axes = (uint32_t)d.sections.size();
  a.table_rows = (uint32_t)std::min<uint64_t>(rows, UINT32_MAX);
  a.io_f16 = input.dtype == DType::F16;
  a.vec4 = d.head_dim % 8 == 0 && d.rot_dim % 8 == 0;
  // a workgroup per token until every CU has eight
  const uint64_t per = std::clamp<uint64_t>(tokens / (8ull * cus), 1, TA_ROPE_GROUP_TOKENS);
  p.launch.symbol = "ta_rope_axes";
  p.launch.gx = (uint32_t)ceil_div(tokens, per);
  return p;
}

} // namespace tensor_ash
