// Host-side unit tests (no GPU) of the drafted-token ops' checks and launch
// geometry (draft_ops.cpp): what is refused, and that what is launched stays
// inside its buffers.  Built and run by tests/test_draft_ops_cpu.py.
#include <cmath>
#include <cstdio>
#include <functional>
#include <string>
#include <vector>

#include "../../tensor-ash_amd/csrc/runtime/internal.hpp"

using namespace tensor_ash;

static int g_fail = 0, g_pass = 0;
#define CHECK(...)                                                                   \
  do {                                                                               \
    if (__VA_ARGS__)                                                                 \
      ++g_pass;                                                                      \
    else {                                                                           \
      ++g_fail;                                                                      \
      std::printf("FAIL %s:%d: %s\n", __FILE__, __LINE__, #__VA_ARGS__);             \
    }                                                                                \
  } while (0)

static std::string error_of(const std::function<void()> &f) {
  try {
    f();
  } catch (const Error &e) {
    return e.what();
  }
  return "";
}
static bool has(const std::string &s, const char *sub) { return s.find(sub) != std::string::npos; }

static const Operand f32(std::vector<uint32_t> s) { return {s, DType::F32}; }
static const Operand f16(std::vector<uint32_t> s) { return {s, DType::F16}; }

static void test_q8() {
  CHECK(q8_cache_bytes({4, 64, 2048}) == 4ull * 64 * (64 * 64 + 128));
  CHECK(q8_cache_bytes({1, 128, 1}) == 64 * 128 + 128);
  CHECK(q8_cache_bytes({8, 128, 33}) == 8ull * 2 * (64 * 128 + 128));
  CHECK(q8_cache_bytes({2, 128, 1u << 31}) == 2ull * (1u << 26) * 8320); // past 32 bits
  CHECK(has(error_of([] { q8_cache_bytes({0, 64, 8}); }), "must be nonzero"));
  CHECK(has(error_of([] { q8_cache_bytes({4, 64, 0}); }), "must be nonzero"));
  CHECK(has(error_of([] { q8_cache_bytes({4, 96, 8}); }), "head dimension 96 unsupported"));
  CHECK(has(error_of([] { q8_cache_bytes({65536, 64, 8}); }), "launch grid"));
  CHECK(has(error_of([] { q8_cache_bytes({1, 64, (1u << 31) + 1}); }), "exceeds 2^31"));

  // every slot of a block once
  uint32_t seen = 0;
  for (uint32_t k = 0; k < 32; ++k)
    seen |= 1u << ta_q8_slot(k);
  CHECK(seen == 0xFFFFFFFFu);

  const CacheShape c{4, 64, 100};
  Q8WriteDesc d;
  d.tokens = 5;
  d.pos_base = 30;
  auto p = q8_write_plan(c, f32({5, 256}), f32({5, 256}), d);
  CHECK(p.launch.symbol == "ta_q8_write_f32_dh64" && p.launch.gx == 2 && p.launch.gy == 4);
  CHECK(p.args.k_stride == 256 && p.args.blocks == 4 && p.args.t_max == 100);
  d.pos_base = 32;
  CHECK(q8_write_plan(c, f16({5, 256}), f16({5, 256}), d).launch.gx == 1);
  d.pos_addr = 64; // the start may be the last position of a block
  CHECK(q8_write_plan(c, f32({5, 256}), f32({5, 256}), d).launch.gx == 2);
  d.pos_addr = 0;
  d.pos_base = 96;
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 256}), f32({5, 256}), d); }), "exceeds t_max 100"));
  d.pos_base = 0xFFFFFFFFu;
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 256}), f32({5, 256}), d); }), "exceeds t_max"));
  d.pos_base = 95;
  CHECK(error_of([&] { q8_write_plan(c, f32({5, 256}), f32({5, 256}), d); }).empty());
  d.tokens = 0;
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 256}), f32({5, 256}), d); }), "tokens must be nonzero"));
  d.tokens = 5;
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 256}), f16({5, 256}), d); }), "share a storage type"));
  CHECK(has(error_of([&] { q8_write_plan(c, f32({4, 256}), f32({5, 256}), d); }), "k rows"));
  d.v_offset = 1;
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 256}), f32({5, 256}), d); }), "v rows"));
  d.v_offset = 512;
  d.k_offset = 256;
  d.k_stride = d.v_stride = 768;
  CHECK(error_of([&] { q8_write_plan(c, f32({5, 768}), f32({5, 768}), d); }).empty());
  d.k_stride = UINT64_MAX; // the span overflows 64 bits
  CHECK(has(error_of([&] { q8_write_plan(c, f32({5, 768}), f32({5, 768}), d); }), "k rows"));

  Q8ReadDesc r{10, 90};
  auto q = q8_read_plan(c, f16({4, 64, 100}), f16({4, 100, 64}), r);
  CHECK(q.launch.symbol == "ta_q8_read_f16_dh64" && q.launch.gx == 1 && q.launch.gy == 4 && q.args.t_dst == 100);
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 99}), f16({4, 99, 64}), r); }), "exceeds"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 200}), f16({4, 200, 64}), {10, 91}); }), "exceeds"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 100}), f16({4, 100, 64}), {0xFFFFFFFFu, 2}); }), "exceeds"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 100}), f16({4, 100, 64}), {0, 0}); }), "must be nonzero"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({2, 64, 100}), f16({2, 100, 64}), r); }), "does not fit"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 128, 100}), f16({4, 100, 128}), r); }), "does not fit"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 100}), f32({4, 100, 64}), r); }), "share a storage type"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 64, 100}), f16({4, 64, 100}), r); }), "inconsistent caches"));
  CHECK(has(error_of([&] { q8_read_plan(c, f16({4, 6400}), f16({4, 100, 64}), r); }), "kt must be"));
  CHECK(q8_read_plan({4, 64, 1000}, f16({4, 64, 1000}), f16({4, 1000, 64}), {127, 2}).launch.gx == 2);
  CHECK(q8_read_plan({4, 64, 1000}, f16({4, 64, 1000}), f16({4, 1000, 64}), {128, 128}).launch.gx == 1);
}

static void test_tree() {
  const CacheShape c{4, 64, 1000};
  TreeDesc d;
  d.kv_len = 992;
  d.tokens = 8;
  const Operand q = f32({8, 2048}), out = f32({8, 2048});
  auto plan = [&](TreeCache kind, const CacheShape &s, const Operand &a, const Operand &b,
                  std::optional<uint32_t> mask, const TreeDesc &t) { return tree_plan("op", 256, kind, s, a, b, mask, t); };
  auto p = plan(TreeCache::F32, c, q, out, 16u, d);
  CHECK(p.stage.symbol == "ta_tree_f32_dh64_r32" && p.args.group == 8 && p.args.row_tiles == 2);
  CHECK(p.args.chunks >= 1 && p.args.chunks <= TA_TREE_MAX_CHUNKS);
  CHECK(p.stage.gx == p.args.row_tiles * p.args.chunks * 4 && p.stage.threads == 256);
  CHECK(p.partial_bytes == (p.args.chunks > 1 ? 2ull * p.args.chunks * 4 * ta_tree_partial(64) * 4 : 0));
  // rows to a workgroup (by rows, head dimension and rows x positions), and
  // caches whose K rows are not whole 16-byte pieces
  auto f16_of = [&](uint32_t tokens, uint32_t dh, uint32_t t_max, bool cell = false) {
    TreeDesc g;
    g.tokens = tokens;
    g.kv_len = cell ? 0 : t_max - tokens;
    g.pos_addr = cell ? 64 : 0;
    const Operand x = f16({tokens, 16 * dh});
    return plan(TreeCache::F16, {4, dh, t_max}, x, x, std::nullopt, g).stage;
  };
  CHECK(f16_of(8, 64, 1000).symbol == "ta_tree_f16_dh64_r32" && f16_of(8, 64, 1000).threads == 256);
  CHECK(f16_of(9, 64, 1001).symbol == "ta_tree_f16_dh64_r32_any" && f16_of(9, 64, 1001).threads == 256);
  CHECK(f16_of(8, 128, 1000).symbol == "ta_tree_f16_dh128_r32");
  CHECK(f16_of(9, 128, 1001).symbol == "ta_tree_f16_dh128_r64_any" && f16_of(9, 128, 1001).threads == 256);
  CHECK(f16_of(16, 128, 65536).symbol == "ta_tree_f16_dh128_r64");
  CHECK(f16_of(64, 128, 4088).symbol == "ta_tree_f16_dh128_r64" && f16_of(64, 64, 4088).symbol == "ta_tree_f16_dh64_r32");
  CHECK(f16_of(64, 128, 4096).symbol == "ta_tree_f16_dh128_r128" && f16_of(64, 64, 4096).threads == 512);
  CHECK(f16_of(64, 64, 4097).symbol == "ta_tree_f16_dh64_r128_any");
  CHECK(f16_of(64, 64, 4096, true).symbol == "ta_tree_f16_dh64_r128");
  CHECK(plan(TreeCache::F16, c, q, out, std::nullopt, d).stage.symbol == "ta_tree_kv16_dh64_r32");
  CHECK(plan(TreeCache::F16, c, f16({8, 2048}), f16({8, 2048}), std::nullopt, d).stage.symbol == "ta_tree_f16_dh64_r32");
  CHECK(plan(TreeCache::Q8, c, f16({8, 2048}), f16({8, 2048}), std::nullopt, d).stage.symbol == "ta_tree_q8_f16_dh64_r32");
  CHECK(plan(TreeCache::Q8, {4, 128, 1000}, q, out, std::nullopt, d).stage.symbol == "ta_tree_q8_dh128_r32");
  CHECK(plan(TreeCache::Q8, {16, 128, 1000}, q, out, std::nullopt, d).stage.symbol == "ta_tree_q8_dh128_r16");
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, f16({8, 2048}), f16({8, 2048}), 16u, d); }), "f16 q over an f32"));
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, f16({8, 2048}), 16u, d); }), "share a storage type"));
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, 15u, d); }), "mask holds 15 words < 16"));
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, f32({8, 2000}), 16u, d); }), "out [8, 2000] must hold"));
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, f32({7, 2048}), out, 16u, d); }), "q rows"));
  TreeDesc e = d;
  e.kv_len = 993;
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, 16u, e); }), "exceeds T_max 1000"));
  e = d;
  e.kv_len = 0xFFFFFFFFu;
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, 16u, e); }), "exceeds T_max"));
  e = d;
  e.kv_len = 0;
  CHECK(error_of([&] { plan(TreeCache::F32, c, q, out, 16u, e); }).empty());
  for (uint32_t t : {0u, 65u}) {
    e = d;
    e.tokens = t;
    CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, std::nullopt, e); }), "out of range 1..=64"));
  }
  for (float s : {INFINITY, -INFINITY, NAN}) {
    e = d;
    e.scale = s;
    CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, 16u, e); }), "scale must be finite"));
  }
  e = d;
  e.q_stride = 3000;
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, q, out, 16u, e); }), "q rows"));
  CHECK(error_of([&] { plan(TreeCache::F32, c, f32({8, 3000}), out, 16u, e); }).empty());
  e.q_offset = 952; // the last row ends with the tensor
  CHECK(error_of([&] { plan(TreeCache::F32, c, f32({8, 3000}), out, 16u, e); }).empty());
  e.q_offset = 953;
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, f32({8, 3000}), out, 16u, e); }), "q rows"));
  e.q_offset = UINT64_MAX;
  CHECK(has(error_of([&] { plan(TreeCache::F32, c, f32({8, 3000}), out, 16u, e); }), "q rows"));
  // a head's dense cache past 32-bit offsets; the 8-bit one has no such bound
  const CacheShape far{1, 128, 1u << 23};
  CHECK(has(error_of([&] { plan(TreeCache::F32, far, q, f32({8, 128}), 16u, d); }), "4 GiB"));
  CHECK(error_of([&] { plan(TreeCache::F16, far, q, f32({8, 128}), 16u, d); }).empty());
  CHECK(error_of([&] { plan(TreeCache::Q8, far, q, f32({8, 128}), 16u, d); }).empty());

  // geometry over many sizes: the grid fits, every chunk has a slot
  for (uint32_t cus : {1u, 64u, 256u, 304u})
    for (uint32_t heads : {1u, 2u, 5u, 8u, 64u})
      for (uint32_t group : {1u, 3u, 8u, 16u})
        for (uint32_t t : {1u, 2u, 31u, 64u})
          for (uint32_t len : {0u, 1u, 255u, 256u, 5000u, 200000u})
            for (TreeCache kind : {TreeCache::F32, TreeCache::F16, TreeCache::Q8})
              for (bool cell : {false, true}) {
                TreeDesc g;
                g.kv_len = len;
                g.tokens = t;
                g.pos_addr = cell ? 64 : 0;
                const Operand x = f32({t, heads * group * 64});
                auto r = tree_plan("op", cus, kind, {heads, 64, len + t}, x, x, 2 * t, g);
                const std::string &n = r.stage.symbol;
                const uint32_t rows = has(n, "_r32") || has(n, "_r16") ? 1 : has(n, "_r64") ? 2 : 4;
                const uint64_t wgs = (uint64_t)((r.args.row_tiles + rows - 1) / rows) * r.args.chunks * heads;
                CHECK(r.args.chunks >= 1 && r.args.chunks <= TA_TREE_MAX_CHUNKS && r.stage.gx == wgs &&
                      r.partial_bytes == (r.args.chunks == 1 ? 0
                                                             : (uint64_t)r.args.row_tiles * r.args.chunks * heads *
                                                                   ta_tree_partial(64) * 4) &&
                      r.args.row_tiles * 32 >= t * group && (r.args.row_tiles - 1) * 32 < t * group &&
                      (r.args.chunks == 1) == (r.combine.gx == 0) &&
                      (r.combine.gx == 0 || r.combine.gx == r.args.row_tiles * 2 * heads));
              }
}

static void test_tree_scale_range() {
  const Operand x = f32({1, 64});
  TreeDesc d;
  d.tokens = 1;
  auto error = [&](float scale) {
    d.scale = scale;
    return error_of([&] { tree_plan("op", 256, TreeCache::F32, {1, 64, 1}, x, x, std::nullopt, d); });
  };
  for (float s : {0.0f, 1e-45f, 1.0f, 2.3e38f, -2.3e38f})
    CHECK(error(s).empty());
  for (float s : {2.4e38f, -2.4e38f, 3.4e38f})
    CHECK(has(error(s), "times log2(e) is past f32"));
}

static void test_rope_axes() {
  RopeAxesDesc d;
  d.heads = 4;
  d.head_dim = 64;
  d.rot_dim = 64;
  d.sections = {8, 12, 12};
  const Operand x = f32({10, 256}), table = f32({100, 32, 2});
  auto p = rope_axes_plan(256, x, table, 30, x, d);
  CHECK(p.args.tokens == 10 && p.args.axes == 3 && p.args.ends[0] == 8 && p.args.ends[1] == 20 &&
        p.args.ends[2] == 32 && p.args.table_rows == 100 && p.args.vec4 == 1 && p.launch.gx == 10);
  CHECK(has(error_of([&] { rope_axes_plan(256, x, table, 29, x, d); }), "positions hold 29 values < 30"));
  CHECK(has(error_of([&] { rope_axes_plan(256, x, table, 30, f16({10, 256}), d); }), "share a storage type"));
  CHECK(has(error_of([&] { rope_axes_plan(256, x, table, 30, f32({10, 4, 64}), d); }), "must equal input shape"));
  CHECK(has(error_of([&] { rope_axes_plan(256, x, f16({100, 32, 2}), 30, x, d); }), "table must be f32"));
  CHECK(has(error_of([&] { rope_axes_plan(256, x, f32({100, 33, 2}), 30, x, d); }), "not a multiple of rot_dim"));
  CHECK(has(error_of([&] { rope_axes_plan(256, f32({10, 250}), table, 30, f32({10, 250}), d); }), "not a multiple"));
  auto bad = [&](std::vector<uint32_t> s, uint32_t rot) {
    RopeAxesDesc e = d;
    e.sections = s;
    e.rot_dim = rot;
    return error_of([&] { rope_axes_plan(256, x, table, 30, x, e); });
  };
  CHECK(has(bad({8, 12, 11}, 64), "sections hold 31 pairs"));
  CHECK(has(bad({0xFFFFFFFFu, 33}, 64), "sections hold"));
  CHECK(has(bad({8, 0, 24}, 64), "sections[1] must be nonzero"));
  CHECK(has(bad({}, 64), "axes out of range"));
  CHECK(has(bad({4, 4, 4, 4, 16}, 64), "axes out of range"));
  CHECK(has(bad({32}, 63), "rot_dim 63 must be even"));
  CHECK(has(bad({33}, 66), "rot_dim 66"));
  CHECK(has(bad({32}, 0), "rot_dim 0"));
  RopeAxesDesc e = d;
  e.heads = 0;
  CHECK(has(error_of([&] { rope_axes_plan(256, x, table, 30, x, e); }), "not a multiple"));
  for (uint32_t t : {1u, 7u, 2047u, 2048u, 2049u, 16384u, 100001u}) {
    RopeAxesDesc g;
    g.heads = 1;
    g.head_dim = g.rot_dim = 2;
    g.sections = {1};
    const Operand y = f32({t, 2});
    auto r = rope_axes_plan(256, y, f32({1, 1, 2}), t, y, g);
    const uint32_t per = (t + r.launch.gx - 1) / r.launch.gx; // as the kernel has it
    CHECK(per <= TA_ROPE_GROUP_TOKENS && (uint64_t)per * r.launch.gx >= t && r.args.vec4 == 0);
  }
}

int main() {
  test_q8();
  test_tree();
  test_tree_scale_range();
  test_rope_axes();
  std::printf("%d checks, %d failed%s\n", g_pass + g_fail, g_fail, g_fail ? "" : ": all passed");
  return g_fail ? 1 : 0;
}
