// C ABI of the attention of drafted token trees over a paged cache. Declared in include/spfa_b200.h.
#include <cmath>

#include "tree_launch.cuh"

namespace spfa {
namespace {

constexpr int kCtas = 296;  // of the tensor-core context kernel: two on each of 148 SMs

struct TreeLayout {
  int d_pad;
  int64_t rows;
  size_t cut, ml, O, total;
};
TreeLayout tree_layout(const spfa_kv_cache* c, int dtype, int64_t n_rows, int64_t n_q_heads) {
  TreeLayout t{};
  // either context kernel must fit: which one runs is settled by the call
  const int64_t pieces = (dtype != SPFA_DTYPE_F32 && c->d <= 128) ? 128 * kCtas : 32 * kCtas;
  t.d_pad = (c->d + 3) / 4 * 4;
  t.rows = n_rows * n_q_heads + pieces;
  t.cut = 0;
  t.ml = align_up((size_t)(c->n_seq + 1) * 8);
  t.O = t.ml + align_up((size_t)t.rows * 8);
  t.total = t.O + align_up((size_t)t.rows * t.d_pad * 4);
  return t;
}

int check_tree(const spfa_kv_cache* c, int dtype, int64_t n_rows, int64_t n_q_heads) {
  const int rc = check_cache(c, dtype);
  if (rc != SPFA_OK) return rc;
  if (n_rows < 0 || n_q_heads < 1 || n_q_heads % c->n_heads) return SPFA_ERR_BAD_ARG;
  if (n_rows > kMost32 || n_q_heads > 65535 || n_rows * n_q_heads > kMost32) return SPFA_ERR_TOO_LARGE;
  return SPFA_OK;
}

// Row tiles that a CTA of the tensor-core kernel takes together: two where a sequence has more rows than one holds, on average. One
// against two, in us: 64 tokens of 8 heads a key head over 16384 float16 / int8 keys 236 : 169, of 4 heads in bfloat16 202 : 164;
// 8 tokens of 4 heads, 256 sequences of 512 keys, 180 : 222, 4 sequences of 8192 e4m3 keys 39 : 52.
int row_tiles_of(const tree::Call& a) { return a.n_rows * a.group > 128LL * a.c.n_seq ? 2 : 1; }

bool tiled_call(const spfa_kv_cache* c, int dtype, const void* Q, const int64_t* Q_stride, int subs) {
  if (dtype == SPFA_DTYPE_F32 || !tree::tiled_shape(c) || !rows_align(Q, Q_stride, 2, 8)) return false;
  return dtype == SPFA_DTYPE_F16 ? tree::usable_f16(c, subs) : tree::usable_bf16(c, subs);
}

// Calls that direct_kernel takes: its CTAs, one on an SM, have their keys in flight at once. The page lists bound the keys; lens is
// not known here. One round against the two kernels (32 query heads of 128, 8 key heads; us): a token over 200 bfloat16 keys
// 11.0 : 12.1, over 500 e4m3 keys 13.1 : 13.2, 16 tokens over 200 bfloat16 keys each 11.6 : 19.4. Two rounds: 500 bfloat16 keys
// 19.0 : 12.1, 16 such tokens 19.7 : 21.2, 200 float32 keys 18.3 : 12.4.
constexpr double kDirectRounds = 1;
bool direct_call(const tree::Call& a, const spfa_kv_cache* c, bool vec) {
  const int size = dtype_bytes(c->dtype);
  // (a cache without pages has no address that a copy of nothing could name)
  if (!vec || c->d > 128 || c->n_pages < 1 || !cache_rows_align(c, 16 / size)) return false;
  const double waves = (double)((a.n_rows * c->n_heads * ((a.group + tree::kDirectRows - 1) / tree::kDirectRows) + 147) / 148);
  const int keys = tree::DirectPlan(c->d * size).warps * 32;
  return waves * (double)((a.c.capacity + keys - 1) / keys) <= kDirectRounds;
}

// One wave of CTAs, or as many as there can be shares of the list: lens is not known here, the page lists bound it.
int grid_of(const tree::Call& a, int ctas) {
  const double tiles = (double)a.tiles_of(a.c.capacity), rows = (double)a.n_rows * a.group / a.unit_rows + a.c.n_seq;
  const double most = tiles * rows * a.c.n_heads;
  return most < ctas ? (most < 1 ? 1 : (int)most) : ctas;
}

}  // namespace
}  // namespace spfa

using namespace spfa;

extern "C" {

size_t spfa_tree_workspace_bytes(const spfa_kv_cache* c, int dtype, int64_t n_rows, int64_t n_q_heads) {
  return check_tree(c, dtype, n_rows, n_q_heads) == SPFA_OK ? tree_layout(c, dtype, n_rows, n_q_heads).total : 0;
}

int spfa_tree_forward(const spfa_kv_cache* c, int dtype, const void* Q, const int64_t* Q_stride, const int32_t* cu_rows,
                      int64_t n_rows, int64_t n_q_heads, const uint8_t* tree_mask, int64_t mask_width, float* m, float* l, void* O,
                      const int64_t* O_stride, int first, void* workspace, size_t workspace_bytes, void* stream) {
  int rc = check_tree(c, dtype, n_rows, n_q_heads);
  if (rc != SPFA_OK) return rc;
  const int size = dtype_bytes(dtype);
  if (!Q || !Q_stride || !cu_rows || !m || !l || !O || !O_stride || mask_width < 0 || (mask_width > 0 && !tree_mask)) return SPFA_ERR_BAD_ARG;
  if (!aligned_to(Q, size) || !aligned_to(O, size) || !aligned4(cu_rows) || !aligned4(m) || !aligned4(l)) return SPFA_ERR_BAD_ARG;
  if (Q_stride[0] < 0 || Q_stride[1] < 0 || O_stride[0] < 0 || O_stride[1] < 0) return SPFA_ERR_BAD_ARG;
  const int64_t count[2] = {n_rows, n_q_heads};
  if (!apart(count, O_stride, 2)) return SPFA_ERR_BAD_ARG;
  const TreeLayout t = tree_layout(c, dtype, n_rows, n_q_heads);
  rc = check_workspace(workspace, workspace_bytes, t.total);
  if (rc != SPFA_OK) return rc;
  if (n_rows == 0 || c->n_seq == 0) return SPFA_OK;

  tree::Call a{};
  a.c = cache_view(c);
  a.Q = static_cast<const char*>(Q);
  a.q_stride[0] = Q_stride[0];
  a.q_stride[1] = Q_stride[1];
  a.cu_rows = cu_rows;
  a.n_rows = n_rows;
  a.n_q_heads = (int32_t)n_q_heads;
  a.group = (int32_t)(n_q_heads / c->n_heads);
  a.scale_log2e = (1.0f / sqrtf((float)c->d)) * kLog2e;
  const bool vec = cache_rows_align(c, 4) && rows_align(Q, Q_stride, size, 4) && rows_align(O, O_stride, size, 4);
  const int subs = row_tiles_of(a);
  a.direct = g_path.load() == SPFA_PATH_AUTO && direct_call(a, c, vec);
  const bool tiled = g_path.load() != SPFA_PATH_GATHER && !a.direct && tiled_call(c, dtype, Q, Q_stride, subs);
  if (g_path.load() == SPFA_PATH_TILED && !tiled) return SPFA_ERR_BAD_ARG;
  if (tiled) {
    a.row_tile = 128 * subs;
    const int ps = a.c.page_size, keys = tree::kTiledKeys;
    a.page_tiles = ps >= keys ? (ps + keys - 1) / keys : 0;
    a.tile_keys = ps >= keys ? keys : keys / ps * ps;
  } else {
    a.row_tile = tree::any_rows(a);
    a.tile_keys = tree::any_tile_keys(tree::any_padded(c->d));
    a.page_tiles = 0;
  }
  // whole tokens, so that a warp of the merge can take rows of one unit, where that leaves less than an eighth of the tile unused
  a.unit_rows = a.group * 8 <= a.row_tile ? a.row_tile / a.group * a.group : a.row_tile;
  a.n_cta = grid_of(a, tiled ? kCtas / subs : tree::any_ctas(c->d));
  char* ws = static_cast<char*>(workspace);
  a.cut = reinterpret_cast<int64_t*>(ws + t.cut);
  a.ml = reinterpret_cast<float2*>(ws + t.ml);
  a.O = reinterpret_cast<float*>(ws + t.O);
  a.d_pad = t.d_pad;
  tree::MergeArgs g{};
  g.mask = tree_mask;
  g.mask_width = mask_width;
  g.m = m;
  g.l = l;
  g.O = static_cast<char*>(O);
  g.o_stride[0] = O_stride[0];
  g.o_stride[1] = O_stride[1];
  g.first = first ? 1 : 0;
  cudaStream_t st = (cudaStream_t)stream;
  g_last_path.store(tiled ? SPFA_PATH_TILED : SPFA_PATH_GATHER);
  if (dtype == SPFA_DTYPE_F16) return tree::launch_f16(c, a, g, vec, tiled, st);
  if (dtype == SPFA_DTYPE_BF16) return tree::launch_bf16(c, a, g, vec, tiled, st);
  return tree::launch_f32(c, a, g, vec, st);
}

}  // extern "C"
