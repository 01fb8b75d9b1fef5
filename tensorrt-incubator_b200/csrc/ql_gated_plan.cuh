// Which part of the gated backward pass's second products each CTA pair computes: tiles of 256 x 256 of the gradients and parts of
// their reductions.  Plain C++ as well, so that it can be checked without a device: every step of every tile once.
#pragma once

#include <stdint.h>

#ifdef __CUDACC__
#define QL_PLAN __host__ __device__ __forceinline__
#else
#define QL_PLAN inline
#endif

namespace ql {

// Bands of `group_m` row tiles walk all column tiles together, so the band's rows stay in L2.
QL_PLAN void band_coords(int tile, int tiles_m, int tiles_n, int group_m, int *mt, int *nt) {
  const int per_group = group_m * tiles_n, grp = tile / per_group, first = grp * group_m, size = tiles_m - first < group_m ? tiles_m - first : group_m, local = tile - grp * per_group;
  *mt = first + local % size;
  *nt = local / size;
}

struct GradArgs {
  int M, I, K;
  int layers;                                            // of dG and dU; with 2 (up to 128 tokens) a dX tile's second 128 rows are the remainders'
  // units: a 256 x 256 tile and one of `*_split` parts of its reduction
  int x_tiles_m, x_tiles_n, x_steps, x_split, x_units;   // dX [M, K]: steps of 64 channels, the gate's first, then the up's
  int w_tiles_m, w_tiles_n, w_steps, w_split, w_units;   // dWg and dWu [I, K] each: steps of 64 tokens of a layer
  int x_per;                                             // dX units of a cluster; one more for the first `heavy` ones,
  int heavy, heavy_w;                                    // which then have `heavy_w` weight units, the others the rest.
  int mixed;                                             // instead: units of one length, all dealt out in turn
  int group_m;
  float *x_parts, *w_parts;                              // [split][layers][M][K], [split][2][I][K]: map_dx or map_dwg lead there
                                                         // then; null where there is one part
  const float *largest;                                  // kRanged: what the first stage's CTAs met
  int num_largest;
  int *status;
};

struct Unit {
  bool is_x;
  int row0, col0;       // of the output (dW: of dWg, or of dWu when `up`)
  bool up;
  int step0, step1, part;
};

// The j-th unit of cluster c: its dX units, then its weight units.  Neighbouring clusters hold neighbouring tiles.
QL_PLAN bool get_unit(const GradArgs &a, int c, int clusters, int j, Unit *u) {
  const int turn = c + j * clusters, nx = a.x_per + (c < a.heavy ? 1 : 0);
  if (a.mixed ? turn < a.x_units : j < nx) {
    const int unit = turn, tiles = a.x_tiles_m * a.x_tiles_n, tile = unit % tiles;
    int mt, nt;
    band_coords(tile, a.x_tiles_m, a.x_tiles_n, a.group_m, &mt, &nt);
    u->is_x = true, u->up = false, u->row0 = mt * 256, u->col0 = nt * 256, u->part = unit / tiles;
    u->step0 = (int)((long long)a.x_steps * u->part / a.x_split), u->step1 = (int)((long long)a.x_steps * (u->part + 1) / a.x_split);
    return true;
  }
  j -= nx;
  int unit;
  if (a.mixed) {
    unit = turn - a.x_units;
  } else if (c < a.heavy) {
    if (j >= a.heavy_w) return false;
    unit = j * a.heavy + c;
  } else {
    unit = a.heavy * a.heavy_w + j * (clusters - a.heavy) + (c - a.heavy);
  }
  if (unit >= a.w_units) return false;
  const int tiles = 2 * a.w_tiles_m * a.w_tiles_n, tile = unit % tiles;
  int mt, nt;
  band_coords(tile, 2 * a.w_tiles_m, a.w_tiles_n, a.group_m, &mt, &nt);
  u->is_x = false, u->up = mt >= a.w_tiles_m, u->row0 = (u->up ? mt - a.w_tiles_m : mt) * 256, u->col0 = nt * 256, u->part = unit / tiles;
  u->step0 = (int)((long long)a.w_steps * u->part / a.w_split), u->step1 = (int)((long long)a.w_steps * (u->part + 1) / a.w_split);
  return true;
}

// Layers of dG and dU, 2 with the roundings' remainders: up to 64 tokens, and up to 128, half of a pair's rows, where a gradient is
// of few values over which roundings would average out.  The remainders cost 1 x 64 x 64 1.5 us (7.7 to 9.3) and 16 x 2744 x 1032 0.2
// (23.3 to 23.5), but 77 x 2744 x 1032 3.5 (24.4 to 27.9) and 128 x 11008 x 4096 20 (121 to 141): four steps of tokens no
// longer hide behind writing the weights' gradients.
inline int grad_layers(int M, int I, int K) { return M <= 64 || (M <= 128 && (I <= 256 || K <= 256)) ? 2 : 1; }

// How the units of the second products are cut and dealt out (see GradArgs), for `pairs` CTA pairs.
struct GradPlan {
  GradArgs a;
  int64_t x_part_floats, w_part_floats;
  int clusters; // to launch: get_unit deals the units out over exactly this many
};
inline GradPlan plan_grads(int M, int I, int K, bool want_x, bool want_w, int pairs) {
  GradPlan p;
  GradArgs &a = p.a;
  a.M = M, a.I = I, a.K = K;
  a.x_tiles_m = (M + 255) / 256, a.x_tiles_n = a.w_tiles_n = (K + 255) / 256, a.w_tiles_m = (I + 255) / 256;
  a.layers = grad_layers(M, I, K);
  a.x_steps = 2 * ((I + 63) / 64), a.w_steps = a.layers * ((M + 63) / 64);
  const int64_t x_tiles = want_x ? (int64_t)a.x_tiles_m * a.x_tiles_n : 0, w_tiles = want_w ? 2ll * a.w_tiles_m * a.w_tiles_n : 0;
  // A unit costs its steps and about 8 more to start and write out.  With two tiles a pair or more, dX's long units come first,
  // cut to a pair's share of all steps where they are fewer than the pairs, and a pair that has one more of them gets as many
  // fewer of the weights' as that is worth.  With fewer tiles both reductions are cut into units of one length, dealt out in
  // turn: the length, of the share and fractions of it down to 8, or the whole, that makes the longest pair's time the shortest.
  // 8192 x 1024 x 512 54 us so (67 with the adding of parts thought free), 153 dealt out the first way; 512 x 11008 x 4096 224 us
  // the first way, 250 the second.
  const int64_t share = (x_tiles * a.x_steps + w_tiles * a.w_steps + pairs - 1) / pairs;
  auto cut = [&](int64_t tiles, int steps, int64_t len) { // what is not wanted has no units and no parts
    if (tiles == 0) return 1;
    const int64_t n = (steps + len - 1) / len;
    return (int)(n > 32 ? 32 : n);
  };
  a.mixed = x_tiles + w_tiles < 2 * pairs;
  if (a.mixed) {
    int64_t best = INT64_MAX;
    for (int part = 0; part <= 4; part++) { // 0: nothing is cut
      const int64_t len = part == 0 ? INT32_MAX : (share / part < 8 ? 8 : share / part);
      const int xs = cut(x_tiles, a.x_steps, len), ws = cut(w_tiles, a.w_steps, len);
      const int64_t x_len = x_tiles ? (a.x_steps + xs - 1) / xs : 0, w_len = w_tiles ? (a.w_steps + ws - 1) / ws : 0;
      const int64_t floats = (x_tiles && xs * a.layers > 1 ? (int64_t)xs * a.layers * M * K : 0) + (ws > 1 ? 2ll * ws * I * K : 0);
      const int64_t join = floats ? 9 + floats * 7 / 1000000 : 0; // adding the parts: 2.5 us and their way to memory and back
      const int64_t cost = (x_tiles * xs + w_tiles * ws + pairs - 1) / pairs * ((x_len > w_len ? x_len : w_len) + 8) + join;
      if (cost < best) best = cost, a.x_split = xs, a.w_split = ws;
    }
  } else {
    a.x_split = x_tiles >= pairs ? 1 : cut(x_tiles, a.x_steps, share < 8 ? 8 : share);
    a.w_split = w_tiles >= pairs ? 1 : cut(w_tiles, a.w_steps, share < 8 ? 8 : share);
  }
  a.x_units = (int)(x_tiles * a.x_split), a.w_units = (int)(w_tiles * a.w_split);
  a.x_per = a.x_units / pairs, a.heavy = a.x_units % pairs;
  const double ux = (double)a.x_steps / a.x_split + 8, uw = (double)a.w_steps / a.w_split + 8;
  const double hw = (a.w_units - (pairs - a.heavy) * ux / uw) / pairs;
  a.heavy_w = hw < 0 ? 0 : (int)(hw + 0.5);
  a.group_m = 8; // row tiles walked together; 4, 8, 16, 32 on 4096 x 11008 x 4096: 1.62, 1.55, 1.59, 1.54 ms; on 1024 x 28672 x 8192: 2.12, 2.10, 2.10, 2.20
  a.x_parts = a.w_parts = nullptr;
  a.largest = nullptr, a.num_largest = 0;
  p.x_part_floats = x_tiles > 0 && a.x_split * a.layers > 1 ? (int64_t)a.x_split * a.layers * M * K : 0;
  p.w_part_floats = w_tiles > 0 && a.w_split > 1 ? 2ll * a.w_split * I * K : 0;
  // units dealt out in turn fit any number of clusters
  p.clusters = a.mixed && a.x_units + a.w_units < pairs ? a.x_units + a.w_units : pairs;
  return p;
}

} // namespace ql
