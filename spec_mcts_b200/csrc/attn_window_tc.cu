// q40_attn_causal_window's kernel for prompts with enough work: that of attn_tc.cuh, and when CTAs share keys.
#include "attn_tc.cuh"

namespace q40 {
namespace window {

int splits_tc(const Args& a) {
  using namespace tc;
  const int64_t blocks = (int64_t)a.H * ((a.S + 2 * BQ - 1) / (2 * BQ));
  Args one = a;
  one.splits = 1;
  const int tiles = Tiles(one, (a.S - 1) / (2 * BQ) * 2 * BQ, 2 * BQ, 0).n;          // of the last block, which has most
  // Least of what a CTA takes for its tiles and what sharing them costs: another launch, and the partial results' way out and back
  // (us; measured: 256 queries x 32 heads, 11 tiles 27.5 alone, 20 in four splits; 512 queries, four tiles 12.7 alone, 19 in two)
  const double tile = a.S > BQ ? 2.1 : 1.4, part = 0.35e-6 * a.S * a.H * (ATTN_D + 2) * sizeof(float);
  int best = 1;
  double least = tile * tiles;
  for (int s = 2; s <= 16 && s * blocks <= 148 && 2 * s <= tiles; ++s) {
    const double t = tile * ((tiles + s - 1) / s) + 3.5 + part * s;
    if (t < least) { least = t; best = s; }
  }
  return best;
}

int launch_tc(const Args& a, int* err, cudaStream_t st) { return tc::launch_form<tc::Plain>(a, err, st); }

}  // namespace window
}  // namespace q40
