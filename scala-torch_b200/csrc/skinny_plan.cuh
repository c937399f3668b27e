// How the skinny form (gemm_skinny.cu) cuts a product and what scratch that takes.  Host arithmetic alone, without CUDA.
#pragma once

#include <algorithm>
#include <cstdint>

namespace stb {

constexpr int SK_BM = 128, SK_BK = 64, SK_ROWS = 64;  // rows of W and columns of K in an iteration; token rows of a block

struct SkinnyPlan {
  int nt, tiles, kbs, grid, pmax;
  long long iters;
  uint64_t x3_bytes, part_bytes;
};

// Token rows of the activation-term tile for a block of M <= 64 rows: 16, 32 or 64.
inline int skinny_nt(int M) { return M <= 16 ? 16 : (M <= 32 ? 32 : 64); }

constexpr int skinny_ctas_per_sm(int nt) { return nt == 64 ? 1 : 2; }

// One block of M <= 64 token rows on `sms` multiprocessors.
inline SkinnyPlan skinny_plan_of(int M, int N, int K, int sms) {
  SkinnyPlan q;
  q.nt = skinny_nt(M);
  q.tiles = (N + SK_BM - 1) / SK_BM;
  q.kbs = (K + SK_BK - 1) / SK_BK;
  q.iters = (long long)q.tiles * q.kbs;
  q.grid = (int)std::min<long long>((long long)skinny_ctas_per_sm(q.nt) * sms, q.iters);
  const long long per = q.iters / q.grid;  // every range holds per or per + 1 iterations
  q.pmax = (int)std::min<long long>(q.grid, (q.kbs + per - 1) / per + 1);
  q.x3_bytes = ((uint64_t)3 * q.nt * K * 2 + 255) & ~255ull;
  q.part_bytes = (uint64_t)q.tiles * q.pmax * M * SK_BM * 4;
  return q;
}

// Scratch of a call of M rows: its blocks of 64 take it in turn.  The last one, of M % 64 rows, may take more than a whole
// one: tiles of 32 rows run on twice as many CTAs, which leave more pieces (6144 x 768: 13 of a tile's against 5).
inline uint64_t skinny_bytes_of(int M, int N, int K, int sms) {
  uint64_t need = 0;
  for (int m : {std::min(M, SK_ROWS), M > SK_ROWS ? M % SK_ROWS : 0})
    if (m > 0) {
      const SkinnyPlan q = skinny_plan_of(m, N, K, sms);
      need = std::max(need, q.x3_bytes + q.part_bytes);
    }
  return need;
}

// Scratch that serves every call of 1 .. rows rows, and of more where rows >= 64: within a tile's height more rows take more.
inline uint64_t skinny_bytes_up_to(int rows, int N, int K, int sms) {
  uint64_t need = 0;
  for (int nt : {16, 32, SK_ROWS}) need = std::max(need, skinny_bytes_of(std::min(nt, std::min(rows, SK_ROWS)), N, K, sms));
  return need;
}

}  // namespace stb
