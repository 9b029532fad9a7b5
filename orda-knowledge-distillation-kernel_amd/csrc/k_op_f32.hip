// k_op_f32.hip -- the projection's and the feed-forward block's kernels in
// fp32: few rows on the native fp32 MFMA, the rest on the split-operand engine.
#include "op_kernels.hpp"
#include "tile_s3.hpp"

namespace orda {

template <class C, int LA, int LB, class Epi>
static hipError_t s3_go(const OpPlan& pl, TileParams P, const Epi& E, hipStream_t s) {
  const int64_t bn = Epi::kDual ? C::kRowsB / 2 : C::kRowsB;
  P.tiles_m = (int)((P.M + C::kRowsA - 1) / C::kRowsA) * (P.pair > 0 ? 2 : 1);
  P.tiles_n = (int)((E.cols + bn - 1) / bn);
  P.splits = pl.splits;
  P.kps = pl.kps;
  const int64_t items = (int64_t)P.tiles_m * P.tiles_n * P.splits, resident = (int64_t)persistent_groups() * (C::MB == 4 ? 1 : 3);
  hipLaunchKernelGGL((k_tile_s3<C, LA, LB, Epi>), dim3((unsigned)(items < resident ? items : resident)), dim3(C::kThreads), 0, s, P, E);
  return hipGetLastError();
}
template <int LA, int LB, class Epi>
static hipError_t s3_tile(const OpPlan& pl, const TileParams& P, const Epi& E, hipStream_t s) {
  return pl.tile == 256 ? s3_go<S3Big, LA, LB>(pl, P, E, s) : s3_go<S3Small, LA, LB>(pl, P, E, s);
}

template <> hipError_t launch_op_linear<float>(const OpPlan& pl, int la, int lb, TileParams P, const EpiLinear<float>& E, float* part, hipStream_t s) {
  if (pl.engine == OP_SKINNY) return la == KMAJ && lb == KMAJ ? skinny_go<float>(P, E, s) : hipErrorInvalidValue;
  return with_splits(pl, P, E, part, s, [&](const auto& e) {
    if (la == MNMAJ) return s3_tile<MNMAJ, MNMAJ>(pl, P, e, s);
    if (lb == MNMAJ) return s3_tile<KMAJ, MNMAJ>(pl, P, e, s);
    return s3_tile<KMAJ, KMAJ>(pl, P, e, s);
  });
}
template <> hipError_t launch_op_gate<float>(const OpPlan& pl, TileParams P, const EpiGate<float>& E, float* part, hipStream_t s) {
  if (pl.engine == OP_SKINNY) return skinny_go<float>(P, E, s);
  return with_splits(pl, P, E, part, s, [&](const auto& e) { return s3_tile<KMAJ, KMAJ>(pl, P, e, s); });
}
template <> hipError_t launch_op_gate_grad<float>(const OpPlan& pl, TileParams P, const EpiGateGrad<float>& E, float* part, hipStream_t s) {
  return with_splits(pl, P, E, part, s, [&](const auto& e) { return s3_tile<KMAJ, MNMAJ>(pl, P, e, s); });
}
template <> hipError_t launch_dz<float>(const DzParams& P, hipStream_t s) { return dz_go<float>(P, s); }
template <> hipError_t launch_colsum<float>(const float* p, int64_t b, int64_t c, void* o, hipStream_t s) { return colsum_go<float>(p, b, c, o, s); }

}  // namespace orda
