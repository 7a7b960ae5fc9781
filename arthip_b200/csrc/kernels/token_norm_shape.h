// How the norm of rows of any width, stride and alignment shares a row out over threads: a group
// of GROUP threads (a warp, or several for wide rows), LANES of them to a row, N elements to a
// lane. Element e of a row is lane e % LANES'. Host code without kernels, so that every width
// can be walked through where there is no GPU.
#pragma once

namespace ah {
namespace token_norm {

// visit.template operator()<GROUP, LANES, N>() with the N of the even numbers [LO, HI] that C of
// [MIN_C, MAX_C] needs: the first that holds the row. N is at most one more than a lane needs, so
// that only elements (N - 2) * LANES on may lie behind the row, and the kernel tests only those.
template <int GROUP, int LANES, int LO, int HI, int MIN_C, int MAX_C, typename Visit>
auto staged_by_count(int C, const Visit& visit) {
  static_assert(LO % 2 == 0 && HI % 2 == 0 && LO <= HI, "an even number of elements a lane");
  static_assert((LO - 2) * LANES <= MIN_C, "untested elements of the narrowest row lie behind it");
  static_assert(MAX_C <= HI * LANES, "the widest row does not fit");
  if constexpr (LO < HI)
    if (C > LO * LANES) return staged_by_count<GROUP, LANES, LO + 2, HI, LO * LANES + 1, MAX_C>(C, visit);
  return visit.template operator()<GROUP, LANES, LO>();
}

// 9 to 16 elements a lane: a row's fixed work (the sums across lanes, the choices) is shared by
// as many rows at once as that leaves lanes for. Above 4096 channels a block has no more threads
// to give.
template <typename Visit>
auto staged_shape(int C, const Visit& visit) {
  if (C <= 32) return staged_by_count<32, 4, 2, 8, 1, 32>(C, visit);
  if (C <= 64) return staged_by_count<32, 4, 10, 16, 33, 64>(C, visit);
  if (C <= 128) return staged_by_count<32, 8, 10, 16, 65, 128>(C, visit);
  if (C <= 256) return staged_by_count<32, 16, 10, 16, 129, 256>(C, visit);
  if (C <= 512) return staged_by_count<32, 32, 10, 16, 257, 512>(C, visit);
  if (C <= 1024) return staged_by_count<64, 64, 10, 16, 513, 1024>(C, visit);
  if (C <= 2048) return staged_by_count<128, 128, 10, 16, 1025, 2048>(C, visit);
  if (C <= 4096) return staged_by_count<256, 256, 10, 16, 2049, 4096>(C, visit);
  return staged_by_count<256, 256, 18, 32, 4097, 8192>(C, visit);
}

}  // namespace token_norm
}  // namespace ah
