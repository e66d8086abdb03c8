// kv4_sweep.h - the order in which a workgroup of kv4_block_kernel (kv4.hip) fills,
// reads and rewrites its LDS stages.
//
// Shared by the kernel and by the host-side replay ttcd_kv4_block_stages (api.hip), so
// that the CPU tests prove the order that the GPU runs: K(t) and V(t), tile t's converted
// keys and values, lie in stage t & 1 of two each; every wavefront writes a part of a
// stage and reads all of it. So between a write and a read of it, either way round, there
// has to be a barrier.
#pragma once

#include "schedule.h"

namespace ttcd {

template <bool V>
struct Bool {
  static constexpr bool value = V;
};

// Folds tiles t0 .. t1 - 1, t0 < t1. load_k(t), load_v(t) give tile t's codes;
// store_k(codes, t), store_v(codes, t) convert them into tile t's stage; scores(s, t)
// reads K(t) into s; settle(s, t) masks s; fold(s, t) reads V(t) and adds s's
// probabilities times it; s0 and s1 are registers for two tiles' scores.
//
// A turn folds tile t: the scores of t + 1 are issued against the exponentials of t, then
// the second product of t against the conversion of K(t + 2) and V(t + 1) from codes that
// were loaded a turn before. One barrier a turn: K(t) was read in the turn before this
// one, V(t - 1) too. The first turn has none before it, so K(t0)'s scores are followed by
// a barrier of their own. The last turn is code of its own, so that the others have no
// branch between products and exponentials. Tiles past the last are read and written as
// the last: memory that is there, and stages that nothing reads any more.
template <class Codes, class Scores, class LoadK, class LoadV, class StoreK, class StoreV,
          class ReadK, class Settle, class Fold, class Barrier>
TTCD_HD void kv4_sweep(int t0, int t1, Scores& s0, Scores& s1, LoadK load_k, LoadV load_v,
                       StoreK store_k, StoreV store_v, ReadK scores, Settle settle, Fold fold,
                       Barrier barrier) {
  const int end = t1 - 1;
  auto at = [end](int tile) __attribute__((always_inline)) { return tile < end ? tile : end; };
  Codes kc, vc;  // loaded, to be converted
  auto turn = [&](Scores& s, Scores& next, int tile, auto more) __attribute__((always_inline)) {
    constexpr bool kMore = decltype(more)::value;
    if constexpr (kMore) scores(next, tile + 1);
    fold(s, tile);
    if constexpr (kMore) {
      store_k(kc, tile + 2);
      store_v(vc, tile + 1);
      load_k(kc, at(tile + 3));
      load_v(vc, at(tile + 2));
      settle(next, tile + 1);
      barrier();
    }
  };
  {
    Codes k0, v0, k1;  // what the first turns need, all asked for at once
    load_k(k0, t0);
    load_v(v0, t0);
    load_k(k1, at(t0 + 1));
    load_v(vc, at(t0 + 1));
    load_k(kc, at(t0 + 2));
    store_k(k0, t0);
    store_v(v0, t0);
    store_k(k1, t0 + 1);
  }
  barrier();
  scores(s0, t0);
  settle(s0, t0);
  barrier();  // the first turn writes K(t0 + 2) where the scores above read
  int tile = t0;
  for (; tile + 2 < t1; tile += 2) {
    turn(s0, s1, tile, Bool<true>());
    turn(s1, s0, tile + 1, Bool<true>());
  }
  if (tile + 1 < t1) {
    turn(s0, s1, tile, Bool<true>());
    turn(s1, s0, tile + 1, Bool<false>());
  } else {
    turn(s0, s1, tile, Bool<false>());
  }
}

}  // namespace ttcd
