// The order in which attention_prompt.hip's waves store tiles into LDS, read them and meet, in units
// of 32 tokens (halves of a tile). Plain C++, so that it can be checked without a GPU.
//
// Step t takes the halves 0 .. halves-1 of tile t, one after the other. Its first half stores, for
// all waves, the keys of tile t + kKeysStaged and the values of tile t + kValuesStaged; each half
// reads the operands of a later one; one half ends with the barrier. Between two barriers waves are
// anywhere, so a store and a read of one buffer need a barrier between them, in either order.
#pragma once

namespace ci8 {

constexpr int kKeyBuffers = 3, kValueBuffers = 2;
constexpr int kPoisonBuffers = 3;  // which values were NaN, stored with the values
constexpr int kKeysStaged = 2, kValuesStaged = 1;

// How many halves before their use operands are read. Tiles of one half (256 channels) read them
// where they are used: the keys in the step before, for the scores of the next tile.
constexpr int keys_ahead(int halves) { return halves > 1 ? 2 : 1; }
constexpr int values_ahead(int halves) { return halves > 1 ? 1 : 0; }

// The half that ends with the barrier: the last one that reads the values of its own tile. By then the
// keys of the tile have been read too, and what this step stored is read after it.
constexpr int barrier_half(int halves) {
  const int last = halves - 1 - values_ahead(halves);
  return last > 0 ? last : 0;
}

// Whether a barrier at the end of half `barrier` of each step parts every read from the stores before
// and after it. Tile u is stored in the first half of step u - staged, its half h is read `ahead`
// halves before half h of step u, and its buffer is stored again `buffers` tiles later.
constexpr bool reads_are_parted(int halves, int barrier, int buffers, int staged, int ahead) {
  const int u = buffers + staged + ahead;  // any tile: times below are not negative
  auto between = [&](int first, int second) {  // a barrier at the end of `first` or later, before `second`
    for (int at = first; at < second; ++at)
      if (at % halves == barrier) return true;
    return false;
  };
  for (int h = 0; h < halves; ++h) {
    const int stored = (u - staged) * halves, read = u * halves + h - ahead;
    if (!between(stored, read) || !between(read, stored + buffers * halves)) return false;
  }
  return true;
}

// Of keys, values, and the NaN marks that the last half of a step reads.
constexpr bool schedule_holds(int halves, int barrier) {
  return reads_are_parted(halves, barrier, kKeyBuffers, kKeysStaged, keys_ahead(halves)) &&
         reads_are_parted(halves, barrier, kValueBuffers, kValuesStaged, values_ahead(halves)) &&
         reads_are_parted(halves, barrier, kPoisonBuffers, kValuesStaged, 0);
}

}  // namespace ci8
