// Host-side check of the ring of bulk copies that the 4-bit cache's attention kernels count with (test infrastructure,
// built and run by tests/test_cpu_kv4_ring.py; no GPU). For rings of 2 to 4 stages, every number of places up to 40 and
// every copy `late` that may fail to land in time (or none), a block's loop is played:
//  - a place's stage holds the place's own copy, and a stage is not refilled before its place was passed;
//  - all places are passed whatever happens;
//  - with a late copy, that wait runs out, and nothing is issued or awaited after it but,
//    at the end, the last copy of each stage;
//  - every copy issued was either seen to land or waited for again.
// `told`: the wait that ran out was another's, and this block's loop learns of it at place `late`, whose copy and
// those after it may be in flight still: none of them is taken for landed.
// Prints "ok <cases>" or the first violation.
#include <cstdint>
#include <cstdio>

#include "../../voxgen_b200/csrc/kv4_rows_attention.cuh"

template <uint32_t kStages>
const char *play(uint32_t places, uint32_t late, bool told) {
  vg::CopyRing<kStages> ring;
  uint32_t holds[kStages], phase[kStages] = {}, next = 0, ran_out = 0, waits = 0;
  const char *fault = nullptr;
  const auto fetch = [&] {
    if (next < places)
      ring.fetch([&](uint32_t stage) {
        if (next >= kStages && ring.passed <= next - kStages) fault = "a stage refilled before its place was passed";
        holds[stage] = next++;
      });
  };
  for (uint32_t i = 0; i < kStages; ++i) fetch();
  for (uint32_t i = 0; i < places; ++i) {
    if (told && i == late) ring.stopped = 1;
    ring.take([&](uint32_t stage, uint32_t parity) {
      ++waits;
      if (holds[stage] != i) fault = "a wait for another place's copy";
      if ((phase[stage] & 1) != parity) fault = "a wait for another phase";
      ++phase[stage];
      ran_out += i == late;
      return i != late;
    });
    fetch();
  }
  if (ring.passed != places) fault = "places left";
  if (ran_out > 1 || waits > (late < places ? late + 1 : places)) fault = "waits after one ran out";
  const uint32_t landed = late < places ? late : places;   // seen to land, in order
  uint32_t first = ring.issued, again = 0;
  if (ring.issued < landed || ring.issued - landed > kStages) fault = "copies issued after a wait ran out";
  ring.drain([&](uint32_t stage, uint32_t parity) {
    // the one copy of the last kStages in this stage and phase
    for (uint32_t i = ring.issued > kStages ? ring.issued - kStages : 0; i < ring.issued; ++i)
      if (i % kStages == stage && (i / kStages & 1) == parity && holds[stage] == i) {
        first = i < first ? i : first;
        ++again;
      }
  });
  if (first > landed || again != ring.issued - first) fault = "a copy left in flight";
  return fault;
}

int main() {
  unsigned long cases = 0;
  for (uint32_t places = 0; places <= 40; ++places)
    for (uint32_t late = 0; late <= places; ++late) {   // late == places: none
      for (const char *fault : {play<2>(places, late, false), play<3>(places, late, false), play<4>(places, late, false),
                                play<2>(places, late, true), play<3>(places, late, true), play<4>(places, late, true)}) {
        ++cases;
        if (fault) {
          printf("%s: %u places, late %u\n", fault, places, late);
          return 1;
        }
      }
    }
  printf("ok %lu\n", cases);
}
