// A wave's choice of a floor in beam search, and the places of the vectors that reach it, on the host.
#include "../karaoke-platform-sidecar-native_amd/csrc/beam_floor.hpp"

// tops: the vectors' largest logits in the order of whole numbers, [vectors of a lane][64 lanes].
// least and count: the floor and how many reach it; the highest place that one of them is put at, -1: none is put.
extern "C" int beam_floor_host(const uint32_t *tops, int lane_vectors, uint32_t lowest, uint32_t highest, int most, int fit,
                               uint32_t *least, int *count) {
    const auto with = [&](uint32_t floor) {
        int n = 0;
        for (int i = 0; i < 64 * lane_vectors; i++) n += tops[i] >= floor;
        return n;
    };
    const vh::BeamFloor chosen = vh::beam_floor(lowest, highest, most, fit, with);
    *least = chosen.least;
    *count = chosen.vectors;
    return chosen.vectors <= fit ? with(chosen.least) - 1 : -1;
}
