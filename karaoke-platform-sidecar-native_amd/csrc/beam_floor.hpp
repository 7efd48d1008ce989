// The floor from which a wave of beam search looks through its vectors of logits.
// Whole numbers only, so that it runs on the host as well.
#pragma once

#include <stdint.h>

namespace vh {

struct BeamFloor {
    uint32_t least;  // logits in the order of whole numbers
    int vectors;     // those that reach it
};

// with(u): how many vectors have a logit of u or more, which falls as u rises; the best
// `most` logits are all in those, as long as they are `most` or more.  lowest: a floor that
// `most` logits reach, highest: the largest logit.  The lowest floor where at most `fit`
// vectors reach it; else, by halves, one that at most `fit` and at least `most` reach; and
// where no trial was one, the lowest with its own, too many, vectors: those of a floor that
// was tried and refused are no one's.
template <typename With>
constexpr BeamFloor beam_floor(uint32_t lowest, uint32_t highest, int most, int fit, With &&with) {
    BeamFloor chosen{lowest, with(lowest)};
    uint32_t lo = lowest, hi = highest;  // at lo too many, above hi too few
    while (chosen.vectors > fit && lo < hi) {
        const uint32_t trial = lo + (hi - lo + 1) / 2;
        const int vectors = with(trial);
        if (vectors < most) {
            hi = trial - 1;
        } else {
            lo = trial;
            if (vectors <= fit) chosen = {trial, vectors};
        }
    }
    return chosen;
}

}  // namespace vh
