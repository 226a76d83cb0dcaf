// How the keys that the waves of a workgroup collected, each in a room of its own,
// are put together. Plain C++: a test on the host walks every place that it gives.
#pragma once

namespace nnops_amd {

// Wave w counted count[w] keys and stored the first `room` of them. Where each wave's
// keys go among all, and how many there are: kWaves * room at most, so that no place
// lies behind that. -1 where a wave counted more than its room holds: then nothing is
// to be moved, the keys are not all there.
template <int kWaves>
constexpr int gather_rooms(const int (&count)[kWaves], int room, int (&to)[kWaves])
{
    int keys = 0, most = 0;
    for (int w = 0; w < kWaves; ++w) {
        to[w] = keys;
        most = count[w] > most ? count[w] : most;
        keys += count[w];
    }
    return most > room ? -1 : keys;
}

}  // namespace nnops_amd
