// Frequencies of the rotary positions in radians per position, and the magnitude of the rotated values (pocket_tts_amd.h).  Host
// only; the library and its Python binding each compile it, so that the frequencies can be had before the library, and with it a
// HIP runtime, is loaded.
#pragma once

#include <algorithm>
#include <cmath>
#include <stdexcept>

namespace ptts {

// Position interpolation (1), the stretched base (2) and the blend by parts (3: ramp over the number of turns that a frequency makes
// within the trained length, magnitude 0.1 ln factor + 1).
inline void rotary_frequencies(int rot_dim, double base, int scaling, double factor, double trained, double fast, double slow, double* out,
                               float* magnitude) {
    if (!out || rot_dim < 2 || rot_dim % 2) throw std::runtime_error("rot_dim must be even and at least 2");
    if (!(base > 1.0) || !std::isfinite(base)) throw std::runtime_error("base must be finite and above 1");
    if (scaling < 0 || scaling > 3) throw std::runtime_error("scaling must be 0 to 3");
    if (scaling != 0 && (!(factor >= 1.0) || !std::isfinite(factor))) throw std::runtime_error("factor must be finite and at least 1");
    if (scaling == 3 && (!(trained > 0.0) || !std::isfinite(trained) || !(slow > 0.0) || !(fast > slow) || !std::isfinite(fast)))
        throw std::runtime_error("by parts needs trained > 0 and fast > slow > 0");
    const int half = rot_dim / 2;
    // base^(2 (half - 1) / rot_dim) grows by `factor`: the lowest frequency is divided by it exactly
    if (scaling == 2 && half > 1) base *= std::pow(factor, rot_dim / static_cast<double>(rot_dim - 2));
    for (int i = 0; i < half; ++i) {
        double f = std::pow(base, -2.0 * i / rot_dim);
        if (scaling == 1) f /= factor;
        if (scaling == 3) {
            const double turns = trained * f / 6.283185307179586477;
            const double keep = std::min(1.0, std::max(0.0, (turns - slow) / (fast - slow)));
            f = f * keep + f / factor * (1.0 - keep);
        }
        out[i] = f;
    }
    if (magnitude) *magnitude = scaling == 3 ? static_cast<float>(0.1 * std::log(factor) + 1.0) : 1.0f;
}

}  // namespace ptts
