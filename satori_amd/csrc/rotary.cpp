// The frequencies of rotary positions, scaled for long contexts (satori_hip_rotary_frequencies). No device code.
#include <cmath>
#include <new>
#include <string>

#include "../../include/satori_hip.h"
#include "host_shapes.hpp"

namespace satori {
namespace {

[[noreturn]] void out_of_range(const char* name) {
    fail(SATORI_HIP_E_ARGUMENT_OUT_OF_RANGE,
         std::string("Specified argument was out of the range of valid values. (Parameter '") + name + "')");
}

constexpr double kPi = 3.14159265358979323846;

double between(double low, double high, double x) { return x < low ? low : x > high ? high : x; }

void frequencies_of(int rotary, double base, int scaling, double factor, int original, double low, double high,
                    double* frequencies, double* magnitude) {
    const int pairs = rotary / 2;
    *magnitude = 1.0;
    // A base that turns the slowest pair `factor` times more slowly and leaves the fastest as it is.
    if (scaling == SATORI_HIP_SCALING_NTK) base *= std::pow(factor, rotary / (rotary - 2.0));
    for (int k = 0; k < pairs; ++k) frequencies[k] = std::pow(base, -2.0 * k / rotary);
    if (scaling == SATORI_HIP_SCALING_LINEAR)
        for (int k = 0; k < pairs; ++k) frequencies[k] /= factor;
    if (scaling == SATORI_HIP_SCALING_YARN) {
        // Pair k turns original * f_k / 2 pi times over the original positions; the pair that turns t times is
        // k = rotary ln(original / (2 pi t)) / (2 ln base). Between those of `high` and `low` turns, both rounded away from
        // each other, the frequencies go from their own to the scaled ones in proportion to k.
        const auto pair_of = [&](double turns) { return rotary * std::log(original / (2 * kPi * turns)) / (2 * std::log(base)); };
        const double from = std::fmax(0.0, std::floor(pair_of(high))), to = std::fmin(rotary - 1.0, std::ceil(pair_of(low)));
        for (int k = 0; k < pairs; ++k) {
            const double scaled = between(0.0, 1.0, (k - from) / std::fmax(0.001, to - from));
            frequencies[k] *= 1.0 - scaled + scaled / factor;
        }
        *magnitude = 1.0 + 0.1 * std::log(factor);
    }
    if (scaling == SATORI_HIP_SCALING_WAVELENGTH)
        for (int k = 0; k < pairs; ++k) {
            const double turns = original * frequencies[k] / (2 * kPi);
            const double kept = between(0.0, 1.0, (turns - low) / (high - low));
            frequencies[k] *= kept + (1.0 - kept) / factor;
        }
}

}  // namespace
}  // namespace satori

extern "C" int satori_hip_rotary_frequencies(int rotary_dimensions, double frequency_base, int scaling, double factor,
                                             int original_positions, double low, double high, double* frequencies,
                                             double* magnitude) {
    using namespace satori;
    try {
        if (!frequencies) fail(SATORI_HIP_E_ARGUMENT_NULL, "Value cannot be null. (Parameter 'frequencies')");
        if (!magnitude) fail(SATORI_HIP_E_ARGUMENT_NULL, "Value cannot be null. (Parameter 'magnitude')");
        if (rotary_dimensions <= 0 || rotary_dimensions % 2 != 0) out_of_range("rotaryDimensions");
        if (!std::isfinite(frequency_base) || frequency_base <= 0) out_of_range("frequencyBase");
        if (scaling < SATORI_HIP_SCALING_NONE || scaling > SATORI_HIP_SCALING_WAVELENGTH) out_of_range("scaling");
        if (scaling != SATORI_HIP_SCALING_NONE && !(std::isfinite(factor) && factor >= 1)) out_of_range("factor");
        if (scaling == SATORI_HIP_SCALING_NTK && rotary_dimensions == 2) out_of_range("rotaryDimensions");
        if (scaling == SATORI_HIP_SCALING_YARN || scaling == SATORI_HIP_SCALING_WAVELENGTH) {
            if (original_positions <= 0) out_of_range("originalPositions");
            if (!(std::isfinite(low) && low > 0)) out_of_range("low");
            if (!(std::isfinite(high) && high > low)) out_of_range("high");
        }
        if (scaling == SATORI_HIP_SCALING_YARN && frequency_base <= 1) out_of_range("frequencyBase");
        frequencies_of(rotary_dimensions, frequency_base, scaling, factor, original_positions, low, high, frequencies,
                       magnitude);
        record_error("");
        return SATORI_HIP_OK;
    } catch (const Failure& f) {
        record_error(f.message);
        return f.status;
    } catch (const std::bad_alloc&) {
        record_error("Out of host memory.");
        return SATORI_HIP_E_OUT_OF_MEMORY;
    } catch (...) {
        record_error("Unexpected failure.");
        return SATORI_HIP_E_DEVICE;
    }
}
