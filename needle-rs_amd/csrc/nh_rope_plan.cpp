// The C ABI of rotary positions (include/needle_hip.h): plans and the call.
#include <math.h>

#include <memory>
#include <new>
#include <string>
#include <vector>

#include "../../include/needle_hip.h"
#include "nh_kv_host.h"
#include "nh_rope.h"

using nh::kv::fail;

extern "C" {

int nh_rope_freqs(int dim, double theta, int scaling, double factor, double original, double low, double high,
                  double* freqs, double* amplitude) {
    if (!freqs || !amplitude) return fail(NH_EINVAL, "null argument");
    if (dim < 2 || dim > 256 || dim % 2) return fail(NH_EINVAL, "2 to 256 dims of a head turn, in pairs");
    if (!(theta > 1.0 && theta < 1e300)) return fail(NH_EINVAL, "theta is above 1");
    if (scaling < NH_ROPE_PLAIN || scaling > NH_ROPE_BANDS) return fail(NH_EINVAL, "no such scaling");
    const bool ranged = scaling == NH_ROPE_PARTS || scaling == NH_ROPE_BANDS;
    if (scaling != NH_ROPE_PLAIN && !(factor >= 1.0 && factor < 1e9)) return fail(NH_EINVAL, "a context is stretched by 1 and more");
    if (ranged && !(original >= 1.0 && original < 1e12)) return fail(NH_EINVAL, "the original length is 1 and more positions");
    if (ranged && !(low > 0.0 && high > low && high < 1e12)) return fail(NH_EINVAL, "turns: 0 < low < high");
    const double two_pi = 6.283185307179586476925;
    if (scaling == NH_ROPE_BASE && dim > 2) theta *= pow(factor, dim / (dim - 2.0));
    double at_high = 0.0, at_low = 0.0;
    if (scaling == NH_ROPE_PARTS) {
        // the (fractional) indices of the pairs that turn `high` and `low` times in the original length
        at_high = fmax(floor(dim * log(original / (high * two_pi)) / (2.0 * log(theta))), 0.0);
        at_low = fmin(ceil(dim * log(original / (low * two_pi)) / (2.0 * log(theta))), dim - 1.0);
    }
    for (int i = 0; i < dim / 2; ++i) {
        const double f = pow(theta, -2.0 * i / dim);
        double keep = 1.0;
        if (scaling == NH_ROPE_LINEAR) keep = 0.0;
        if (scaling == NH_ROPE_BANDS) keep = (original * f / two_pi - low) / (high - low);
        if (scaling == NH_ROPE_PARTS) keep = 1.0 - (i - at_high) / fmax(at_low - at_high, 0.001);
        keep = fmin(fmax(keep, 0.0), 1.0);
        freqs[i] = scaling == NH_ROPE_BASE ? f : f * keep + (keep < 1.0 ? f / factor * (1.0 - keep) : 0.0);
    }
    *amplitude = scaling == NH_ROPE_PARTS ? 0.1 * log(factor) + 1.0 : 1.0;
    return NH_OK;
}

int nh_rope_new(const double* freqs, int pairs, double amplitude, int layout, nh_rope** out) {
    if (!out) return fail(NH_EINVAL, "null argument");
    *out = nullptr;
    if (pairs < 1 || pairs > 128) return fail(NH_EINVAL, "1 to 128 pairs of dims");
    if (!freqs) return fail(NH_EINVAL, "null argument");
    if (layout != NH_ROPE_HALF && layout != NH_ROPE_INTERLEAVED) return fail(NH_EINVAL, "no such layout");
    if (!(fabs(amplitude) <= 1e30)) return fail(NH_EINVAL, "the amplitude is not finite");
    for (int i = 0; i < pairs; ++i)
        if (!(fabs(freqs[i]) <= 1e6)) return fail(NH_EINVAL, "a frequency is at most 10^6 radians a position");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    return nh::kv::guarded([&]() -> int {
        // Turns modulo 1 as fractions of 2^64, in 80 bits (x87): 2^-64 of a turn.
        std::vector<uint64_t> turns(pairs);
        for (int i = 0; i < pairs; ++i) {
            long double t = (long double)freqs[i] / 6.283185307179586476925286766559005768L;
            t -= floorl(t);
            const long double scaled = roundl(ldexpl(t, 64));
            turns[i] = scaled >= 18446744073709551616.0L ? 0 : (uint64_t)scaled;
        }
        auto r = std::make_unique<nh_rope>();
        NH_TRY(hipGetDevice(&r->device), "hipGetDevice");
        hipError_t e = hipMalloc(&r->turns, pairs * sizeof(uint64_t));
        if (e == hipSuccess) e = hipMemcpy(r->turns, turns.data(), pairs * sizeof(uint64_t), hipMemcpyHostToDevice);
        if (e != hipSuccess) {
            if (r->turns) hipFree(r->turns);
            (void)hipGetLastError();  // an allocation that failed is this call's error alone
            return fail(NH_ENOMEM, std::string("rope allocation: ") + hipGetErrorString(e));
        }
        r->v.turns = r->turns;
        r->v.amplitude = amplitude;
        r->v.pairs = pairs;
        r->v.interleaved = layout == NH_ROPE_INTERLEAVED;
        *out = r.release();
        return NH_OK;
    });
}

int nh_rope_free(nh_rope* r) {
    if (!r) return NH_OK;
    // (also while this thread captures a graph of other work, as a cache's release)
    hipStreamCaptureMode mode = hipStreamCaptureModeRelaxed;
    const bool relaxed = hipThreadExchangeStreamCaptureMode(&mode) == hipSuccess;
    if (r->turns) hipFree(r->turns);
    if (relaxed) hipThreadExchangeStreamCaptureMode(&mode);
    delete r;
    return NH_OK;
}

int nh_rope_apply(const nh_rope* r, const int32_t* pos, int64_t rows, int dim, const void* q, int64_t ldq, int heads,
                  void* q_out, int64_t ldqo, const void* k, int64_t ldk, int kv_heads, void* k_out, int64_t ldko, int type,
                  int transposed, void* stream) {
    if (!r) return fail(NH_EINVAL, "null plan");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    int dev = -1;
    NH_TRY(hipGetDevice(&dev), "hipGetDevice");
    if (dev != r->device) return fail(NH_EINVAL, "the plan belongs to another device than the current one");
    if (!nh::kv::known_type(type)) return fail(NH_EINVAL, "no such type");
    if (rows < 0 || rows > INT32_MAX) return fail(NH_EINVAL, "0 to 2^31 - 1 rows");
    if (heads < 0 || kv_heads < 0 || heads > (1 << 20) || kv_heads > (1 << 20)) return fail(NH_EINVAL, "0 to 2^20 heads");
    if (dim < 2 * r->v.pairs || dim > (1 << 20)) return fail(NH_EINVAL, "a head holds the plan's pairs, and at most 2^20 dims");
    if (rows == 0 || heads + kv_heads == 0) return NH_OK;
    if (!pos || (heads && (!q || !q_out)) || (kv_heads && (!k || !k_out))) return fail(NH_EINVAL, "null argument");
    const int64_t wq = (int64_t)heads * dim, wk = (int64_t)kv_heads * dim;
    if (ldq < wq || ldqo < wq || ldk < wk || ldko < wk) return fail(NH_EINVAL, "rows overlap: a row holds every head");
    if ((heads && q == q_out && ldq != ldqo) || (kv_heads && k == k_out && ldk != ldko))
        return fail(NH_EINVAL, "rows turned in place stay where they are");
    nh::RopeArgs a{r->v, pos, {q, q_out, ldq, ldqo, heads}, {k, k_out, ldk, ldko, kv_heads}, rows, dim, transposed != 0};
    NH_TRY(nh::launch_rope(a, type, (hipStream_t)stream), "rope");
    return NH_OK;
}

}  // extern "C"
