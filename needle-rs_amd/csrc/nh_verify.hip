// Verification of drafted tokens against the target's logits
// (nh_verify_drafts in include/needle_hip.h).
//
//   p = softmax(l / T); draft x_i is kept while u_i q(x_i) < p_i(x_i), in
//   turn; the token after the last kept one is drawn from max(p - q, 0) where
//   a draft was refused (from p without it for drafts without probabilities),
//   else from p, at the uniform u_n: the first t with w_0 + .. + w_t > u_n W.
//
// Two launches.  k_verify_rows reads every logit once, a workgroup a slice of
// a row, and leaves the slice's maximum and sum of weights: bound by the read
// (50 MB of bf16 logits, 192 rows of 131,072: 15 us, 3.3 TB/s; a workgroup a row
// took 358).  k_verify_pick joins the slices of a
// sequence's rows, checks its drafts and walks to the slice, then the token,
// that the uniform falls on.  With probabilities the one row that is drawn from
// is weighed slice by slice first, a workgroup each; the last to finish picks: 21
// us for 32 sequences of 131,072 tokens, three round trips to memory one after
// the other (slices, weighed slice, picked slice) around 64-bit series.  Without
// them 7.5 us (one sequence of 8,192 tokens), greedy 3.4.
//
// A draw next to a border must not depend on how a sum was split: the weights
// of the row that is drawn from, and every sum of more than a few terms, are in
// f64; the slices' sums (of f32 weights, each good to an f32 rounding) are too.
#include <math.h>

#include <algorithm>

#include "../../include/needle_hip.h"
#include "nh_kv4_device.h"

namespace nh {

constexpr int VR_THREADS = 256;
constexpr int VR_EACH = 16;                        // logits of a thread
constexpr int VR_SLICE = VR_THREADS * VR_EACH;     // of a workgroup
constexpr int VR_WAVES = VR_THREADS / 64;
// The picking kernel takes a slice 4 neighbours a thread: by 1024 threads where
// one workgroup does a sequence and waits for each step; by 256 four times
// where many weigh slices, so that all of them are resident (32 sequences of
// 131,072 tokens are 1024 workgroups).
constexpr int VP_EACH = 4;

struct VerifySlice {
    double sum;  // of the weights against the slice's maximum
    float max;
    int best;    // the first index of the maximum (greedy), -1: only NaN
};

struct VerifyArgs {
    const void* logits;
    const int* drafts;
    const int* counts;   // or null: n each
    const void* probs;   // or null
    const float* u;
    int* accepted;
    int* tokens;
    VerifySlice* slices; // [rows][slices]
    double* rest;        // [batch][slices]: sums of what the drafts left
    int* arrived;        // [batch]
    int64_t ldl, ldp;
    int batch, n, vocab, nslices;
    int aligned, paligned;  // rows of logits and of probs start at 16-byte borders
    double c;            // log2(e) / T; 0: greedy
};

// The weights of logits l beside the largest, m, in 64 bits (NaN weighs
// nothing): 2^y, y = (l - m) log2(e) / T, by y = n + f, |f| <= 1/2, and the
// exponential series of f ln 2 up to the 11th power (the rest is below 2^-47 of
// it).  The N series run in step, so their code is one copy of the constants.
template <int N>
__device__ __forceinline__ void verify_weights(const float* l, float m, double c, double* w) {
    constexpr double L = 0.69314718055994530942;
    constexpr double K[12] = {1.0, L, L * L / 2, L * L * L / 6, L * L * L * L / 24, L * L * L * L * L / 120,
                              L * L * L * L * L * L / 720, L * L * L * L * L * L * L / 5040,
                              L * L * L * L * L * L * L * L / 40320, L * L * L * L * L * L * L * L * L / 362880,
                              L * L * L * L * L * L * L * L * L * L / 3628800,
                              L * L * L * L * L * L * L * L * L * L * L / 39916800};
    double f[N];
    int n[N];
#pragma unroll
    for (int k = 0; k < N; ++k) {
        const double y = fmax(((double)l[k] - (double)m) * c, -2000.0), r = rint(y);
        f[k] = y - r;
        n[k] = (int)r;
        w[k] = K[11];
    }
#pragma unroll
    for (int i = 10; i >= 0; --i)
#pragma unroll
        for (int k = 0; k < N; ++k) w[k] = __builtin_fma(w[k], f[k], K[i]);
#pragma unroll
    for (int k = 0; k < N; ++k) w[k] = l[k] == m ? 1.0 : l[k] < m ? __builtin_amdgcn_ldexp(w[k], n[k]) : 0.0;
}
__device__ __forceinline__ double verify_weight(float l, float m, double c) {
    double w;
    verify_weights<1>(&l, m, c, &w);
    return w;
}

// (value, index) of the first maximum of two; index -1: none yet.
__device__ __forceinline__ void verify_best(float& v, int& i, float w, int j) {
    if (j >= 0 && (i < 0 || w > v || (w == v && j < i))) v = w, i = j;
}

// v moved by a DPP control; lanes without a source, and rows outside the mask, get 0.
template <int CTRL, int ROWS>
__device__ __forceinline__ double dpp_f64(double v) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)x, CTRL, ROWS, 0xF, true);
    const uint32_t hi = __builtin_amdgcn_update_dpp(0, (int)(uint32_t)(x >> 32), CTRL, ROWS, 0xF, true);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
// Sum over the lanes up to and with this one: row shifts by 1, 2, 4, 8, then
// the rows' last lanes to the rows after them (no LDS round trips).
__device__ __forceinline__ double wave_scan(double v) {
    v += dpp_f64<0x111, 0xF>(v);
    v += dpp_f64<0x112, 0xF>(v);
    v += dpp_f64<0x114, 0xF>(v);
    v += dpp_f64<0x118, 0xF>(v);
    v += dpp_f64<0x142, 0xA>(v);
    v += dpp_f64<0x143, 0xC>(v);
    return v;
}
__device__ __forceinline__ double lane_f64(double v, int lane) {
    const uint64_t x = __builtin_bit_cast(uint64_t, v);
    const uint32_t lo = __builtin_amdgcn_readlane((int)(uint32_t)x, lane);
    const uint32_t hi = __builtin_amdgcn_readlane((int)(uint32_t)(x >> 32), lane);
    return __builtin_bit_cast(double, (uint64_t)hi << 32 | lo);
}
__device__ __forceinline__ double wave_sum(double v) { return lane_f64(wave_scan(v), 63); }

// A slice of a row of logits.  The weights are f32 with the rounding of their
// argument carried (x / T log2 e as two f32 numbers, for f32 logits also what
// l - max rounds off), so each is off by its own last rounding alone and a sum
// of many by far less; 16 a thread are summed in f32, the rest in f64.
template <int LT, bool GREEDY>
__global__ __launch_bounds__(VR_THREADS) void k_verify_rows(VerifyArgs a) {
    typedef typename Kv4Elem<LT>::T T;
    constexpr int VEC = 16 / sizeof(T);
    typedef T Vec __attribute__((ext_vector_type(VEC)));
    __shared__ float sv[VR_WAVES];
    __shared__ int si[VR_WAVES];
    __shared__ double ss[VR_WAVES];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const int slice = blockIdx.x % a.nslices;
    const int64_t row = blockIdx.x / a.nslices;
    const int t0 = slice * VR_SLICE;
    const T* x = reinterpret_cast<const T*>(a.logits) + row * a.ldl + t0;
    const int n = min(VR_SLICE, a.vocab - t0);
    if (slice == 0 && tid == 0 && row % (a.n + 1) == 0) a.arrived[row / (a.n + 1)] = 0;
    // Logit k of a thread: VEC neighbours, then the workgroup's next ones.
    float v[VR_EACH];
#pragma unroll
    for (int k = 0; k < VR_EACH; k += VEC) {
        const int t = (k / VEC * VR_THREADS + tid) * VEC;
        if (a.aligned && t + VEC <= n) {
            const Vec y = *reinterpret_cast<const Vec*>(x + t);
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k + e] = (float)y[e];
        } else {
#pragma unroll
            for (int e = 0; e < VEC; ++e) v[k + e] = t + e < n ? Kv4Elem<LT>::get(x + t + e) : __builtin_nanf("");
        }
    }
    VerifySlice* to = a.slices + row * a.nslices + slice;
    if constexpr (GREEDY) {
        float best = 0.0f;
        int at = -1;
#pragma unroll
        for (int k = 0; k < VR_EACH; ++k)
            if (v[k] == v[k]) verify_best(best, at, v[k], (k / VEC * VR_THREADS + tid) * VEC + k % VEC);
#pragma unroll
        for (int h = 1; h < 64; h <<= 1) {
            const float w = lane_xor(best, h, lane);
            const int j = __float_as_int(lane_xor(__int_as_float(at), h, lane));
            verify_best(best, at, w, j);
        }
        if (lane == 0) sv[wave] = best, si[wave] = at;
        __syncthreads();
        if (tid == 0) {
            for (int w = 1; w < VR_WAVES; ++w) verify_best(best, at, sv[w], si[w]);
            to->max = best;
            to->best = at < 0 ? -1 : at + t0;
        }
    } else {
        float m = -__builtin_inff();
#pragma unroll
        for (int k = 0; k < VR_EACH; ++k) m = fmaxf(m, v[k]);
#pragma unroll
        for (int h = 1; h < 64; h <<= 1) m = fmaxf(m, lane_xor(m, h, lane));
        if (lane == 0) sv[wave] = m;
        __syncthreads();
#pragma unroll
        for (int w = 0; w < VR_WAVES; ++w) m = fmaxf(m, sv[w]);
        // (a temperature below 2^-127 has a factor past f32: held at its end, so that the maximum's 0 times it is 0)
        constexpr float END = 3.402823466e38f;
        const float ch = a.c < (double)END ? (float)a.c : END, cl = ch < END ? (float)(a.c - (double)ch) : 0.0f;
        float sum = 0.0f;
#pragma unroll
        for (int k = 0; k < VR_EACH; ++k) {
            const float l = v[k], d = l - m;
            const float t = d * ch;
            float r = __builtin_fmaf(d, cl, __builtin_fmaf(d, ch, -t));
            if constexpr (LT == KV4_F32) {
                const float b = d - l;
                r = __builtin_fmaf((l - (d - b)) - (m + b), ch, r);
            }
            const float e = __builtin_amdgcn_exp2f(t);
            const float w = __builtin_fmaf(e, r * 0.69314718055994530942f, e);
            // (not for NaN, infinite arguments, or weights below 2^-126)
            sum += t > -126.0f ? w : 0.0f;
        }
        if (fabsf(m) == __builtin_inff()) {
            // Infinite logits share the whole; a slice of -inf and NaN has none.
            sum = 0.0f;
#pragma unroll
            for (int k = 0; k < VR_EACH; ++k) sum += m > 0.0f && v[k] == m ? 1.0f : 0.0f;
        }
        const double s = wave_sum((double)sum);
        if (lane == 0) ss[wave] = s;
        __syncthreads();
        if (tid == 0) {
            to->sum = (ss[0] + ss[1]) + (ss[2] + ss[3]);
            to->max = m;
            to->best = 0;
        }
    }
}

// A sequence's drafts and its next token.  With RESIDUE (sampling, with the
// drafter's probabilities) nslices workgroups a sequence weigh a slice each of
// the row to be drawn from; else one.
template <int LT, int PT, bool GREEDY, bool RESIDUE>
__global__ __launch_bounds__(RESIDUE ? 256 : 1024) void k_verify_pick(VerifyArgs a) {
    constexpr int VP_THREADS = RESIDUE ? 256 : 1024, VP_WAVES = VP_THREADS / 64;
    constexpr int SUB = VR_SLICE / (VP_THREADS * VP_EACH);  // strips of a slice
    typedef typename Kv4Elem<LT>::T T;
    typedef typename Kv4Elem<PT>::T P;
    __shared__ double s_sum, ss[2][VP_WAVES];
    __shared__ float s_max;
    __shared__ int s_kept, s_best, s_slice, s_pick, s_last, s_left, s_out;
    __shared__ double s_goal, s_part[64];
    const int tid = threadIdx.x, lane = tid & 63, wave = tid >> 6, n = a.n;
    const int b = RESIDUE ? blockIdx.x / a.nslices : blockIdx.x, mine = RESIDUE ? blockIdx.x % a.nslices : 0;
    const int64_t row0 = (int64_t)b * (n + 1);
    const T* logits = reinterpret_cast<const T*>(a.logits) + row0 * a.ldl;
    const P* probs = reinterpret_cast<const P*>(a.probs) + (int64_t)b * n * a.ldp;
    const int* drafts = a.drafts + (int64_t)b * n;
    const float* u = a.u + row0;
    const int cnt = a.counts ? min(max(a.counts[b], 0), n) : n;

    // A row a wavefront: the slices joined, the draft checked.
    if (tid == 0) s_kept = cnt;
    for (int i0 = 0; i0 <= cnt; i0 += VP_WAVES) {
        const int i = i0 + wave;
        __syncthreads();
        if (s_kept < i0) break;  // (the same in every thread: written before the barrier)
        double sum = 0.0, part = 0.0;  // part: of slice `lane`
        float m = -__builtin_inff();
        int best = -1, draft = 0;
        bool ok = true;
        if (i <= cnt) {
            const VerifySlice* sl = a.slices + (row0 + i) * a.nslices;
            // Every load that does not wait for another is issued first: the slices, the
            // uniform, the draft; then what the draft names.
            float ml = -__builtin_inff();
            double sl0 = 0.0;
            if (!GREEDY && lane < a.nslices) ml = sl[lane].max, sl0 = sl[lane].sum;
            const float ui = GREEDY ? 0.0f : u[i];
            const float first = GREEDY ? Kv4Elem<LT>::get(logits + i * a.ldl) : 0.0f;
            const int x = i < cnt ? drafts[i] : 0;
            const bool in = (unsigned)x < (unsigned)a.vocab;
            const float lx = !GREEDY && in ? Kv4Elem<LT>::get(logits + i * a.ldl + x) : 0.0f;
            const double q = RESIDUE && in && i < cnt ? (double)Kv4Elem<PT>::get(probs + i * a.ldp + x) : 1.0;
            draft = x;
            if constexpr (GREEDY) {
                for (int k = lane; k < a.nslices; k += 64) verify_best(m, best, sl[k].max, sl[k].best);
#pragma unroll
                for (int h = 1; h < 64; h <<= 1) {
                    const float w = lane_xor(m, h, lane);
                    const int j = __float_as_int(lane_xor(__int_as_float(best), h, lane));
                    verify_best(m, best, w, j);
                }
                if (first != first || best < 0) best = 0;  // as nh_argmax has it
                ok = in && x == best;
            } else {
                m = ml;
                for (int k = lane + 64; k < a.nslices; k += 64) m = fmaxf(m, sl[k].max);
#pragma unroll
                for (int h = 1; h < 64; h <<= 1) m = fmaxf(m, lane_xor(m, h, lane));
                // (the draft's own weight in the same series)
                const float l2[2] = {ml, lx};
                double w2[2];
                verify_weights<2>(l2, m, a.c, w2);
                part = sl0 * w2[0];
                sum = part;
#pragma unroll 1
                for (int k = lane + 64; k < a.nslices; k += 64) sum += sl[k].sum * verify_weight(sl[k].max, m, a.c);
                sum = wave_sum(sum);
                ok = in && sum > 0.0 && (double)ui * q * sum < w2[1];
            }
            if (i < cnt && !ok && lane == 0) atomicMin(&s_kept, i);
        }
        __syncthreads();
        if (i == s_kept) {
            s_part[lane] = part;
            if (lane == 0) s_sum = sum, s_max = m, s_best = best, s_out = draft;
        }
    }
    __syncthreads();
    const int kept = s_kept;
    int pick = GREEDY ? s_best : 0;
    if constexpr (!GREEDY) {
        const double sum = s_sum, scale = sum > 0.0 ? 1.0 / sum : 0.0;
        const float m = s_max;
        const T* x = logits + kept * a.ldl;
        const bool refused = kept < cnt;
        const P* q = probs + (refused ? kept : 0) * a.ldp;
        const int out = refused && !RESIDUE ? s_out : -1;
        const float un = u[n];
        const VerifySlice* sl = a.slices + (row0 + kept) * a.nslices;
        // A thread's neighbours t .. t + VP_EACH - 1: the logits, and what the drafter gave them; then their weights.
        auto fetch = [&](int t, bool left, float* l, float* d) {
            typedef T VecT __attribute__((ext_vector_type(VP_EACH)));
            typedef P VecP __attribute__((ext_vector_type(VP_EACH)));
            const bool whole = t + VP_EACH <= a.vocab;
            if (whole && a.aligned) {
                const VecT y = *reinterpret_cast<const VecT*>(x + t);
#pragma unroll
                for (int k = 0; k < VP_EACH; ++k) l[k] = (float)y[k];
            } else {
#pragma unroll
                for (int k = 0; k < VP_EACH; ++k) l[k] = t + k < a.vocab ? Kv4Elem<LT>::get(x + t + k) : __builtin_nanf("");
            }
            if (RESIDUE && left) {
                if (whole && a.paligned) {
                    const VecP y = *reinterpret_cast<const VecP*>(q + t);
#pragma unroll
                    for (int k = 0; k < VP_EACH; ++k) d[k] = (float)y[k];
                } else {
#pragma unroll
                    for (int k = 0; k < VP_EACH; ++k) d[k] = t + k < a.vocab ? Kv4Elem<PT>::get(q + t + k) : 0.0f;
                }
            }
        };
        auto weigh = [&](int t, bool left, const float* l, const float* d, double* w) {
            double s = 0.0;
            verify_weights<VP_EACH>(l, m, a.c, w);
#pragma unroll
            for (int k = 0; k < VP_EACH; ++k) {
                w[k] *= scale;
                if (left && RESIDUE) {
                    const double rest = w[k] - (double)d[k];
                    w[k] = rest > 0.0 ? rest : 0.0;
                }
                if (left && !RESIDUE && t + k == out) w[k] = 0.0;
                s += w[k];
            }
            return s;
        };
        // A slice's weights, and their sum over the workgroup in wavefront order.
        auto weigh_slice = [&](int k, bool left) {
            // (every strip's loads are issued first)
            float l[SUB][VP_EACH], d[SUB][VP_EACH];
            double s = 0.0, w[VP_EACH];
            const int t = k * VR_SLICE + tid * VP_EACH;
#pragma unroll
            for (int y = 0; y < SUB; ++y) fetch(t + y * VP_THREADS * VP_EACH, left, l[y], d[y]);
#pragma unroll
            for (int y = 0; y < SUB; ++y) s += weigh(t + y * VP_THREADS * VP_EACH, left, l[y], d[y], w);
            s = wave_sum(s);
            __syncthreads();
            if (lane == 0) ss[0][wave] = s;
            __syncthreads();
            s = 0.0;
#pragma unroll
            for (int x = 0; x < VP_WAVES; ++x) s += ss[0][x];
            return s;
        };
        if constexpr (RESIDUE) {
            const double s = refused && sum > 0.0 ? weigh_slice(mine, true) : 0.0;
            if (tid == 0) {
                // The sums are stored and read as device-wide atomics, so no cache has to be
                // written back or dropped: the store has reached memory before the count goes up.
                __hip_atomic_store(a.rest + (int64_t)b * a.nslices + mine, s, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                asm volatile("s_waitcnt vmcnt(0)" ::: "memory");
                s_last = __hip_atomic_fetch_add(a.arrived + b, 1, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT) == a.nslices - 1;
            }
            __syncthreads();
            if (!s_last) return;
        }
        if (sum > 0.0) {
            bool left = refused;  // draw from what the draft left, from all of p if that is nothing
            double out_slice = 0.0;
            if (!RESIDUE && left) {
                // The refused token's slice without it, summed anew: a difference would lose what is small beside it.
                out_slice = weigh_slice(out >= 0 && out < a.vocab ? out / VR_SLICE : 0, true);
            }
            if (wave == 0) {
                auto slice_sum = [&](int k) -> double {
                    if (k >= a.nslices) return 0.0;
                    if (RESIDUE && left)
                        return __hip_atomic_load(a.rest + (int64_t)b * a.nslices + k, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
                    if (!RESIDUE && left && out >= 0 && out < a.vocab && k == out / VR_SLICE) return out_slice;
                    return (k < 64 ? s_part[k] : sl[k].sum * verify_weight(sl[k].max, m, a.c)) * scale;
                };
                // The whole; then the first slice whose cumulative sum passes the
                // goal, else the last that weighs anything.
                double goal = 0.0, at_before = 0.0;
                int at = -1;
                bool seek = false;
                double mine0 = slice_sum(lane);
#pragma unroll 1
                for (;;) {
                    double before = 0.0;
                    bool found = false;
#pragma unroll 1
                    for (int k0 = 0; k0 < a.nslices && !found; k0 += 64) {
                        const double s = k0 ? slice_sum(k0 + lane) : mine0, c = before + wave_scan(s);
                        before = lane_f64(c, 63);
                        if (!seek) continue;
                        const uint64_t some = __ballot(s > 0.0), over = __ballot(s > 0.0 && c > goal);
                        const int l = over ? __builtin_ctzll(over) : some ? 63 - __builtin_clzll(some) : -1;
                        if (l >= 0) {
                            at = k0 + l;
                            at_before = lane_f64(c - s, l);
                        }
                        found = over != 0;
                    }
                    if (seek) break;
                    if (before > 0.0) {
                        // (no sum passes a uniform of 1: not left to the whole's last bits, which the
                        // walk within a slice, by 64-bit weights, does not share)
                        goal = un < 1.0f ? (double)un * before : (double)__builtin_inff();
                        seek = true;
                    } else if (left) {
                        left = false;
                        mine0 = slice_sum(lane);
                    } else
                        break;
                }
                if (lane == 0) {
                    s_slice = at;
                    s_goal = goal - at_before;
                    s_left = left;  // (not s_last: a wavefront may still be reading it)
                    s_pick = VR_SLICE;
                    s_best = -1;
                }
            }
            __syncthreads();
            const int at = s_slice;
            if (at >= 0) {
                // Inside the slice, a strip at a time: the threads' sums scanned.
                left = s_left;
                double before = 0.0;
#pragma unroll 1
                for (int y = 0; y < SUB; ++y) {
                    float l[VP_EACH], d[VP_EACH];
                    double w[VP_EACH];
                    const int t0 = (y * VP_THREADS + tid) * VP_EACH;
                    fetch(at * VR_SLICE + t0, left, l, d);
                    const double s = weigh(at * VR_SLICE + t0, left, l, d, w), z = wave_scan(s);
                    if (lane == 63) ss[y & 1][wave] = z;
                    __syncthreads();
                    double run = before + (z - s);
#pragma unroll
                    for (int x = 0; x < VP_WAVES; ++x) {
                        if (x < wave) run += ss[y & 1][x];
                        before += ss[y & 1][x];
                    }
                    int over = -1, last = -1;
#pragma unroll
                    for (int k = 0; k < VP_EACH; ++k) {
                        run += w[k];
                        if (w[k] > 0.0) last = t0 + k;
                        if (w[k] > 0.0 && over < 0 && run > s_goal) over = t0 + k;
                    }
                    // (the wavefront's first and last: one lane each goes to LDS)
                    const uint64_t overs = __ballot(over >= 0), lasts = __ballot(last >= 0);
                    if (overs && lane == __builtin_ctzll(overs)) atomicMin(&s_pick, over);
                    if (lasts && lane == 63 - __builtin_clzll(lasts)) atomicMax(&s_best, last);
                    if (before > s_goal) break;  // (the same in every thread)
                }
                __syncthreads();
                // (the same in every thread, each in a register of its own: slower wavefronts still read s_best)
                pick = at * VR_SLICE + max(s_pick < VR_SLICE ? s_pick : s_best, 0);
            }
        }
    }
    for (int i = tid; i <= n; i += VP_THREADS)
        a.tokens[row0 + i] = i < kept ? drafts[i] : i == kept ? pick : -1;
    if (tid == 0) a.accepted[b] = kept;
}

static int slices_of(int vocab) { return (vocab + VR_SLICE - 1) / VR_SLICE; }

static size_t verify_ws(int batch, int n, int vocab) {
    const size_t k = slices_of(vocab);
    return (size_t)batch * ((n + 1) * k * sizeof(VerifySlice) + k * 8 + 16);
}

template <int LT, int PT>
static void launch_verify(const VerifyArgs& a, hipStream_t s) {
    const dim3 rows((unsigned)((int64_t)a.batch * (a.n + 1) * a.nslices)), one(a.batch), t(VR_THREADS), many(256), few(1024);
    if (a.c == 0.0) {
        hipLaunchKernelGGL((k_verify_rows<LT, true>), rows, t, 0, s, a);
        hipLaunchKernelGGL((k_verify_pick<LT, KV4_F32, true, false>), one, few, 0, s, a);
    } else {
        hipLaunchKernelGGL((k_verify_rows<LT, false>), rows, t, 0, s, a);
        if (a.probs)
            hipLaunchKernelGGL((k_verify_pick<LT, PT, false, true>), dim3(a.batch * a.nslices), many, 0, s, a);
        else
            hipLaunchKernelGGL((k_verify_pick<LT, KV4_F32, false, false>), one, few, 0, s, a);
    }
}

template <int LT>
static hipError_t launch_verify(const VerifyArgs& a, int ptype, hipStream_t s) {
    if (ptype == KV4_F32) launch_verify<LT, KV4_F32>(a, s);
    else if (ptype == KV4_F16) launch_verify<LT, KV4_F16>(a, s);
    else launch_verify<LT, KV4_BF16>(a, s);
    return hipGetLastError();
}

}  // namespace nh

namespace {

int fail(int code, const std::string& msg) {
    nh::set_error(msg);
    return code;
}

int check_sizes(int batch, int n, int vocab) {
    if (batch < 0 || n < 0 || n > 1024 || vocab < 1 || vocab > (1 << 30))
        return fail(NH_EINVAL, "a batch of 0 to 1024 drafts over 1 to 2^30 tokens");
    // (a launch takes fewer than 2^32 threads: a workgroup of 256 a slice of a row, one of 1024 a sequence)
    if ((int64_t)batch * (n + 1) * nh::slices_of(vocab) >= (1 << 24) || batch >= (1 << 22))
        return fail(NH_EINVAL, "too many rows");
    return NH_OK;
}

bool known_type(int t) { return t == NH_F32 || t == NH_F16 || t == NH_BF16; }

}  // namespace

extern "C" {

int64_t nh_verify_drafts_ws_bytes(int batch, int n, int vocab) {
    if (int rc = check_sizes(batch, n, vocab)) return rc;
    return (int64_t)nh::verify_ws(batch, n, vocab);
}

int nh_verify_drafts(const void* logits, int type, int64_t ldl, const int32_t* drafts, const int32_t* counts,
                     const void* probs, int probs_type, int64_t ldp, const float* u, float temperature, int batch, int n,
                     int vocab, int32_t* accepted, int32_t* tokens, void* ws, uint64_t ws_bytes, void* stream) {
    if (int rc = check_sizes(batch, n, vocab)) return rc;
    if (!known_type(type) || (probs && !known_type(probs_type))) return fail(NH_EINVAL, "no such type");
    if (!(temperature >= 0.0f && temperature < INFINITY)) return fail(NH_EINVAL, "the temperature is 0 (greedy) or positive");
    if (ldl < vocab || (probs && n > 0 && ldp < vocab)) return fail(NH_EINVAL, "rows overlap");
    if (!nh::ready()) return fail(NH_ESTATE, "nh_init has not been called");
    if (batch == 0) return NH_OK;
    if (!logits || !accepted || !tokens || (n > 0 && !drafts) || (temperature > 0.0f && !u))
        return fail(NH_EINVAL, "null argument");
    if (!ws || (uintptr_t)ws % 16 != 0) return fail(NH_EINVAL, "no 16-byte aligned workspace");
    if (ws_bytes < nh::verify_ws(batch, n, vocab)) return fail(NH_ESMALL, "the workspace is too small");
    const int k = nh::slices_of(vocab);
    nh::VerifyArgs a{};
    a.logits = logits, a.drafts = drafts, a.counts = counts, a.probs = n > 0 ? probs : nullptr, a.u = u;
    a.accepted = accepted, a.tokens = tokens;
    a.slices = (nh::VerifySlice*)ws;
    a.rest = (double*)(a.slices + (size_t)batch * (n + 1) * k);
    a.arrived = (int*)(a.rest + (size_t)batch * k);
    a.ldl = ldl, a.ldp = ldp, a.batch = batch, a.n = n, a.vocab = vocab, a.nslices = k;
    const int es = type == NH_F32 ? 4 : 2;
    a.aligned = (uintptr_t)logits % 16 == 0 && ldl * es % 16 == 0;
    a.paligned = (uintptr_t)probs % 16 == 0 && ldp * (probs_type == NH_F32 ? 4 : 2) % 16 == 0;
    a.c = temperature > 0.0f ? 1.4426950408889634074 / (double)temperature : 0.0;
    const hipStream_t st = (hipStream_t)stream;
    const int pt = probs ? probs_type : NH_F32;
    const hipError_t e = type == NH_F32   ? nh::launch_verify<nh::KV4_F32>(a, pt, st)
                         : type == NH_F16 ? nh::launch_verify<nh::KV4_F16>(a, pt, st)
                                          : nh::launch_verify<nh::KV4_BF16>(a, pt, st);
    if (e != hipSuccess) return fail(NH_EDEVICE, std::string("verify: ") + hipGetErrorString(e));
    return NH_OK;
}

}  // extern "C"
