// Verification of drafted tokens against the target's logits
// (nh_verify_drafts in include/needle_hip.h).
//
//   p = softmax(l / T); draft x_i is kept while u_i q(x_i) < p_i(x_i), in
//   turn; the token after the last kept one is drawn from max(p - q, 0) where
//   a draft was refused (from p without it for drafts without probabilities),
//   else from p, at the uniform u_n: the first t with w_0 + .. + w_t > u_n W.
//
// Sums and weights are in f64: a pick next to a border of the cumulative sum
// does not depend on how the sum was split.
#include <math.h>

#include "../../include/needle_hip.h"
#include "nh_kv4_device.h"

namespace nh {

struct VerifyArgs {
    const void* logits;
    const int* drafts;
    const int* counts;   // or null: n each
    const void* probs;   // or null
    const float* u;
    int* accepted;
    int* tokens;
    void* ws;
    int64_t ldl, ldp;
    int batch, n, vocab;
    double inv_t;        // 0: greedy
};

struct VerifyRow {
    double sum;  // of the weights, the largest is 1
    float max;
    int best;    // the first index of the maximum, as nh_argmax has it
};

// The weight of logit l beside the row's largest, m (NaN weighs nothing).
__device__ __forceinline__ double verify_weight(float l, float m, double inv_t) {
    if (l == m) return 1.0;
    const double x = ((double)l - (double)m) * inv_t;
    return l < m ? exp(x) : 0.0;
}

// (value, index) of the first maximum of two; index -1: none yet.
__device__ __forceinline__ void verify_best(float& v, int& i, float w, int j) {
    if (j >= 0 && (i < 0 || w > v || (w == v && j < i))) v = w, i = j;
}

template <int LT>
__global__ __launch_bounds__(256) void k_verify_rows(VerifyArgs a) {
    typedef typename Kv4Elem<LT>::T T;
    __shared__ float sv[256];
    __shared__ int si[256];
    __shared__ double ss[256];
    const int row = blockIdx.x, tid = threadIdx.x;
    const T* x = reinterpret_cast<const T*>(a.logits) + (int64_t)row * a.ldl;
    float v = 0.0f;
    int at = -1;
    for (int t = tid; t < a.vocab; t += 256) {
        const float l = Kv4Elem<LT>::get(x + t);
        if (l == l) verify_best(v, at, l, t);
    }
    sv[tid] = v, si[tid] = at;
    __syncthreads();
    for (int h = 128; h; h >>= 1) {
        if (tid < h) verify_best(sv[tid], si[tid], sv[tid + h], si[tid + h]);
        __syncthreads();
    }
    const float m = si[0] >= 0 ? sv[0] : -__builtin_inff();
    double sum = 0.0;
    if (a.inv_t != 0.0 && m > -__builtin_inff())
        for (int t = tid; t < a.vocab; t += 256) sum += verify_weight(Kv4Elem<LT>::get(x + t), m, a.inv_t);
    ss[tid] = sum;
    __syncthreads();
    for (int h = 128; h; h >>= 1) {
        if (tid < h) ss[tid] += ss[tid + h];
        __syncthreads();
    }
    if (tid == 0) {
        const float first = Kv4Elem<LT>::get(x);
        VerifyRow* r = reinterpret_cast<VerifyRow*>(a.ws) + row;
        r->sum = ss[0];
        r->max = m;
        r->best = first != first || si[0] < 0 ? 0 : si[0];
    }
}

template <int LT, int PT>
__global__ __launch_bounds__(256) void k_verify_pick(VerifyArgs a) {
    typedef typename Kv4Elem<LT>::T T;
    typedef typename Kv4Elem<PT>::T P;
    __shared__ int s_kept;
    __shared__ double ss[256];
    __shared__ int s_last, s_pick;
    const int b = blockIdx.x, tid = threadIdx.x, n = a.n;
    const VerifyRow* rows = reinterpret_cast<const VerifyRow*>(a.ws) + (int64_t)b * (n + 1);
    const T* logits = reinterpret_cast<const T*>(a.logits) + (int64_t)b * (n + 1) * a.ldl;
    const P* probs = a.probs ? reinterpret_cast<const P*>(a.probs) + (int64_t)b * n * a.ldp : nullptr;
    const int cnt = a.counts ? min(max(a.counts[b], 0), n) : n;
    if (tid == 0) {
        int i = 0;
        for (; i < cnt; ++i) {
            const int x = a.drafts[(int64_t)b * n + i];
            const VerifyRow r = rows[i];
            bool ok = (unsigned)x < (unsigned)a.vocab;
            if (ok && a.inv_t == 0.0) ok = x == r.best;
            else if (ok) {
                const double p = r.sum > 0.0 ? verify_weight(Kv4Elem<LT>::get(logits + i * a.ldl + x), r.max, a.inv_t) / r.sum : 0.0;
                const double q = probs ? (double)Kv4Elem<PT>::get(probs + i * a.ldp + x) : 1.0;
                ok = (double)a.u[(int64_t)b * (n + 1) + i] * q < p;
            }
            if (!ok) break;
        }
        s_kept = i;
        s_last = -1;
        s_pick = -1;
    }
    __syncthreads();
    const int kept = s_kept;
    const VerifyRow r = rows[kept];
    int pick = r.best;
    if (a.inv_t != 0.0 && r.sum > 0.0) {
        const T* x = logits + kept * a.ldl;
        const P* q = probs && kept < cnt ? probs + kept * a.ldp : nullptr;
        const int out = kept < cnt ? a.drafts[(int64_t)b * n + kept] : -1;
        bool rest = kept < cnt;  // weigh what the draft left
        auto weight = [&](int t) -> double {
            const double p = verify_weight(Kv4Elem<LT>::get(x + t), r.max, a.inv_t) / r.sum;
            if (!rest) return p;
            if (!q) return t == out ? 0.0 : p;
            const double d = p - (double)Kv4Elem<PT>::get(q + t);
            return d > 0.0 ? d : 0.0;
        };
        double total = 0.0;
        for (int pass = 0; pass < 2; ++pass) {
            double sum = 0.0;
            int last = -1;
            for (int t = tid; t < a.vocab; t += 256) {
                const double w = weight(t);
                sum += w;
                if (w > 0.0) last = t;
            }
            ss[tid] = sum;
            if (last >= 0) atomicMax(&s_last, last);
            __syncthreads();
            for (int h = 128; h; h >>= 1) {
                if (tid < h) ss[tid] += ss[tid + h];
                __syncthreads();
            }
            total = ss[0];
            __syncthreads();
            if (total > 0.0 || !rest) break;
            rest = false;
        }
        const double goal = (double)a.u[(int64_t)b * (n + 1) + n] * total;
        double before = 0.0;
        for (int t0 = 0; t0 < a.vocab; t0 += 256) {
            ss[tid] = t0 + tid < a.vocab ? weight(t0 + tid) : 0.0;
            __syncthreads();
            for (int h = 1; h < 256; h <<= 1) {
                const double w = tid >= h ? ss[tid - h] : 0.0;
                __syncthreads();
                ss[tid] += w;
                __syncthreads();
            }
            const double mine = before + ss[tid], prev = before + (tid ? ss[tid - 1] : 0.0);
            before += ss[255];
            if (mine > goal && (tid == 0 || !(prev > goal))) s_pick = t0 + tid;
            __syncthreads();
            if (s_pick >= 0) break;
        }
        pick = s_pick >= 0 ? min(s_pick, s_last) : max(s_last, 0);
    }
    for (int i = tid; i <= n; i += 256)
        a.tokens[(int64_t)b * (n + 1) + i] = i < kept ? a.drafts[(int64_t)b * n + i] : i == kept ? pick : -1;
    if (tid == 0) a.accepted[b] = kept;
}

static size_t verify_ws(int batch, int n, int) { return (size_t)batch * (n + 1) * sizeof(VerifyRow); }

template <int LT>
static hipError_t launch_verify(const VerifyArgs& a, int ptype, hipStream_t s) {
    hipLaunchKernelGGL(k_verify_rows<LT>, dim3(a.batch * (a.n + 1)), dim3(256), 0, s, a);
    auto kern = ptype == KV4_F32 ? k_verify_pick<LT, KV4_F32> : ptype == KV4_F16 ? k_verify_pick<LT, KV4_F16> : k_verify_pick<LT, KV4_BF16>;
    hipLaunchKernelGGL(kern, dim3(a.batch), dim3(256), 0, s, a);
    return hipGetLastError();
}

}  // namespace nh

namespace {

int fail(int code, const std::string& msg) {
    nh::set_error(msg);
    return code;
}

int check_sizes(int batch, int n, int vocab) {
    if (batch < 0 || n < 0 || n > 1024 || vocab < 1) return fail(NH_EINVAL, "a batch of 0 to 1024 drafts over at least one token");
    if ((int64_t)batch * (n + 1) > (1 << 24)) return fail(NH_EINVAL, "too many rows");
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
    nh::VerifyArgs a{logits, drafts, counts, n > 0 ? probs : nullptr, u, accepted, tokens, ws, ldl, ldp, batch, n, vocab,
                     temperature > 0.0f ? 1.0 / (double)temperature : 0.0};
    const hipStream_t st = (hipStream_t)stream;
    const int pt = probs ? probs_type : NH_F32;
    const hipError_t e = type == NH_F32   ? nh::launch_verify<nh::KV4_F32>(a, pt, st)
                         : type == NH_F16 ? nh::launch_verify<nh::KV4_F16>(a, pt, st)
                                          : nh::launch_verify<nh::KV4_BF16>(a, pt, st);
    if (e != hipSuccess) return fail(NH_EDEVICE, std::string("verify: ") + hipGetErrorString(e));
    return NH_OK;
}

}  // extern "C"
