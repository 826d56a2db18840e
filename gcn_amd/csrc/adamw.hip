// The optimiser's two passes over all parameter tensors at once: the gradients' norm and the AdamW step,
// with moments in 32 bits or in 8.  They stand beside the update rules of forward.hip (plain and AdaGrad).
//
// Both read a list of tensors of any sizes in as few launches as possible: the list travels in the
// kernel's arguments (LIST tensors a launch), every tensor is cut into chunks, and a workgroup finds
// its chunk's tensor by bisection over the chunk counts.
#include <cmath>

#include "numeric.h"
#include "profile.h"

namespace ccnn {

constexpr int LIST = 64;          // tensors per launch: the argument block stays under 4 KB
constexpr int BLOCK = CCNN_MOMENT_BLOCK;

// ---------------------------------------------------------------------------- gradient norm
constexpr long NORM_CHUNK = 16384;

struct NormList {
    const void *data[LIST];
    long n[LIST];
    int chunk0[LIST + 1];   // first chunk of each tensor; [count] = all
    int count;
};

template <typename L>
__device__ __forceinline__ int find(const L &list, int chunk)
{
    int lo = 0, hi = list.count;   // chunk0[lo] <= chunk < chunk0[hi]
    while (hi - lo > 1) {
        const int mid = (lo + hi) >> 1;
        if (list.chunk0[mid] <= chunk) lo = mid;
        else hi = mid;
    }
    return lo;
}

// Sum over a workgroup of 256 in a fixed order; the result is in thread 0.
__device__ __forceinline__ double block_sum(double v, double *lds)
{
    for (int off = 32; off > 0; off >>= 1) v += __shfl_down(v, off);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    return lds[0] + lds[1] + lds[2] + lds[3];
}

template <typename T>
__global__ __launch_bounds__(256) void norm_partial(NormList list, double *__restrict__ partial)
{
    __shared__ double lds[4];
    const int i = find(list, blockIdx.x);
    const T *p = (const T *)list.data[i];
    const long lo = (long)(blockIdx.x - list.chunk0[i]) * NORM_CHUNK;
    const long n = min(list.n[i], lo + NORM_CHUNK);
    double s = 0;
    for (long k = lo + threadIdx.x; k < n; k += 256) {
        const double g = widen(p[k]);
        s += g * g;
    }
    s = block_sum(s, lds);
    if (threadIdx.x == 0) partial[blockIdx.x] = s;
}

__global__ __launch_bounds__(256) void norm_total(const double *__restrict__ partial, int n, double max_norm,
                                                  double *__restrict__ out)
{
    __shared__ double lds[4];
    double s = 0;
    for (int k = threadIdx.x; k < n; k += 256) s += partial[k];
    s = block_sum(s, lds);
    if (threadIdx.x == 0) {
        const double norm = sqrt(s);
        out[0] = norm;
        out[1] = !(norm < __builtin_huge_val()) ? __builtin_nan("") : norm > max_norm ? max_norm / norm : 1.0;
    }
}

// ---------------------------------------------------------------------------- AdamW
constexpr long STEP_CHUNK = 4096;

struct StepList {
    void *param[LIST];
    const void *grad[LIST];
    long n[LIST], first[LIST];
    int block[LIST];
    double decay[LIST];
    int chunk0[LIST + 1];
    int count;
};

struct StepArgs {
    void *m, *v;
    float *m_scale, *v_scale, *master;
    const double *clock;
    double beta1, beta2, eps;
};

// clock: t, beta1^t, beta2^t | lr, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), gradient factor (NaN: no step)
__global__ void adamw_clock(double *clock, double lr, const double *lr_device, double beta1, double beta2, const double *clip)
{
    const double scale = clip ? clip[1] : 1.0;
    clock[6] = scale;
    if (!(fabs(scale) < __builtin_huge_val())) {
        clock[6] = __builtin_nan("");
        return;
    }
    const double rate = lr_device ? *lr_device : lr;
    clock[0] += 1;
    clock[1] *= beta1;
    clock[2] *= beta2;
    clock[3] = rate;
    clock[4] = rate / (1 - clock[1]);
    clock[5] = 1 / sqrt(1 - clock[2]);
}

template <typename A>
struct Rates {
    A scale, lr_decay, rate, root, eps;
    double scale64;
    bool skip;
    __device__ Rates(const StepArgs &a, double decay)
        : scale((A)a.clock[6]), lr_decay((A)(a.clock[3] * decay)), rate((A)a.clock[4]), root((A)a.clock[5]), eps((A)a.eps),
          scale64(a.clock[6]), skip(!(a.clock[6] == a.clock[6]))
    {
    }
};

template <typename A>
__device__ __forceinline__ A stepped(A p, A m, A v_root, const Rates<A> &r)
{
    return p - (r.lr_decay * p + r.rate * m / (v_root * r.root + r.eps));
}

template <typename P, typename G>
__global__ __launch_bounds__(256) void adamw_wide(StepList list, StepArgs a)
{
    typedef Wide<P> A;
    constexpr bool COPY = sizeof(P) == 2;   // the parameter is the rounding of its master copy
    const int i = find(list, blockIdx.x);
    const Rates<A> r(a, list.decay[i]);
    if (r.skip) return;
    P *param = (P *)list.param[i];
    const G *grad = (const G *)list.grad[i];
    A *m = (A *)a.m + list.first[i], *v = (A *)a.v + list.first[i];
    float *master = COPY ? a.master + list.first[i] : nullptr;
    const long lo = (long)(blockIdx.x - list.chunk0[i]) * STEP_CHUNK;
    const long n = min(list.n[i], lo + STEP_CHUNK);
    const A b1 = (A)(1 - a.beta1), b2 = (A)(1 - a.beta2);
    for (long k = lo + threadIdx.x; k < n; k += 256) {
        const A g = (A)widen(grad[k]) * r.scale;
        const A mk = m[k] + b1 * (g - m[k]), vk = v[k] + b2 * (g * g - v[k]);
        m[k] = mk;
        v[k] = vk;
        A p;
        if constexpr (COPY) p = master[k];
        else p = param[k];
        p = stepped(p, mk, (A)sqrt(vk), r);
        if constexpr (COPY) master[k] = p;
        narrow(p, param[k]);
    }
}

// e4m3: values 2^-9 apart below 2^-6, then eight to each power of two up to 448.
__device__ __forceinline__ float decode8(unsigned code)
{
    return __builtin_amdgcn_cvt_f32_fp8((int)code, 0);
}

// The code nearest to 0 <= y <= 448, ties to the even code, decided in 64 bits.
__device__ __forceinline__ unsigned encode8(double y)
{
    if (!(y >= 0x1p-6)) return y == y ? (unsigned)rint(y * 0x1p9) : 0x7fu;
    const unsigned long long u = __double_as_longlong(y) + ((1ull << 48) - 1) + ((__double_as_longlong(y) >> 49) & 1);
    return (unsigned)(u >> 49) - ((1023u - 7u) << 3);
}

// Largest of 64 lanes; any NaN wins (compared as the bits of magnitudes).
__device__ __forceinline__ float wave_high(double v)
{
    unsigned u = __float_as_uint(fabsf((float)v));
    for (int off = 32; off > 0; off >>= 1) u = max(u, (unsigned)__shfl_xor((int)u, off));
    return __uint_as_float(u);
}

// beta old + (1 - beta) new, every product and the sum rounded by itself.  With a beta like 9/10 the result
// often lies exactly between two fp32 values, so a block's fp32 scale would hang on how the compiler
// contracts the expression.
__device__ __forceinline__ double decay_to(double beta, double old, double now)
{
#pragma clang fp contract(off)
    const double a = beta * old, b = (1 - beta) * now;
    return a + b;
}

__device__ __forceinline__ unsigned pack_codes(const double (&x)[4], float scale, bool floor)
{
    unsigned w = 0;
    for (int e = 0; e < 4; e++) {
        const double y = fabs(x[e]);
        unsigned c = scale > 0 ? encode8(fmin(y / scale, 448.0)) : scale == 0 ? 0u : 0x7fu;
        if (y != y) c = 0x7f;
        if (floor && y > 0 && scale > 0 && c == 0) c = 1;
        if (x[e] < 0) c |= 0x80;
        w |= c << (8 * e);
    }
    return w;
}

// One wave per block of 256 elements, four to a lane.
template <typename P, typename G>
__global__ __launch_bounds__(256) void adamw_coded(StepList list, StepArgs a)
{
    constexpr bool COPY = sizeof(P) == 2;
    const int i = find(list, blockIdx.x);
    const Rates<float> r(a, list.decay[i]);
    if (r.skip) return;
    P *param = (P *)list.param[i];
    const G *grad = (const G *)list.grad[i];
    float *master = COPY ? a.master + list.first[i] : nullptr;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const long lo = (long)(blockIdx.x - list.chunk0[i]) * STEP_CHUNK;
    const long n = list.n[i], hi = min(n, lo + STEP_CHUNK);
    for (long b = lo + wave * BLOCK; b < hi; b += 4 * BLOCK) {
        const long blk = list.block[i] + b / BLOCK;
        unsigned *mw = (unsigned *)a.m + blk * (BLOCK / 4) + lane, *vw = (unsigned *)a.v + blk * (BLOCK / 4) + lane;
        const unsigned mc = *mw, vc = *vw;
        const double ms = a.m_scale[blk], vs = a.v_scale[blk];
        double m[4], v[4], root[4];
        double hm = 0, hv = 0;
        bool nan_m = false, nan_v = false;
        for (int e = 0; e < 4; e++) {
            const long k = b + lane * 4 + e;
            const double g = k < n ? (double)widen(grad[k]) * r.scale64 : 0.0;
            const double mo = decode8((mc >> (8 * e)) & 255) * ms, vo = decode8((vc >> (8 * e)) & 255) * vs;
            m[e] = decay_to(a.beta1, mo, g);
            v[e] = decay_to(a.beta2, vo * vo, g * g);
            root[e] = sqrt(v[e]);
            hm = fmax(hm, fabs(m[e]));
            hv = fmax(hv, root[e]);
            nan_m |= !(fabs(m[e]) < __builtin_huge_val());
            nan_v |= !(v[e] < __builtin_huge_val());
        }
        const float high_m = wave_high(nan_m ? __builtin_nan("") : hm), high_v = wave_high(nan_v ? __builtin_nan("") : hv);
        const float sm = high_m / 448.0f, sv = high_v / 448.0f;
        *mw = pack_codes(m, sm, false);
        *vw = pack_codes(root, sv, true);
        if (lane == 0) a.m_scale[blk] = sm, a.v_scale[blk] = sv;
        for (int e = 0; e < 4; e++) {
            const long k = b + lane * 4 + e;
            if (k >= n) break;
            float p;
            if constexpr (COPY) p = master[k];
            else p = param[k];
            p = stepped(p, (float)m[e], (float)root[e], r);
            if constexpr (COPY) master[k] = p;
            narrow(p, param[k]);
        }
    }
}

__global__ __launch_bounds__(256) void adamw_decode(StepList list, const unsigned char *__restrict__ m,
                                                    const unsigned char *__restrict__ v, const float *__restrict__ m_scale,
                                                    const float *__restrict__ v_scale, float *__restrict__ m_out,
                                                    float *__restrict__ v_out)
{
    const int i = find(list, blockIdx.x);
    const long lo = (long)(blockIdx.x - list.chunk0[i]) * STEP_CHUNK;
    const long n = min(list.n[i], lo + STEP_CHUNK);
    for (long k = lo + threadIdx.x; k < n; k += 256) {
        const long at = (long)list.block[i] * BLOCK + k, blk = at / BLOCK;
        const double root = (double)decode8(v[at]) * v_scale[blk];
        m_out[list.first[i] + k] = (float)((double)decode8(m[at]) * m_scale[blk]);
        v_out[list.first[i] + k] = (float)(root * root);
    }
}

// ---------------------------------------------------------------------------- host
// Hands tensors [0, count) that `take` accepts to `go`, LIST at a time, with their chunks counted.
template <typename List, typename Take, typename Go>
int in_lists(int count, long chunk, Take take, Go go)
{
    List list;
    list.count = 0;
    list.chunk0[0] = 0;
    for (int i = 0; i <= count; i++) {
        long chunks = 0;
        if (i < count) {
            const long n = take(list, i);
            if (n <= 0) continue;
            chunks = (n + chunk - 1) / chunk;
            if (chunks > 0x3fffffffL) return CCNN_E_RANGE;
        }
        const bool full = list.count == LIST || (list.count > 0 && list.chunk0[list.count] + chunks > 0x7fffffffL);
        if (list.count > 0 && (i == count || full)) {
            if (int e = go(list)) return e;
            list.count = 0;
        }
        if (i < count) {
            take(list, i);   // the slot may have moved to the front of a new list
            list.chunk0[list.count + 1] = list.chunk0[list.count] + (int)chunks;
            list.count++;
        }
    }
    return 0;
}

}  // namespace ccnn

using namespace ccnn;

extern "C" {

size_t ccnn_grad_norm_workspace_bytes(const ccnn_tensor_t *tensors, int count)
{
    if (!tensors || count < 0) return 0;
    size_t chunks = 1;
    for (int i = 0; i < count; i++)
        if (tensors[i].n > 0) chunks += (size_t)((tensors[i].n + NORM_CHUNK - 1) / NORM_CHUNK);
    return chunks * sizeof(double);
}

int ccnn_grad_norm(const ccnn_tensor_t *tensors, int count, double max_norm, double *out, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (count < 0 || (count > 0 && !tensors) || !out || !(max_norm > 0)) return CCNN_E_INVALID;
    for (int i = 0; i < count; i++)
        if (!type_bytes(tensors[i].type) || tensors[i].n < 0 || (tensors[i].n > 0 && !tensors[i].data)) return CCNN_E_INVALID;
    const size_t need = ccnn_grad_norm_workspace_bytes(tensors, count);
    if (need / sizeof(double) > 0x7fffffffu) return CCNN_E_RANGE;
    if (!workspace || workspace_bytes < need) return CCNN_E_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    double *partial = (double *)workspace;
    int done = 0;
    for (int type = CCNN_TYPE_F32; type <= CCNN_TYPE_F16; type++) {
        const int e = in_lists<NormList>(
            count, NORM_CHUNK,
            [&](NormList &list, int i) -> long {
                if (tensors[i].type != type) return 0;
                if (list.count < LIST) {
                    list.data[list.count] = tensors[i].data;
                    list.n[list.count] = tensors[i].n;
                }
                return tensors[i].n;
            },
            [&](const NormList &list) -> int {
                const int chunks = list.chunk0[list.count];
                const dim3 grid((unsigned)chunks), block(256);
                if (type == CCNN_TYPE_F32) launch("norm_partial", norm_partial<float>, grid, block, 0, st, list, partial + done);
                else if (type == CCNN_TYPE_F64) launch("norm_partial", norm_partial<double>, grid, block, 0, st, list, partial + done);
                else if (type == CCNN_TYPE_BF16) launch("norm_partial", norm_partial<Bf16>, grid, block, 0, st, list, partial + done);
                else launch("norm_partial", norm_partial<F16>, grid, block, 0, st, list, partial + done);
                CCNN_LAUNCH_CHECK();
                done += chunks;
                return 0;
            });
        if (e) return e;
    }
    launch("norm_total", norm_total, dim3(1), dim3(256), 0, st, partial, done, max_norm, out);
    CCNN_LAUNCH_CHECK();
    return 0;
}

int ccnn_adamw_step(const ccnn_adamw_tensor_t *tensors, int count, int moment_bits, void *m, void *v, float *m_scale,
                    float *v_scale, float *master, double *clock, double lr, const double *lr_device, double beta1,
                    double beta2, double eps, const double *clip, void *stream)
{
    if (count < 0 || (count > 0 && !tensors) || !clock) return CCNN_E_INVALID;
    if (moment_bits != 32 && moment_bits != 8) return CCNN_E_INVALID;
    if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps >= 0)) return CCNN_E_INVALID;
    bool wide = false, other = false, any = false;
    for (int i = 0; i < count; i++) {
        const ccnn_adamw_tensor_t &t = tensors[i];
        const bool half = t.type == CCNN_TYPE_BF16 || t.type == CCNN_TYPE_F16;
        if (!type_bytes(t.type) || (t.grad_type != t.type && !(half && t.grad_type == CCNN_TYPE_F32))) return CCNN_E_INVALID;
        if (t.n < 0 || (t.n > 0 && (!t.param || !t.grad || t.first < 0 || t.block < 0))) return CCNN_E_INVALID;
        if (moment_bits == 8 && t.block > 0x7fffffffL) return CCNN_E_RANGE;
        if (half && t.n > 0 && !master) return CCNN_E_INVALID;
        (t.type == CCNN_TYPE_F64 ? wide : other) = true;
        any |= t.n > 0;
    }
    if (wide && (other || moment_bits == 8)) return CCNN_E_INVALID;
    if (any && (!m || !v || (moment_bits == 8 && (!m_scale || !v_scale)))) return CCNN_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    launch("adamw_clock", adamw_clock, dim3(1), dim3(1), 0, st, clock, lr, lr_device, beta1, beta2, clip);
    CCNN_LAUNCH_CHECK();
    const StepArgs args = {m, v, m_scale, v_scale, master, clock, beta1, beta2, eps};
    typedef void (*Kern)(StepList, StepArgs);
    const struct {
        int type, grad_type;
        Kern wide, coded;
    } kinds[] = {
        {CCNN_TYPE_F32, CCNN_TYPE_F32, adamw_wide<float, float>, adamw_coded<float, float>},
        {CCNN_TYPE_F64, CCNN_TYPE_F64, adamw_wide<double, double>, nullptr},
        {CCNN_TYPE_BF16, CCNN_TYPE_BF16, adamw_wide<Bf16, Bf16>, adamw_coded<Bf16, Bf16>},
        {CCNN_TYPE_BF16, CCNN_TYPE_F32, adamw_wide<Bf16, float>, adamw_coded<Bf16, float>},
        {CCNN_TYPE_F16, CCNN_TYPE_F16, adamw_wide<F16, F16>, adamw_coded<F16, F16>},
        {CCNN_TYPE_F16, CCNN_TYPE_F32, adamw_wide<F16, float>, adamw_coded<F16, float>},
    };
    for (const auto &kind : kinds) {
        const int e = in_lists<StepList>(
            count, STEP_CHUNK,
            [&](StepList &list, int i) -> long {
                const ccnn_adamw_tensor_t &t = tensors[i];
                if (t.type != kind.type || t.grad_type != kind.grad_type) return 0;
                if (const int c = list.count; c < LIST) {
                    list.param[c] = t.param;
                    list.grad[c] = t.grad;
                    list.n[c] = t.n;
                    list.first[c] = t.first;
                    list.block[c] = (int)t.block;
                    list.decay[c] = t.decay;
                }
                return t.n;
            },
            [&](const StepList &list) -> int {
                launch(moment_bits == 8 ? "adamw_coded" : "adamw_wide", moment_bits == 8 ? kind.coded : kind.wide,
                       dim3((unsigned)list.chunk0[list.count]), dim3(256), 0, st, list, args);
                CCNN_LAUNCH_CHECK();
                return 0;
            });
        if (e) return e;
    }
    return 0;
}

int ccnn_adamw_moments(const ccnn_adamw_tensor_t *tensors, int count, const void *m, const void *v, const float *m_scale,
                       const float *v_scale, float *m_out, float *v_out, void *stream)
{
    if (count < 0 || (count > 0 && !tensors)) return CCNN_E_INVALID;
    for (int i = 0; i < count; i++) {
        if (tensors[i].n < 0 || tensors[i].first < 0 || tensors[i].block < 0) return CCNN_E_INVALID;
        if (tensors[i].n > 0 && (!m || !v || !m_scale || !v_scale || !m_out || !v_out)) return CCNN_E_INVALID;
        if (tensors[i].block > 0x7fffffffL) return CCNN_E_RANGE;
    }
    return in_lists<StepList>(
        count, STEP_CHUNK,
        [&](StepList &list, int i) -> long {
            if (const int c = list.count; c < LIST) {
                list.n[c] = tensors[i].n;
                list.first[c] = tensors[i].first;
                list.block[c] = (int)tensors[i].block;
            }
            return tensors[i].n;
        },
        [&](const StepList &list) -> int {
            launch("adamw_decode", adamw_decode, dim3((unsigned)list.chunk0[list.count]), dim3(256), 0, (hipStream_t)stream,
                   list, (const unsigned char *)m, (const unsigned char *)v, m_scale, v_scale, m_out, v_out);
            CCNN_LAUNCH_CHECK();
            return 0;
        });
}

}  // extern "C"
