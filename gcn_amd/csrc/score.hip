// Log probabilities of given classes with entropy and the most likely alternatives, and their
// gradient to the logits.  Beside the forward pass's probabilities and argmax (forward.hip) this is
// the scored answer, and the loss of a training step.
//
//   m = max_j x_j      l = log sum_j exp(x_j - m)      log p_j = x_j - m - l
//   logp = log p_y     H = -sum_j p_j log p_j = l - sum_j e^(x_j - m)(x_j - m) / sum_j e^(x_j - m)
//   dx_j = dL (1[j = y] - p_j) - dH p_j (log p_j + H)
//
// m and l are kept apart in `stats`: their sum would lose l's low bits next to a large m, and the
// gradient subtracts them one after the other.
#include "numeric.h"
#include "profile.h"

namespace ccnn {

template <typename A>
struct ScoreOut {
    A *logp, *entropy, *top_logp, *stats;   // entropy and top_logp optional
    int *top_index;
    int top;
};

struct Targets {
    const void *p;
    int bytes;
    __device__ __forceinline__ long at(long r) const
    {
        return bytes == 8 ? (long)((const long long *)p)[r] : (long)((const int *)p)[r];
    }
};

// Running softmax sums of part of a row: maximum m, s = sum e^(x-m), t = sum e^(x-m)(x-m).
template <typename A>
struct Sums {
    A m, s, t;
};

__device__ __forceinline__ float expw(float v) { return __builtin_amdgcn_exp2f(v * 1.4426950408889634f); }
__device__ __forceinline__ double expw(double v) { return exp(v); }
__device__ __forceinline__ float logw(float v) { return logf(v); }
__device__ __forceinline__ double logw(double v) { return log(v); }

// A sum about maximum m seen from the larger maximum `to`: e^(x-to) = e^(x-m) e^(m-to), and
// sum e^(x-to)(x-to) = (t + (m - to) s) e^(m-to).  An empty part (m = -inf, s = t = 0) adds nothing.
template <typename A>
__device__ __forceinline__ void shift(Sums<A> &a, A to)
{
    const A far = a.m - to, d = a.m == to ? A(0) : far < A(-1e4) ? A(-1e4) : far;   // e^-1e4 is 0 in either type
    const A f = expw(d);
    a.t = (a.t + d * a.s) * f;
    a.s = a.s * f;
    a.m = to;
}

template <typename A>
__device__ __forceinline__ Sums<A> join(Sums<A> a, Sums<A> b)
{
    const A m = a.m > b.m ? a.m : b.m;
    shift(a, m);
    shift(b, m);
    return {m, a.s + b.s, a.t + b.t};
}

template <typename A>
__device__ __forceinline__ void add_element(Sums<A> &a, A x)
{
    if (x > a.m) shift(a, x);
    if (a.m == ninf(A()) && x == a.m) return;   // nothing allowed so far
    const A d = x - a.m, e = expw(d);
    a.s += e;
    if (e > A(0)) a.t += e * d;                 // -inf and far values weigh nothing, and 0 * inf is not wanted
}

template <typename A>
__device__ __forceinline__ bool before(A v, int i, A w, int j) { return v > w || (v == w && i < j); }

template <typename A>
__device__ __forceinline__ void finish_row(const Sums<A> &a, long r, A given, long y, int classes, const ScoreOut<A> &o)
{
    const bool empty = a.m == ninf(A()) && a.s == A(0);
    const A l = empty ? ninf(A()) : logw(a.s), nan = nan_of(A());
    const bool bad = l != l;
    o.stats[2 * r] = bad ? nan : a.m;
    o.stats[2 * r + 1] = bad ? nan : l;
    o.logp[r] = bad || y >= classes ? nan : y < 0 ? A(0) : empty ? ninf(A()) : (given - a.m) - l;
    if (o.entropy) o.entropy[r] = bad ? nan : empty ? A(0) : l - a.t / a.s;
}

template <typename T>
__global__ __launch_bounds__(256) void log_probs_row(const T *__restrict__ logits, int classes, long stride, Targets targets,
                                                     ScoreOut<Wide<T>> o)
{
    typedef Wide<T> A;
    __shared__ A sm[256], ss[256], stt[256];
    __shared__ int si[256];
    const long r = blockIdx.x;
    const T *row = logits + r * stride;
    const int tid = threadIdx.x;
    Sums<A> a = {ninf(A()), A(0), A(0)};
    for (int j = tid; j < classes; j += 256) add_element(a, (A)widen(row[j]));
    sm[tid] = a.m, ss[tid] = a.s, stt[tid] = a.t;
    __syncthreads();
    for (int h = 128; h > 0; h >>= 1) {
        if (tid < h) {
            a = join(a, {sm[tid + h], ss[tid + h], stt[tid + h]});
            sm[tid] = a.m, ss[tid] = a.s, stt[tid] = a.t;
        }
        __syncthreads();
    }
    a = {sm[0], ss[0], stt[0]};
    const long y = targets.at(r);
    if (tid == 0) finish_row(a, r, y >= 0 && y < classes ? (A)widen(row[y]) : A(0), y, classes, o);
    const bool bad = !(a.s == a.s);
    const A l = a.s == A(0) ? ninf(A()) : logw(a.s);
    A last = A(0);
    int lasti = -1;
    for (int k = 0; k < o.top; k++) {
        __syncthreads();
        A v = ninf(A());
        int i = 0x7fffffff;
        for (int j = tid; j < classes; j += 256) {
            const A x = widen(row[j]);
            if ((k == 0 || before(last, lasti, x, j)) && (before(x, j, v, i))) v = x, i = j;
        }
        sm[tid] = v, si[tid] = i;
        __syncthreads();
        for (int h = 128; h > 0; h >>= 1) {
            if (tid < h && before(sm[tid + h], si[tid + h], sm[tid], si[tid])) sm[tid] = sm[tid + h], si[tid] = si[tid + h];
            __syncthreads();
        }
        last = sm[0], lasti = si[0];
        if (tid == 0) {
            o.top_index[r * o.top + k] = bad ? -1 : lasti;
            o.top_logp[r * o.top + k] = bad ? nan_of(A()) : last == ninf(A()) ? last : (last - a.m) - l;
        }
    }
}

template <typename T>
__global__ __launch_bounds__(256) void log_probs_grad_row(const T *logits, int classes, long stride, Targets targets,
                                                          const Wide<T> *__restrict__ stats, const Wide<T> *__restrict__ entropy,
                                                          const Wide<T> *__restrict__ d_logp,
                                                          const Wide<T> *__restrict__ d_entropy, T *d_logits, long d_stride)
{
    typedef Wide<T> A;
    const long r = blockIdx.x;
    const long y = targets.at(r);
    const A m = stats[2 * r], l = stats[2 * r + 1];
    const A dl = d_logp && y >= 0 ? d_logp[r] : A(0), dh = d_entropy ? d_entropy[r] : A(0), h = d_entropy ? entropy[r] : A(0);
    const bool empty = m == ninf(A()), bad = y >= classes;
    for (int j = threadIdx.x; j < classes; j += 256) {
        const A lp = ((A)widen(logits[r * stride + j]) - m) - l, p = expw(lp);
        A g = (y == j ? dl : A(0)) - dl * p;
        if (p > A(0)) g -= dh * p * (lp + h);
        narrow(bad ? nan_of(A()) : empty ? A(0) : g, d_logits[r * d_stride + j]);
    }
}

template <typename T>
int score_impl(const void *logits, long rows, int classes, long stride, Targets targets, int top, void *logp, void *entropy,
               void *top_logp, int *top_index, void *stats, hipStream_t st)
{
    typedef Wide<T> A;
    const ScoreOut<A> o = {(A *)logp, (A *)entropy, (A *)top_logp, (A *)stats, top_index, top};
    launch("log_probs_row", log_probs_row<T>, dim3((unsigned)rows), dim3(256), 0, st, (const T *)logits, classes, stride, targets, o);
    CCNN_LAUNCH_CHECK();
    return 0;
}

template <typename T>
int score_grad_impl(const void *logits, long rows, int classes, long stride, Targets targets, const void *stats,
                    const void *entropy, const void *d_logp, const void *d_entropy, void *d_logits, long d_stride,
                    hipStream_t st)
{
    typedef Wide<T> A;
    launch("log_probs_grad_row", log_probs_grad_row<T>, dim3((unsigned)rows), dim3(256), 0, st, (const T *)logits, classes,
           stride, targets, (const A *)stats, (const A *)entropy, (const A *)d_logp, (const A *)d_entropy, (T *)d_logits,
           d_stride);
    CCNN_LAUNCH_CHECK();
    return 0;
}

int score_args(const void *logits, int type, long rows, int classes, long stride, const void *targets, int target_bytes)
{
    if (!type_bytes(type) || rows < 0 || classes < 1 || stride < classes) return CCNN_E_INVALID;
    if (rows > 0 && (!logits || !targets || (target_bytes != 4 && target_bytes != 8))) return CCNN_E_INVALID;
    if (rows > 0x7fffffffL || classes > CCNN_MAX_LOGITS) return CCNN_E_RANGE;
    return 0;
}

}  // namespace ccnn

using namespace ccnn;

extern "C" {

size_t ccnn_log_probs_workspace_bytes(long rows, int classes, int top, int type)
{
    (void)rows, (void)classes, (void)top, (void)type;
    return 0;
}

int ccnn_log_probs(const void *logits, int type, long rows, int classes, long stride, const void *targets, int target_bytes,
                   int top, void *logp, void *entropy, void *top_logp, int *top_index, void *stats, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (int e = score_args(logits, type, rows, classes, stride, targets, target_bytes)) return e;
    if (top < 0 || top > CCNN_MAX_TOP || top > classes) return CCNN_E_INVALID;
    if (rows == 0) return 0;
    if (!logp || !stats || (top > 0 && (!top_logp || !top_index))) return CCNN_E_INVALID;
    if (workspace_bytes < ccnn_log_probs_workspace_bytes(rows, classes, top, type)) return CCNN_E_WORKSPACE;
    const Targets t = {targets, target_bytes};
    switch (type) {
    case CCNN_TYPE_F32: return score_impl<float>(logits, rows, classes, stride, t, top, logp, entropy, top_logp, top_index, stats, (hipStream_t)stream);
    case CCNN_TYPE_F64: return score_impl<double>(logits, rows, classes, stride, t, top, logp, entropy, top_logp, top_index, stats, (hipStream_t)stream);
    case CCNN_TYPE_BF16: return score_impl<Bf16>(logits, rows, classes, stride, t, top, logp, entropy, top_logp, top_index, stats, (hipStream_t)stream);
    default: return score_impl<F16>(logits, rows, classes, stride, t, top, logp, entropy, top_logp, top_index, stats, (hipStream_t)stream);
    }
}

int ccnn_log_probs_grad(const void *logits, int type, long rows, int classes, long stride, const void *targets,
                        int target_bytes, const void *stats, const void *entropy, const void *d_logp, const void *d_entropy,
                        void *d_logits, long d_stride, void *stream)
{
    if (int e = score_args(logits, type, rows, classes, stride, targets, target_bytes)) return e;
    if (d_stride < classes) return CCNN_E_INVALID;
    if (rows == 0) return 0;
    if (!stats || !d_logits || (!d_logp && !d_entropy) || (d_entropy && !entropy)) return CCNN_E_INVALID;
    if (d_logits == logits && d_stride != stride) return CCNN_E_INVALID;
    const Targets t = {targets, target_bytes};
    switch (type) {
    case CCNN_TYPE_F32: return score_grad_impl<float>(logits, rows, classes, stride, t, stats, entropy, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    case CCNN_TYPE_F64: return score_grad_impl<double>(logits, rows, classes, stride, t, stats, entropy, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    case CCNN_TYPE_BF16: return score_grad_impl<Bf16>(logits, rows, classes, stride, t, stats, entropy, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    default: return score_grad_impl<F16>(logits, rows, classes, stride, t, stats, entropy, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    }
}

}  // extern "C"
