// The optimiser's two passes over all parameter tensors at once: the gradients' norm and the AdamW step,
// with moments in 32 bits or in 8.  They stand beside the update rules of forward.hip (plain and AdaGrad).
//
// Both read a list of tensors of any sizes in as few launches as possible: the list travels in the
// kernel's arguments, every tensor is cut into chunks, and a workgroup finds its chunk's tensor there.
#include <cmath>
#include <type_traits>

#include "numeric.h"
#include "profile.h"

namespace ccnn {

// Tensors per launch: the argument block stays under 4 KB, and is short where a launch's latency counts (3 KB of
// arguments cost the host 1.8 us more than a few words).
constexpr int NORM_TENSORS = 192, STEP_TENSORS = 64, FEW_TENSORS = 16;
constexpr int BLOCK = CCNN_MOMENT_BLOCK;

// ---------------------------------------------------------------------------- gradient norm
// Squares are summed in fp64, in an order that the sizes alone fix: those of fp32 and 16-bit gradients are exact there and fit, and
// the sum of n of them is off by at most (n / 64 + 40) 2^-53 of itself, a rounding for each addition.  Squares of fp64 gradients
// may not fit: where a sum of theirs shows that, what is beyond 2^480 or below 2^-480 is summed apart, brought near 1 by a
// power of two.  The look costs 47 k fp64 gradients 0.1 us (4.9 of the device), 131 k to 8 M 0.4 (7.5 to 16.2) and 210 M
// nothing (247 us, 6.8 TB/s).
// A wave to a chunk: short ones while they are needed to fill the device, long ones beyond (202 M bf16 gradients: 65 us, 6.2 TB/s;
// 78 with workgroups of 256 to 16 K, 73 with a wave to 16 K).  Just beyond the border the long ones are too few waves: fp32, 31 M
// take 24 us, 36 M 49, 52 M 53, 105 M 70 (6.0 TB/s) and 210 M 127 (6.6); bf16 19, 39, 41, 49 (4.3) and 66 (6.4).
inline long norm_chunk(long total) { return total < (1L << 25) ? 4096 : 32768; }
constexpr int NORM_THREADS = 64;

template <int N>
struct NormList {
    static constexpr int MOST = N;
    const void *data[MOST];
    long n[MOST];
    int chunk0[MOST + 1];   // first chunk of each tensor; [count] = all
    int count;
};

// The tensor of a chunk: how many of the list's first chunks are not behind it, 64 looked at at once (a bisection
// is six loads after each other).
template <typename L>
__device__ __forceinline__ int find(const L &list, int chunk)
{
    int before = -1;
    for (int base = 0; base < list.count; base += 64) {
        const int i = base + (threadIdx.x & 63);
        before += __popcll(__ballot(i < list.count && list.chunk0[i] <= chunk));
    }
    return __builtin_amdgcn_readfirstlane(before);
}

// Sum over a workgroup of N threads in a fixed order; the result is in every thread.
template <int N>
__device__ __forceinline__ double block_sum(double v, double *lds)
{
    v = lanes_sum<64>(v);
    if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = v;
    __syncthreads();
    v = 0;
#pragma unroll
    for (int w = 0; w < N / 64; w++) v += lds[w];
    return v;
}

// Sums of squares: of numbers within 2^480 and 2^-480, of those beyond times 2^-600, of those below times 2^600.
struct Squares {
    double mid = 0, big = 0, tiny = 0;
};
constexpr double FAR = 0x1p480, BACK = 0x1p600;

// A sum of squares that stands for Squares::mid as it is: none was lost then but some below 2^-1022.  So does that of zeros.
__device__ __forceinline__ bool stands(double s) { return s >= 0x1p-900 && s < 0x1p960; }

// Squares of fp64 numbers one by one, those of packs [k, n) of W, `step` apart.
template <int W>
__device__ __forceinline__ void add_apart(Squares &s, const double *p, long k, long n, long step)
{
#pragma unroll 1
    for (; k < n; k += step)
#pragma unroll 1
        for (long j = k; j < min(k + W, n); j++) {
            const double a = fabs(p[j]), b = a * (1 / BACK), t = a * BACK;
            if (a > FAR) s.big += b * b;
            else if (a < 1 / FAR) s.tiny += t * t;
            else s.mid += a * a;
        }
}

template <typename T>
__global__ __launch_bounds__(NORM_THREADS) void norm_partial(NormList<NORM_TENSORS> list, int chunk, double *__restrict__ partial,
                                                             double *__restrict__ apart, long apart_stride)
{
    constexpr int W = 16 / sizeof(T), U = 8, STRIDE = NORM_THREADS * W;
    const int i = find(list, blockIdx.x);
    const long at = (long)(blockIdx.x - list.chunk0[i]) * chunk;
    const T *p = (const T *)list.data[i] + at;
    const int n = (int)min(list.n[i] - at, (long)chunk);
    double sum = 0;
    unsigned high = 0, low = 0;       // bits of any fp64 number: without one they are zeros
    auto add = [&](T x) {
        sum += (double)widen(x) * (double)widen(x);
        if constexpr (sizeof(T) == 8) {
            const unsigned long long b = __double_as_longlong(x);
            high |= (unsigned)(b >> 32), low |= (unsigned)b;
        }
    };
    for (int k = threadIdx.x * W; k < n; k += U * STRIDE) {
        Pack<T, W> x[U];
#pragma unroll
        for (int u = 0; u < U; u++)
            if (k + u * STRIDE + W <= n) x[u] = load_pack<W>(p + k + u * STRIDE);
#pragma unroll
        for (int u = 0; u < U; u++) {
            const int j0 = k + u * STRIDE;
            if (j0 + W <= n) {
#pragma unroll
                for (int e = 0; e < W; e++) add(x[u].v[e]);
            } else {
                for (int j = j0; j < n; j++) add(p[j]);
            }
        }
    }
    if constexpr (sizeof(T) == 8) {
        const bool falls = !stands(sum) && (high << 1 | low) != 0;
        if (__builtin_expect(__any(falls), 0)) {
            Squares s;
            if (falls) add_apart<W>(s, p, threadIdx.x * W, n, STRIDE);
            else s.mid = sum;
            s = {lanes_sum<64>(s.mid), lanes_sum<64>(s.big), lanes_sum<64>(s.tiny)};
            if (threadIdx.x == 0) {                 // a sign: something is apart
                partial[blockIdx.x] = -s.mid;
                apart[blockIdx.x] = s.big, apart[apart_stride + blockIdx.x] = s.tiny;
            }
            return;
        }
    }
    sum = lanes_sum<64>(sum);
    if (threadIdx.x == 0) partial[blockIdx.x] = sum;
}

__device__ __forceinline__ void put_norm(const Squares &s, double max_norm, double *out)
{
    double squares = s.mid, unit = 1;
    if (__builtin_expect(s.big > 0, 0)) squares = s.big + s.mid * (1 / BACK) * (1 / BACK), unit = BACK;
    else if (s.mid == 0) squares = s.tiny, unit = 1 / BACK;
    else squares += s.tiny * (1 / BACK) * (1 / BACK);
    const double norm = sqrt(squares) * unit;
    out[0] = norm;
    out[1] = !(norm < __builtin_huge_val()) ? __builtin_nan("") : norm > max_norm ? max_norm / norm : 1.0;
}

constexpr int TOTAL_THREADS = 1024;

template <bool F64>
__global__ __launch_bounds__(TOTAL_THREADS) void norm_total(const double *__restrict__ partial, int n, const double *__restrict__ apart,
                                                            long apart_stride, double max_norm, double *__restrict__ out)
{
    __shared__ double lds[F64 ? 3 : 1][TOTAL_THREADS / 64];
    Squares s;
    bool any = false;       // a sign in memory or, from wave to wave, in LDS: something is apart
#pragma unroll 4
    for (int k = threadIdx.x; k < n; k += TOTAL_THREADS) {
        const double mid = partial[k];
        s.mid += F64 ? fabs(mid) : mid;
        any |= F64 && signbit(mid);
    }
    if constexpr (F64) {
        s.mid = lanes_sum<64>(s.mid);
        any = __any(any);
        if ((threadIdx.x & 63) == 0) lds[0][threadIdx.x >> 6] = any ? -s.mid : s.mid;
        __syncthreads();
        s.mid = 0;
#pragma unroll
        for (int w = 0; w < TOTAL_THREADS / 64; w++) s.mid += fabs(lds[0][w]), any |= signbit(lds[0][w]);
        if (any) {
            for (int k = threadIdx.x; k < n; k += TOTAL_THREADS)
                if (signbit(partial[k])) s.big += apart[k], s.tiny += apart[apart_stride + k];
            s.big = block_sum<TOTAL_THREADS>(s.big, lds[1]);
            s.tiny = block_sum<TOTAL_THREADS>(s.tiny, lds[2]);
        }
    } else {
        s.mid = block_sum<TOTAL_THREADS>(s.mid, lds[0]);
    }
    if (threadIdx.x == 0) put_norm(s, max_norm, out);
}

// Few gradients, of any types: one workgroup for all of them, each of its waves taking every 16th piece, in place of two
// launches and a workspace.  Its one CU's fp64 conversions and sums bound it: 47 k fp32 gradients take 5.1 us of the device
// and 5.0 a call (two launches: 5.8 and 8.2), 80 k 6.7 and 6.6 (6.0 and 8.2), 130 k 9.5 and 9.4 (6.0 and 8.0).  Pieces of
// 1024 are 3 % slower at 47 k, of 512 17 %.
constexpr long PIECE = 2048, ONE_PIECES = 40;

struct FewList : NormList<FEW_TENSORS> {
    int type[FEW_TENSORS];
};

template <typename T>
__device__ __forceinline__ double piece_squares(const void *data, long at, long n)
{
    constexpr int W = 16 / sizeof(T), U = PIECE / (64 * W);
    Pack<T, W> x[U];
    double s = 0;
#pragma unroll
    for (int u = 0; u < U; u++) x[u] = load_some<W>((const T *)data, at + ((threadIdx.x & 63) + u * 64) * W, n);
#pragma unroll
    for (int u = 0; u < U; u++)
#pragma unroll
        for (int e = 0; e < W; e++) s += (double)widen(x[u].v[e]) * (double)widen(x[u].v[e]);
    return s;
}

// Whether the plain sum of all stands is seen at the end; where it does not, the fp64 pieces are read again.
template <bool F64>
__global__ __launch_bounds__(TOTAL_THREADS) void norm_one(FewList list, double max_norm, double *__restrict__ out)
{
    __shared__ double lds[F64 ? 4 : 1][TOTAL_THREADS / 64];
    Squares s;
    double s64 = 0;
    for (int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); c < list.chunk0[list.count]; c += TOTAL_THREADS / 64) {
        const int i = find(list, c), type = list.type[i];
        const long at = (c - list.chunk0[i]) * PIECE, n = list.n[i];
        if (F64 && type == CCNN_TYPE_F64) s64 += piece_squares<double>(list.data[i], at, n);
        else
            s.mid += type == CCNN_TYPE_F32    ? piece_squares<float>(list.data[i], at, n)
                     : type == CCNN_TYPE_BF16 ? piece_squares<Bf16>(list.data[i], at, n)
                                              : piece_squares<F16>(list.data[i], at, n);
    }
    if constexpr (F64) {
        const double all = block_sum<TOTAL_THREADS>(s.mid + s64, lds[0]);
        if (stands(all)) {
            s.mid = all;
        } else {
            for (int c = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6); c < list.chunk0[list.count]; c += TOTAL_THREADS / 64) {
                const int i = find(list, c);
                const long at = (c - list.chunk0[i]) * PIECE;
                if (list.type[i] == CCNN_TYPE_F64)
                    add_apart<1>(s, (const double *)list.data[i], at + (threadIdx.x & 63), min(at + PIECE, list.n[i]), 64);
            }
            s.mid = block_sum<TOTAL_THREADS>(s.mid, lds[1]);
            s.big = block_sum<TOTAL_THREADS>(s.big, lds[2]);
            s.tiny = block_sum<TOTAL_THREADS>(s.tiny, lds[3]);
        }
    } else {
        s.mid = block_sum<TOTAL_THREADS>(s.mid, lds[0]);
    }
    if (threadIdx.x == 0) put_norm(s, max_norm, out);
}

// ---------------------------------------------------------------------------- AdamW
constexpr long DECODE_CHUNK = 4096;
constexpr int coded_chunk(bool alone) { return (alone ? 4 : 8) * BLOCK; }

template <int N>
struct StepList {
    static constexpr int MOST = N;
    void *param[MOST];
    const void *grad[MOST];
    long n[MOST], first[MOST];
    int block[MOST];
    double decay[MOST];
    int chunk0[MOST + 1];
    int count;
};

struct StepArgs {
    void *m, *v;
    float *m_scale, *v_scale, *master;
    double *clock;
    double beta1, beta2, eps, lr;
    const double *lr_device, *clip;
    bool alone;   // the launch is the whole step, and moves the clock
};

// What a step takes from the clock, for all its elements alike.
struct Tick {
    double t, beta1_t, beta2_t, lr, rate, root, scale;   // steps, powers; lr, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), gradient factor
    bool skip;
    __device__ Tick() {}
    __device__ explicit Tick(const StepArgs &a)
    {
        scale = a.clip ? a.clip[1] : 1.0;
        lr = a.lr_device ? *a.lr_device : a.lr;
        t = a.clock[0] + 1;
        beta1_t = a.clock[1] * a.beta1;
        beta2_t = a.clock[2] * a.beta2;
        rate = lr / (1 - beta1_t);
        root = 1 / sqrt(1 - beta2_t);
        skip = !(fabs(scale) < __builtin_huge_val());
    }
    __device__ void keep(double *clock) const
    {
        clock[0] = t, clock[1] = beta1_t, clock[2] = beta2_t;
    }
};

// clock: t, beta1^t, beta2^t | lr, lr / (1 - beta1^t), 1 / sqrt(1 - beta2^t), gradient factor (NaN: no step) | arrivals,
// of all and of each group
__global__ void adamw_clock(StepArgs a)
{
    const Tick tick(a);
    if (!tick.skip) tick.keep(a.clock);
    a.clock[3] = tick.lr;
    a.clock[4] = tick.rate;
    a.clock[5] = tick.root;
    a.clock[6] = tick.skip ? __builtin_nan("") : tick.scale;
}

// In fp32 the gradient factor is two: one that is no normal number - large gradients clipped to a small norm - would lose
// what the product keeps, or be 0.
// FITS: lr m is within A whatever the moments hold.
template <typename A, bool FITS>
struct Rates {
    A scale, scale2, lr_decay, rate, root, eps;
    bool skip;
    __device__ Rates(double factor, double lr, double decay, double rate, double root, double eps, bool skip)
        : scale((A)factor), scale2(1), lr_decay((A)(lr * decay)), rate((A)rate), root((A)root), eps((A)eps), skip(skip)
    {
        if constexpr (!FITS) {      // lr m may be beyond the type where m is not: the power of two in an lr of 1 or more goes below the line
            const int down = -max(__builtin_amdgcn_frexp_exp(lr), 0);
            this->rate = (A)ldexp(rate, down), this->root = (A)ldexp(root, down);
            this->eps = (A)fmax(ldexp(eps, down), sizeof(A) == 4 ? 0x1p-149 : 0x1p-1074);
        }
        if constexpr (sizeof(A) == 4) {
            const double size = fabs(factor);
            if (size < 0x1p-126) scale = 0x1p-126f, scale2 = (A)(factor * 0x1p126);
            if (size > 0x1p127) scale = 0x1p127f, scale2 = (A)(factor * 0x1p-127);
        }
    }
    __device__ Rates(const StepArgs &a, double decay)
        : Rates(a.clock[6], a.clock[3], decay, a.clock[4], a.clock[5], a.eps, !(a.clock[6] == a.clock[6]))
    {
    }
    __device__ Rates(const StepArgs &a, const Tick &tick, double decay)
        : Rates(tick.scale, tick.lr, decay, tick.rate, tick.root, a.eps, tick.skip)
    {
    }
};

// A launch that is the whole step moves the clock itself: every wave has read it when its workgroup arrives here, the
// last to arrive writes it and leaves the counts at 0.  One count takes an arrival some 7 ns after the one before, so
// beyond a few workgroups they arrive in groups, each counting in a cache line of its own, and then the groups do
// (1 M fp32 parameters in 3907 workgroups: 48 us with one count, 6.9 with 32 groups, 8.3 with 16; 400 k: 4.9 us with 32,
// 5.7 with 128).
constexpr unsigned ARRIVE_AT_ONCE = 64, ARRIVE_GROUPS = 32, ARRIVE_LINE = 16;
static_assert(CCNN_ADAMW_CLOCK == ARRIVE_LINE * (ARRIVE_GROUPS + 1), "a line of the clock, and one for each group");

template <int THREADS>
__device__ __forceinline__ void arrive(const StepArgs &a, const Tick &tick)
{
    if (THREADS > 64) __syncthreads();
    else __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");     // the reads above are done
    if (threadIdx.x != 0) return;
    unsigned *all = reinterpret_cast<unsigned *>(a.clock + 7);
    unsigned parts = gridDim.x;
    if (parts > ARRIVE_AT_ONCE) {
        const unsigned group = blockIdx.x % ARRIVE_GROUPS, members = (gridDim.x - group + ARRIVE_GROUPS - 1) / ARRIVE_GROUPS;
        unsigned *mine = reinterpret_cast<unsigned *>(a.clock + ARRIVE_LINE * (1 + group));
        if (atomicAdd(mine, 1u) != members - 1) return;
        *mine = 0;
        parts = ARRIVE_GROUPS;
    }
    if (atomicAdd(all, 1u) == parts - 1) {
        tick.keep(a.clock);
        *all = 0;
    }
}

template <typename A>
__device__ __forceinline__ A stepped(A p, A m, A v_root, const Rates<A, false> &r)
{
    return p - (r.lr_decay * p + r.rate * m / (v_root * r.root + r.eps));
}

// A wave to a chunk, U packs of four elements in flight per lane.  Bound by the memory: 202 M bf16 parameters with fp32
// master copy and moments (28 bytes each) in 951 us, 5.9 TB/s; with workgroups of 256 4 % slower, with three packs
// 5, with eight 20.
constexpr int WIDE_THREADS = 64;

template <typename P, typename G, int U>
__global__ __launch_bounds__(WIDE_THREADS) void adamw_wide(StepList<U == 1 ? FEW_TENSORS : STEP_TENSORS> list, StepArgs a)
{
    typedef Wide<P> A;
    constexpr bool COPY = sizeof(P) == 2;   // the parameter is the rounding of its master copy
    typedef std::conditional_t<COPY, float, P> S;
    constexpr int W = 4;
    const int i = find(list, blockIdx.x);
    P *param = (P *)list.param[i];
    const G *grad = (const G *)list.grad[i];
    A *m = (A *)a.m + list.first[i], *v = (A *)a.v + list.first[i];
    S *held;
    if constexpr (COPY) held = a.master + list.first[i];
    else held = param;
    const long k0 = (long)(blockIdx.x - list.chunk0[i]) * (U * WIDE_THREADS * W) + threadIdx.x * W, n = list.n[i];
    Pack<A, W> mk[U], vk[U];
    Pack<S, W> pk[U];
    Pack<G, W> gk[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long k = k0 + u * WIDE_THREADS * W;
        gk[u] = load_some<W>(grad, k, n);
        mk[u] = load_some<W>(m, k, n);
        vk[u] = load_some<W>(v, k, n);
        pk[u] = load_some<W>(held, k, n);
    }
    const bool alone = U == 1 || a.alone;
    const Tick tick = alone ? Tick(a) : Tick();
    typedef Rates<A, false> R;
    const R r = alone ? R(a, tick, list.decay[i]) : R(a, list.decay[i]);
    if (r.skip) return;
    const A b1 = (A)(1 - a.beta1), b2 = (A)(1 - a.beta2), twice_b1 = 2 * b1, half2 = A(0.5) * r.scale2;
#pragma unroll
    for (int u = 0; u < U; u++) {
        const long k = k0 + u * WIDE_THREADS * W;
        Pack<P, W> out;
#pragma unroll
        for (int e = 0; e < W; e++) {
            const A x = (A)widen(gk[u].v[e]) * r.scale, g = sizeof(A) == 4 ? x * r.scale2 : x;
            mk[u].v[e] += twice_b1 * (x * half2 - A(0.5) * mk[u].v[e]);     // g - m may be beyond the type, half of it is not
            const A old_v = vk[u].v[e];
            vk[u].v[e] += b2 * (g * g - (old_v == -ninf(A()) ? A(0) : old_v));   // what is beyond the type stays infinite
            pk[u].v[e] = stepped((A)pk[u].v[e], mk[u].v[e], (A)sqrt(vk[u].v[e]), r);
            narrow(pk[u].v[e], out.v[e]);
        }
        store_some<W>(m, k, n, mk[u]);
        store_some<W>(v, k, n, vk[u]);
        if constexpr (COPY) store_some<W>(held, k, n, pk[u]);
        store_some<W>(param, k, n, out);
    }
    if (alone) arrive<WIDE_THREADS>(a, tick);
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

// Four codes of x / scale; positive: no sign, and what v says is above 0 keeps at least the smallest code.  `in` of them, or
// more, are in the tensor: of a scale that is NaN all codes are, but for those behind its end, which stay 0.
template <bool POSITIVE>
__device__ __forceinline__ unsigned exact_codes(const double (&x)[4], const double (&v)[4], float scale, long in)
{
    if (scale == 0) return 0;
    unsigned w = 0;
#pragma unroll
    for (int e = 0; e < 4; e++) {
        const double y = fabs(x[e]) / scale;
        unsigned c = y == y ? encode8(fmin(y, 448.0)) : 0x7fu;
        if (POSITIVE && c == 0 && v[e] > 0) c = 1;
        if (!POSITIVE && x[e] < 0) c |= 0x80;
        w |= c << (8 * e);
    }
    if (scale != scale && in < 4) w &= in > 0 ? (1u << (8 * in)) - 1 : 0;
    return w;
}

// The same, for all but a few in a hundred blocks: y in fp32 is within 2^-21.5 of itself (three roundings and a
// reciprocal), so where 2^-21 less and 2^-21 more give the same codes, no border lies between it and the
// exact quotient.  Blocks with an undecided element or a root to be kept above 0, and scales outside the range
// where that holds, go the way above.
template <bool POSITIVE>
__device__ __forceinline__ unsigned codes(const double (&x)[4], const double (&v)[4], const float (&x32)[4], float scale, long in)
{
    const float inv = __builtin_amdgcn_rcpf(scale), more = inv * (1.0f + 0x1p-21f), less = inv * (1.0f - 0x1p-21f);
    unsigned up = 0, down = 0;
    up = __builtin_amdgcn_cvt_pk_fp8_f32(x32[0] * more, x32[1] * more, up, false);
    up = __builtin_amdgcn_cvt_pk_fp8_f32(x32[2] * more, x32[3] * more, up, true);
    down = __builtin_amdgcn_cvt_pk_fp8_f32(x32[0] * less, x32[1] * less, down, false);
    down = __builtin_amdgcn_cvt_pk_fp8_f32(x32[2] * less, x32[3] * less, down, true);
    bool open = up != down;
    if (POSITIVE) open |= ((down - 0x01010101u) & ~down & 0x80808080u) != 0;     // a byte of 0
    if (!(scale > 1e-30f && scale < 1e30f) || __any(open)) return exact_codes<POSITIVE>(x, v, scale, in);
    return up;
}

// beta old + (1 - beta) new, every product and the sum rounded by itself.  With a beta like 9/10 the result
// often lies exactly between two fp32 values, so a block's fp32 scale would hang on how the compiler
// contracts the expression.
__device__ __forceinline__ double decay_to(double beta, double rest, double old, double now)
{
#pragma clang fp contract(off)
    const double a = beta * old, b = rest * now;
    return a + b;
}

// sqrt to the last bit or two: the hardware's 2^-24 start and two corrections.  0 gives 1e-150, which no fp32 and
// no step can tell from it (but 1 / sqrt(0) * 0 could not be corrected).
__device__ __forceinline__ double root64(double v)
{
    v += 1e-300;
    const double y = __builtin_amdgcn_rsq(v), h = 0.5 * y;
    double s = v * y;
    s = fma(fma(-s, s, v), h, s);
    return fma(fma(-s, s, v), h, s);
}

// h / 448, correctly rounded: of every fp32 from 1e-30 on the product with RN(1/448) is corrected to it by its
// residual, below the quotient may be subnormal.
__device__ __forceinline__ float scale_of(float h)
{
    constexpr float INV = 1.0f / 448.0f;
    if (h < 1e-30f) return h / 448.0f;
    const float q = h * INV;
    return fmaf(fmaf(-448.0f, q, h), INV, q);
}

// One wave per block of 256 elements, four to a lane, two blocks in flight (one costs 6 % at 100 M parameters, four
// 2 %; a small step has one, 100 k bf16 parameters in 5.3 us instead of 6.1).  Moments, root and step in fp64, so that codes,
// scales and steps are those of the definition whatever the order of operations.  101 M bf16 parameters with fp32 master copy (16 bytes each) in 297 us, 5.4 TB/s; the vector
// units are busy for 84 % of the CUs' cycles meanwhile (561 operations a wave for two blocks), so that both bound it.
template <typename P, typename G, bool ALONE>
__global__ __launch_bounds__(256) void adamw_coded(StepList<STEP_TENSORS> list, StepArgs a)
{
    constexpr bool COPY = sizeof(P) == 2;
    typedef std::conditional_t<COPY, float, P> S;
    constexpr int U = ALONE ? 1 : 2, CHUNK = coded_chunk(ALONE);
    const int i = find(list, blockIdx.x);
    P *param = (P *)list.param[i];
    const G *grad = (const G *)list.grad[i];
    S *held;
    if constexpr (COPY) held = a.master + list.first[i];
    else held = param;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const long n = list.n[i], b0 = (long)(blockIdx.x - list.chunk0[i]) * CHUNK + wave * (U * BLOCK);
    const long blk0 = list.block[i] + b0 / BLOCK;
    const double rest1 = 1 - a.beta1, rest2 = 1 - a.beta2;
    Pack<G, 4> gk[U];
    Pack<S, 4> pk[U];
    unsigned mc[U], vc[U];
    float ms[U], vs[U];
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (b0 + u * BLOCK >= n) break;
        const long k = b0 + u * BLOCK + lane * 4;
        gk[u] = load_some<4>(grad, k, n);
        pk[u] = load_some<4>(held, k, n);
        mc[u] = ((const unsigned *)a.m)[(blk0 + u) * (BLOCK / 4) + lane];
        vc[u] = ((const unsigned *)a.v)[(blk0 + u) * (BLOCK / 4) + lane];
        ms[u] = a.m_scale[blk0 + u];
        vs[u] = a.v_scale[blk0 + u];
    }
    const Tick tick = ALONE ? Tick(a) : Tick();
    typedef Rates<double, true> R;
    const R r = ALONE ? R(a, tick, list.decay[i]) : R(a, list.decay[i]);
    if (r.skip) return;
#pragma unroll
    for (int u = 0; u < U; u++) {
        if (b0 + u * BLOCK >= n) break;
        const long k = b0 + u * BLOCK + lane * 4;
        double m[4], v[4], root[4];
        float m32[4], root32[4];
        Pack<P, 4> out;
        const auto m01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], false), m23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)mc[u], true);
        const auto v01 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[u], false), v23 = __builtin_amdgcn_cvt_pk_f32_fp8((int)vc[u], true);
        const float old_m[4] = {m01[0], m01[1], m23[0], m23[1]}, old_v[4] = {v01[0], v01[1], v23[0], v23[1]};
#pragma unroll
        for (int e = 0; e < 4; e++) {
            const double g = (double)widen(gk[u].v[e]) * r.scale, vo = (double)old_v[e] * (double)vs[u];
            m[e] = decay_to(a.beta1, rest1, (double)old_m[e] * (double)ms[u], g);
            v[e] = decay_to(a.beta2, rest2, vo * vo, g * g);
            root[e] = root64(v[e]);
            m32[e] = (float)m[e];
            root32[e] = (float)root[e];
            const double d = fma(root[e], r.root, r.eps);
            double x = __builtin_amdgcn_rcp(d);
            x = fma(fma(-d, x, 1.0), x, x);
            const double p = pk[u].v[e];
            pk[u].v[e] = (float)(p - fma(r.lr_decay, p, r.rate * m[e] * x));
            narrow(pk[u].v[e], out.v[e]);
        }
        if constexpr (COPY) store_some<4>(held, k, n, pk[u]);
        store_some<4>(param, k, n, out);
        // the block's largest magnitudes; what is not finite is so in both moments, and its bits are above all others'
        const unsigned high_m = lanes_max<64>(__float_as_uint(fmaxf(fmaxf(fabsf(m32[0]), fabsf(m32[1])), fmaxf(fabsf(m32[2]), fabsf(m32[3])))));
        const unsigned high_v = lanes_max<64>(max(max(__float_as_uint(root32[0]), __float_as_uint(root32[1])), max(__float_as_uint(root32[2]), __float_as_uint(root32[3]))));
        const bool lost = high_v >= 0x7f800000u || high_m >= 0x7f800000u;
        const float sm = lost ? __builtin_nanf("") : scale_of(__uint_as_float(high_m));
        const float sv = lost ? __builtin_nanf("") : scale_of(__uint_as_float(high_v));
        ((unsigned *)a.m)[(blk0 + u) * (BLOCK / 4) + lane] = codes<false>(m, v, m32, sm, n - k);
        ((unsigned *)a.v)[(blk0 + u) * (BLOCK / 4) + lane] = codes<true>(root, v, root32, sv, n - k);
        if (lane == 0) a.m_scale[blk0 + u] = sm, a.v_scale[blk0 + u] = sv;
    }
    if (ALONE) arrive<256>(a, tick);
}

// 8-bit moments read out: 101 M of each in 142 us, 7.1 TB/s, four fifths of it written.
__global__ __launch_bounds__(256) void adamw_decode(StepList<STEP_TENSORS> list, const unsigned *__restrict__ m, const unsigned *__restrict__ v,
                                                    const float *__restrict__ m_scale, const float *__restrict__ v_scale,
                                                    float *__restrict__ m_out, float *__restrict__ v_out)
{
    constexpr int U = DECODE_CHUNK / (4 * 256);
    const int i = find(list, blockIdx.x);
    const long n = list.n[i], k0 = (long)(blockIdx.x - list.chunk0[i]) * DECODE_CHUNK + threadIdx.x * 4;
    const long at0 = (long)list.block[i] * BLOCK + k0;
    unsigned mc[U], vc[U];
    float ms[U], vs[U];
#pragma unroll
    for (int u = 0; u < U; u++)
        if (k0 + u * 1024 < n) {
            const long at = at0 + u * 1024;
            mc[u] = m[at / 4], vc[u] = v[at / 4];
            ms[u] = m_scale[at / BLOCK], vs[u] = v_scale[at / BLOCK];
        }
#pragma unroll
    for (int u = 0; u < U; u++)
        if (k0 + u * 1024 < n) {
            Pack<float, 4> mo, vo;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                const double root = (double)decode8((vc[u] >> (8 * e)) & 255) * vs[u];
                mo.v[e] = (float)((double)decode8((mc[u] >> (8 * e)) & 255) * ms[u]);
                vo.v[e] = (float)(root * root);
            }
            store_some<4>(m_out + list.first[i], k0 + u * 1024, n, mo);
            store_some<4>(v_out + list.first[i], k0 + u * 1024, n, vo);
        }
}

// ---------------------------------------------------------------------------- host
// A step of one pair of types is one launch that moves the clock itself.  Of few tensors and up to WIDE_SMALL elements it has
// one pack a lane and a short argument block: fp32, 47 k in 4.9 us of the device and 1 M in 6.9 (four packs 6.2 and 8.3,
// the clock in a launch of its own 7.2 and 8.9), 4 M in 21.2 (four packs 20.2).  With 8-bit moments working out the
// step's rates in every wave pays up to ALONE_CODED: bf16, 1 M in 7.2 us instead of 8.8, 4.3 M in 18.7 either way, 8 M
// in 30 instead of 28.5.
constexpr long WIDE_SMALL = 1 << 20, ALONE_CODED = 5 << 20;

// Hands tensors [0, count) that `take` accepts to `go`, a list at a time, with their chunks counted.
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
        const bool full = list.count == List::MOST || (list.count > 0 && list.chunk0[list.count] + chunks > 0x7fffffffL);
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

inline long sum_of(const long *n, int count)
{
    long total = 0;
    for (int i = 0; i < count; i++)
        if (n[i] > 0) total += n[i];
    return total;
}

inline bool norm_in_one(const long *n, int count)
{
    if (count > FEW_TENSORS) return false;
    long pieces = 0;
    for (int i = 0; i < count && pieces <= ONE_PIECES; i++)
        if (n[i] > 0) pieces += n[i] / PIECE + (n[i] % PIECE != 0);
    return pieces <= ONE_PIECES;
}

}  // namespace ccnn

using namespace ccnn;

extern "C" {

size_t ccnn_grad_norm_workspace_bytes(const long *n, int count)
{
    if (!n || count < 0 || norm_in_one(n, count)) return 0;
    const long chunk = norm_chunk(sum_of(n, count));
    size_t chunks = 1;
    for (int i = 0; i < count; i++)
        if (n[i] > 0) chunks += (size_t)(n[i] / chunk + (n[i] % chunk != 0));
    return chunks * sizeof(Squares);
}

int ccnn_grad_norm(const void *const *data, const long *n, const int *types, int count, double max_norm, double *out,
                   void *workspace, size_t workspace_bytes, void *stream)
{
    if (count < 0 || (count > 0 && (!data || !n || !types)) || !out || !(max_norm > 0)) return CCNN_E_INVALID;
    bool used[CCNN_TYPE_F16 + 1] = {};
    for (int i = 0; i < count; i++) {
        if (!type_bytes(types[i]) || n[i] < 0 || (n[i] > 0 && !data[i])) return CCNN_E_INVALID;
        used[types[i]] = true;
    }
    const size_t need = ccnn_grad_norm_workspace_bytes(n, count);
    if (need / sizeof(Squares) > 0x7fffffffu) return CCNN_E_RANGE;
    if (workspace_bytes < need || (need && !workspace)) return CCNN_E_WORKSPACE;
    hipStream_t st = (hipStream_t)stream;
    if (norm_in_one(n, count)) {
        FewList list;
        list.count = list.chunk0[0] = 0;
        for (int i = 0; i < count; i++) {
            if (n[i] == 0) continue;
            const int c = list.count++;
            list.data[c] = data[i];
            list.n[c] = n[i];
            list.type[c] = types[i];
            list.chunk0[c + 1] = list.chunk0[c] + (int)((n[i] + PIECE - 1) / PIECE);
        }
        launch("norm_one", used[CCNN_TYPE_F64] ? norm_one<true> : norm_one<false>, dim3(1), dim3(TOTAL_THREADS), 0, st, list, max_norm, out);
        CCNN_LAUNCH_CHECK();
        return 0;
    }
    const long apart_stride = (long)(need / sizeof(Squares));
    double *partial = (double *)workspace, *apart = partial + apart_stride;
    const long chunk = norm_chunk(sum_of(n, count));
    int done = 0;
    auto take = [&](auto &list, int i, int type) -> long {
        if (types[i] != type) return 0;
        if (list.count < list.MOST) {
            list.data[list.count] = data[i];
            list.n[list.count] = n[i];
        }
        return n[i];
    };
    for (int type = CCNN_TYPE_F32; type <= CCNN_TYPE_F16; type++) {
        if (!used[type]) continue;
        typedef NormList<NORM_TENSORS> List;
        const int e = in_lists<List>(
            count, chunk, [&](List &list, int i) { return take(list, i, type); },
            [&](const List &list) -> int {
                const int chunks = list.chunk0[list.count];
                launch("norm_partial", type == CCNN_TYPE_F32    ? norm_partial<float>
                                       : type == CCNN_TYPE_F64  ? norm_partial<double>
                                       : type == CCNN_TYPE_BF16 ? norm_partial<Bf16>
                                                                : norm_partial<F16>,
                       dim3((unsigned)chunks), dim3(NORM_THREADS), 0, st, list, (int)chunk, partial + done, apart + done, apart_stride);
                CCNN_LAUNCH_CHECK();
                done += chunks;
                return 0;
            });
        if (e) return e;
    }
    launch("norm_total", used[CCNN_TYPE_F64] ? norm_total<true> : norm_total<false>, dim3(1), dim3(TOTAL_THREADS), 0, st, partial, done, apart, apart_stride,
           max_norm, out);
    CCNN_LAUNCH_CHECK();
    return 0;
}

int ccnn_adamw_step(const ccnn_adamw_tensor_t *tensors, const void *const *grads, const int *grad_types, int count,
                    int moment_bits, void *m, void *v, float *m_scale, float *v_scale, float *master, double *clock, double lr,
                    const double *lr_device, double beta1, double beta2, double eps, const double *clip, void *stream)
{
    if (count < 0 || (count > 0 && (!tensors || !grads || !grad_types)) || !clock) return CCNN_E_INVALID;
    if (moment_bits != 32 && moment_bits != 8) return CCNN_E_INVALID;
    if (!(beta1 >= 0 && beta1 < 1) || !(beta2 >= 0 && beta2 < 1) || !(eps > 0)) return CCNN_E_INVALID;
    bool wide = false, other = false;
    long total = 0;
    for (int i = 0; i < count; i++) {
        const ccnn_adamw_tensor_t &t = tensors[i];
        const bool half = t.type == CCNN_TYPE_BF16 || t.type == CCNN_TYPE_F16;
        if (!type_bytes(t.type) || (grad_types[i] != t.type && !(half && grad_types[i] == CCNN_TYPE_F32))) return CCNN_E_INVALID;
        if (t.n < 0 || (t.n > 0 && (!t.param || !grads[i] || t.first < 0 || t.block < 0))) return CCNN_E_INVALID;
        if (moment_bits == 8 && t.block > 0x7fffffffL) return CCNN_E_RANGE;
        if (half && t.n > 0 && !master) return CCNN_E_INVALID;
        (t.type == CCNN_TYPE_F64 ? wide : other) = true;
        total += t.n;
    }
    if (wide && (other || moment_bits == 8)) return CCNN_E_INVALID;
    if (other && !((float)eps > 0)) return CCNN_E_INVALID;     // without a gradient yet the quotient would be 0 / 0
    if (total > 0 && (!m || !v || (moment_bits == 8 && (!m_scale || !v_scale)))) return CCNN_E_INVALID;
    hipStream_t st = (hipStream_t)stream;
    StepArgs args = {m, v, m_scale, v_scale, master, clock, beta1, beta2, eps, lr, lr_device, clip, false};
    typedef StepList<FEW_TENSORS> Few;
    typedef StepList<STEP_TENSORS> Many;
    const struct {
        int type, grad_type;
        void (*one)(Few, StepArgs);
        void (*four)(Many, StepArgs);
        void (*coded)(Many, StepArgs), (*coded_alone)(Many, StepArgs);
    } kinds[] = {
        {CCNN_TYPE_F32, CCNN_TYPE_F32, adamw_wide<float, float, 1>, adamw_wide<float, float, 4>, adamw_coded<float, float, false>, adamw_coded<float, float, true>},
        {CCNN_TYPE_F64, CCNN_TYPE_F64, adamw_wide<double, double, 1>, adamw_wide<double, double, 4>, nullptr, nullptr},
        {CCNN_TYPE_BF16, CCNN_TYPE_BF16, adamw_wide<Bf16, Bf16, 1>, adamw_wide<Bf16, Bf16, 4>, adamw_coded<Bf16, Bf16, false>, adamw_coded<Bf16, Bf16, true>},
        {CCNN_TYPE_BF16, CCNN_TYPE_F32, adamw_wide<Bf16, float, 1>, adamw_wide<Bf16, float, 4>, adamw_coded<Bf16, float, false>, adamw_coded<Bf16, float, true>},
        {CCNN_TYPE_F16, CCNN_TYPE_F16, adamw_wide<F16, F16, 1>, adamw_wide<F16, F16, 4>, adamw_coded<F16, F16, false>, adamw_coded<F16, F16, true>},
        {CCNN_TYPE_F16, CCNN_TYPE_F32, adamw_wide<F16, float, 1>, adamw_wide<F16, float, 4>, adamw_coded<F16, float, false>, adamw_coded<F16, float, true>},
    };
    bool alike = true;
    for (int i = 1; i < count; i++) alike &= tensors[i].type == tensors[0].type && grad_types[i] == grad_types[0];
    args.alone = alike && total > 0 && count <= STEP_TENSORS && (moment_bits == 32 || total < ALONE_CODED);
    const bool small = args.alone && moment_bits == 32 && total < WIDE_SMALL && count <= FEW_TENSORS;
    if (!args.alone) {
        launch("adamw_clock", adamw_clock, dim3(1), dim3(1), 0, st, args);
        CCNN_LAUNCH_CHECK();
    }
    for (const auto &kind : kinds) {
        auto take = [&](auto &list, int i) -> long {
            const ccnn_adamw_tensor_t &t = tensors[i];
            if (t.type != kind.type || grad_types[i] != kind.grad_type) return 0;
            if (const int c = list.count; c < list.MOST) {
                list.param[c] = t.param;
                list.grad[c] = grads[i];
                list.n[c] = t.n;
                list.first[c] = t.first;
                list.block[c] = (int)t.block;
                list.decay[c] = t.decay;
            }
            return t.n;
        };
        int e;
        if (small)
            e = in_lists<Few>(count, WIDE_THREADS * 4, take, [&](const Few &list) -> int {
                launch("adamw_wide", kind.one, dim3((unsigned)list.chunk0[list.count]), dim3(WIDE_THREADS), 0, st, list, args);
                CCNN_LAUNCH_CHECK();
                return 0;
            });
        else
            e = in_lists<Many>(count, moment_bits == 8 ? coded_chunk(args.alone) : WIDE_THREADS * 16, take, [&](const Many &list) -> int {
                launch(moment_bits == 8 ? "adamw_coded" : "adamw_wide", moment_bits == 32 ? kind.four : args.alone ? kind.coded_alone : kind.coded,
                       dim3((unsigned)list.chunk0[list.count]), dim3(moment_bits == 8 ? 256 : WIDE_THREADS), 0, st, list, args);
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
    typedef StepList<STEP_TENSORS> List;
    return in_lists<List>(
        count, DECODE_CHUNK,
        [&](List &list, int i) -> long {
            if (const int c = list.count; c < list.MOST) {
                list.n[c] = tensors[i].n;
                list.first[c] = tensors[i].first;
                list.block[c] = (int)tensors[i].block;
            }
            return tensors[i].n;
        },
        [&](const List &list) -> int {
            launch("adamw_decode", adamw_decode, dim3((unsigned)list.chunk0[list.count]), dim3(256), 0, (hipStream_t)stream,
                   list, (const unsigned *)m, (const unsigned *)v, m_scale, v_scale, m_out, v_out);
            CCNN_LAUNCH_CHECK();
            return 0;
        });
}

}  // extern "C"
