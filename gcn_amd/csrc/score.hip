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
    A *logp, *entropy, *high, *log_sum;   // [rows] each: the rows of stats
    A *top_logp;
    int *top_index;
    int top, want_entropy;
    ScoreOut from(long r) const
    {
        return {logp + r, entropy + r, high + r, log_sum + r, top_logp + r * top, top_index + r * top, top, want_entropy};
    }
};

struct Targets {
    const void *p;
    int bytes;
    __device__ __forceinline__ long at(long r) const
    {
        return bytes == 8 ? (long)((const long long *)p)[r] : (long)((const int *)p)[r];
    }
    Targets from(long r) const { return {(const char *)p + r * bytes, bytes}; }
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

// The largest of several (a NaN is passed over: the sums carry it), and a distance that times 0 is 0.
__device__ __forceinline__ float max_of(float a, float b)
{
    asm("v_max_f32 %0, %1, %2" : "=v"(a) : "v"(a), "v"(b));
    return a;
}
__device__ __forceinline__ double max_of(double a, double b) { return fmax(a, b); }
template <int W>
__device__ __forceinline__ float max_of(const float (&x)[W])
{
    static_assert(W % 2 == 0, "pairs behind the first");
    float m = x[0];
#pragma unroll
    for (int e = 1; e < W - 1; e += 2) asm("v_max3_f32 %0, %1, %2, %3" : "=v"(m) : "v"(m), "v"(x[e]), "v"(x[e + 1]));
    return max_of(m, x[W - 1]);
}
template <int W>
__device__ __forceinline__ double max_of(const double (&x)[W])
{
    double m = x[0];
#pragma unroll
    for (int e = 1; e < W; e++) m = fmax(m, x[e]);
    return m;
}
__device__ __forceinline__ float floor_of(float d) { return fmaxf(d, -1e4f); }
__device__ __forceinline__ double floor_of(double d) { return fmax(d, -1e4); }

// Joined over the wave's lanes, the same in all of them.
template <typename A>
__device__ __forceinline__ Sums<A> over_wave(Sums<A> a)
{
    shift(a, lanes_max<64>(a.m));
    return {a.m, lanes_sum<64>(a.s), lanes_sum<64>(a.t)};
}

template <typename A>
__device__ __forceinline__ void finish_row(const Sums<A> &a, long r, A given, long y, int classes, const ScoreOut<A> &o)
{
    const bool empty = a.m == ninf(A()) && a.s == A(0);
    const A l = empty ? ninf(A()) : logw(a.s), nan = nan_of(A());
    const bool bad = l != l;
    o.high[r] = bad ? nan : a.m;
    o.log_sum[r] = bad ? nan : l;
    o.logp[r] = bad || y >= classes ? nan : y < 0 ? A(0) : empty ? ninf(A()) : (given - a.m) - l;
    if (o.want_entropy) o.entropy[r] = bad ? nan : empty ? A(0) : l - a.t / a.s;
}

// ---------------------------------------------------------------------------- order of the alternatives
// One whole number per element, larger = earlier: the value's order above the index's complement, so
// that equal values (both zeros among them) come in the order of their indices.
template <typename A> struct KeyOf { typedef unsigned long long type; };
template <> struct KeyOf<double> { typedef unsigned __int128 type; };
template <typename A> using Key = typename KeyOf<A>::type;

// A number's order as a signed whole number, above its lowest value.
__device__ __forceinline__ int order_of(float v)
{
    const int u = __float_as_int(v + 0.0f);
    return u ^ ((u >> 31) & 0x7fffffff);
}
__device__ __forceinline__ long long order_of(double v)
{
    const long long u = __double_as_longlong(v + 0.0);
    return u ^ ((u >> 63) & 0x7fffffffffffffffll);
}
__device__ __forceinline__ unsigned long long order_key(int order, unsigned i)
{
    return (unsigned long long)((unsigned)order ^ 0x80000000u) << 32 | (unsigned)~i;
}
__device__ __forceinline__ unsigned __int128 order_key(long long order, unsigned i)
{
    return (unsigned __int128)((unsigned long long)order ^ 0x8000000000000000ull) << 32 | (unsigned)~i;
}
template <typename A>
__device__ __forceinline__ Key<A> key_of(A v, unsigned i)
{
    return order_key(order_of(v), i);
}
__device__ __forceinline__ unsigned key_high(unsigned long long k) { return (unsigned)(k >> 32); }
__device__ __forceinline__ unsigned long long key_high(unsigned __int128 k) { return (unsigned long long)(k >> 32); }
__device__ __forceinline__ unsigned key_index(unsigned long long k) { return ~(unsigned)k; }
__device__ __forceinline__ unsigned key_index(unsigned __int128 k) { return ~(unsigned)k; }
__device__ __forceinline__ float key_value(unsigned long long k)
{
    const int u = (int)(k >> 32);
    return __int_as_float(u ^ (~(u >> 31) | (int)0x80000000));
}
__device__ __forceinline__ double key_value(unsigned __int128 k)
{
    const long long u = (long long)(k >> 32);
    return __longlong_as_double(u ^ (~(u >> 63) | (long long)0x8000000000000000ull));
}
template <typename A>
__device__ __forceinline__ void put_top(const ScoreOut<A> &o, long r, int place, A v, int index, A m, A l)
{
    const bool bad = l != l;
    o.top_index[r * o.top + place] = bad ? -1 : index;
    o.top_logp[r * o.top + place] = bad ? nan_of(A()) : v == ninf(A()) ? v : (v - m) - l;
}

// ---------------------------------------------------------------------------- up to 1024 classes
// G lanes to a row, E elements to a lane, all of them in registers, loaded W at once: element e of lane i is class
// (e / W) G W + i W + e % W.  The sums are one pass over the registers.  Alternatives, with a wave to a row: value
// by value, the largest left, all elements that equal it placed in the order of their classes and struck out.
// With several rows to a wave: one by one, the lane whose best was taken looking for its next - what one row needs
// all rows of the wave wait for, and equal values of one row would be looked for in all (20000 x 1000 bf16, 20
// alternatives: 54 us the first way, 101 the second; 207400 x 13 fp32, 3 alternatives: 11.7 and 8.1).
template <typename T, int G, int E>
__global__ __launch_bounds__(256) void log_probs_small(const T *__restrict__ logits, long rows, int classes, long stride,
                                                       Targets targets, ScoreOut<Wide<T>> o)
{
    typedef Wide<T> A;
    constexpr int FULL = 16 / sizeof(T), W = E < FULL ? E : FULL;
    const int lane = threadIdx.x % G;
    const long r = (long)blockIdx.x * (256 / G) + threadIdx.x / G;
    if (r >= rows) return;               // whole groups leave: the others' exchanges stay among themselves
    const T *row = logits + r * stride;
    auto place_of = [&](int e) { return e / W * (G * W) + lane * W + e % W; };
    A x[E];
#pragma unroll
    for (int c = 0; c < E; c += W) {
        const Pack<T, W> p = load_some<W>(row, place_of(c), classes);
#pragma unroll
        for (int e = 0; e < W; e++) x[c + e] = place_of(c + e) < classes ? (A)widen(p.v[e]) : ninf(A());
    }
    const long y = targets.at(r);
    const A given = lane == 0 && y >= 0 && y < classes ? (A)widen(row[y]) : A(0);
    A m = x[0];
#pragma unroll
    for (int e = 1; e < E; e++) m = x[e] > m ? x[e] : m;
    m = lanes_max<G>(m);
    const A from = m == ninf(A()) ? A(0) : m;
    A s = 0, t = 0;
#pragma unroll
    for (int e = 0; e < E; e++) {
        const A d = x[e] - from, w = expw(d);
        s += w;
        t += w * floor_of(d);       // 0 * inf is not wanted
    }
    const Sums<A> sums = {m, s = lanes_sum<G>(s), t = lanes_sum<G>(t)};
    if (lane == 0) finish_row(sums, r, given, y, classes, o);
    if (o.top == 0) return;
    const A l = m == ninf(A()) && s == A(0) ? ninf(A()) : logw(s);
    if (l != l) {
        for (int k = lane; k < o.top; k += G) put_top(o, r, k, m, -1, m, l);
        return;
    }
    if constexpr (G == 64) {
        const A gone = nan_of(A());             // not equal to, and passed over by the maximum of, anything
#pragma unroll
        for (int e = 0; e < E; e++)
            if (place_of(e) >= classes) x[e] = gone;
        for (int k = 0; k < o.top;) {
            const A high = over_lanes<G>(max_of(x), [](A a, A b) { return max_of(a, b); });
#pragma unroll
            for (int c = 0; c < E; c += W) {
                unsigned long long all[W], any = 0;
#pragma unroll
                for (int e = 0; e < W; e++) any |= all[e] = __ballot(x[c + e] == high);
                if (!any) continue;
                int place = k;
#pragma unroll
                for (int e = 0; e < W; e++) {
                    place += __popcll(all[e] & ((1ull << lane) - 1));     // in the lanes before
                    k += __popcll(all[e]);
                }
#pragma unroll
                for (int e = 0; e < W; e++)
                    if (x[c + e] == high) {
                        if (place < o.top) put_top(o, r, place, high, place_of(c + e), m, l);
                        place++;
                        x[c + e] = gone;
                    }
            }
        }
    } else {
        typedef decltype(order_of(A())) Order;
        const Order gone = sizeof(Order) == 4 ? (Order)0x80000000u : (Order)0x8000000000000000ull;     // below every number
        Order left[E];
#pragma unroll
        for (int e = 0; e < E; e++) left[e] = place_of(e) < classes ? order_of(x[e]) : gone;
        Key<A> best;
        int at;
        auto next = [&]() {                     // the first of the lane's largest elements not taken yet
            Order v = left[0];
            at = 0;
#pragma unroll
            for (int e = 1; e < E; e++)
                if (left[e] > v) v = left[e], at = e;
            best = order_key(v, place_of(at));
        };
        next();
        for (int k = 0; k < o.top; k++) {
            const Key<A> high = lanes_max<G>(best);
            if (lane == 0) put_top(o, r, k, key_value(high), (int)key_index(high), m, l);
            if (best == high && k + 1 < o.top) {
#pragma unroll
                for (int e = 0; e < E; e++) left[e] = e == at ? gone : left[e];
                next();
            }
        }
    }
}

// ---------------------------------------------------------------------------- more classes
// A workgroup streams a slice of a row, 16 bytes a load, once.  Each thread keeps the running sums and its
// largest element with the load it came in.  The k-th largest of 64 groups' largest is a bar that the
// top k elements all reach and few others do; only the threads that hold such an element look at their part
// again, what reaches the bar is collected in LDS and put in order by counting.
// Of 16-bit logits the vector units bound it, busy for 92 % of the CUs' cycles without entropy (8 operations an element and an
// exponential that counts for four) and for 93 % with it (10.5): 4096 x 128000 bf16 in 161 us, 6.5 TB/s, and 2048 x 128000 with
// 5 alternatives in 92 us; x L - c in one multiply-add in place of (x - m) L changes nothing there and costs short rows 8 %.
// Of fp32 it is the memory (63 %): 3001 x 32003 in 65 us, 5.9 TB/s; of fp64 the vector units again (80 %): 1024 x 128000 in 195 us,
// 5.4 TB/s.
// One row of 128000 with 20 alternatives takes 10.9 us, two fifths of it to join the slices; of 61 x 50251 fp16 the alternatives
// are a third of 9.9 us: the bar, what reaches it read again, its order.
constexpr int SLICE_THREADS = 512;   // or 64: see wave_rows
constexpr int CANDIDATES = 1024;      // of the joining workgroup
// The bar is the k-th of the groups up to here: 52 of them are expected to bring 107 elements, enough for the most
// alternatives, and all 64 some 300 or, now and then, far more (2000 x 4096 bf16 with 64: 422 us).  Where it brings too few, k
// is used after all.
constexpr int BAR_RANK = 52;

template <typename A>
struct SliceOut {
    Sums<A> *sums;    // [rows][slices], null: one slice, results go straight to ScoreOut
    Key<A> *keys;     // [rows][slices][top]
    int slices;
    long length;      // elements of a slice (the last may be shorter), a multiple of the load width
};

template <typename A, int NT>
struct SliceLds {
    static constexpr int MOST = NT == 64 ? 512 : 1024;    // candidates
    Key<A> key[NT];
    decltype(key_high(Key<A>())) high[64];
    Key<A> found[MOST];
    A m[NT / 64], s[NT / 64], t[NT / 64];
    Key<A> bar;
    int owners[NT];
    int n_owners, n_found;
};

// k-th largest (k >= 1) of the wave's 64 keys, 0 if fewer are not 0.  Ranked by the values alone, a compare and an add
// each; of the lanes that share the k-th value the one whose index comes next is looked for then.
template <typename K, typename H>
__device__ __forceinline__ K wave_kth(K mine, int k, H *lds)
{
    const int lane = threadIdx.x & 63;
    const H high = key_high(mine);
    lds[lane] = high;
    __builtin_amdgcn_fence(__ATOMIC_ACQ_REL, "workgroup");
    __builtin_amdgcn_wave_barrier();
    int rank = 0;
#pragma unroll
    for (int j = 0; j < 64; j++) rank += lds[j] > high;
    unsigned long long same = 0;
    int r = k;
    while (!same) same = __ballot(rank == --r);         // rank 0 is there
    const unsigned index = key_index(mine);
    for (unsigned long long left = same; left; left &= left - 1) {
        const int one = __ffsll(left) - 1;
        const unsigned at = __builtin_amdgcn_readlane(index, one);
        if (__popcll(same & __ballot(index < at)) == k - 1 - r) {
            const H value = lds[one];
            return value == 0 ? K(0) : (K)value << 32 | (unsigned)~at;
        }
    }
    return K(0);
}

// The first `top` of n keys in LDS, handed to put(place, key) in falling order.
template <typename K, typename Put>
__device__ __forceinline__ void in_order(const K *keys, int n, int top, Put put)
{
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const K mine = keys[i];
        int rank = 0;
        for (int j = 0; j < n; j++) rank += keys[j] > mine;
        if (rank < top) put(rank, mine);
    }
}

// The same from any number of keys, one round over all of them for each place.
template <typename K, typename Get, typename Put>
__device__ __forceinline__ void in_rounds(Get get, int n, int top, K *lds, Put put)
{
    K last = ~K(0);
    for (int k = 0; k < top; k++) {
        K high = 0;
        for (int j = threadIdx.x; j < n; j += blockDim.x) {
            const K w = get(j);
            high = w < last && w > high ? w : high;
        }
        high = lanes_max<64>(high);
        __syncthreads();
        if ((threadIdx.x & 63) == 0) lds[threadIdx.x >> 6] = high;
        __syncthreads();
        high = lds[0];
        for (int w = 1; w < (int)(blockDim.x >> 6); w++) high = lds[w] > high ? lds[w] : high;
        if (threadIdx.x == 0) put(k, high);
        last = high;
    }
}

template <typename T, bool ENTROPY, int NT>
__global__ __launch_bounds__(NT) void log_probs_slice(const T *__restrict__ logits, int classes, long stride, Targets targets,
                                                      ScoreOut<Wide<T>> o, SliceOut<Wide<T>> part)
{
    typedef Wide<T> A;
    constexpr int W = 16 / sizeof(T), U = 4, MOST = SliceLds<A, NT>::MOST;
    __shared__ SliceLds<A, NT> lds;
    const long r = blockIdx.x / part.slices;
    const int slice = blockIdx.x % part.slices, tid = threadIdx.x, lane = tid & 63, wave = tid >> 6;
    const long begin = slice * part.length;
    const int n = (int)min((long)classes - begin, part.length);
    const T *row = logits + r * stride + begin;
    const int loads = n / W;                    // whole loads; what is left of the row is one more, partial one
    long y = -1;
    A given = A(0);
    if (tid == 0 && !part.sums) {               // under way while the row streams
        y = targets.at(r);
        if (y >= 0 && y < classes) given = widen(logits[r * stride + y]);
    }
    // Sums about `from`, which follows the largest element so far at a distance of up to LAG: e^LAG costs the sums
    // nothing, and only a wave that meets a larger element moves them.
    constexpr A LAG = 4;
    A from = 0, limit = ninf(A()), s = 0, t = 0, best = ninf(A());
    int best_at = -1;
    auto take = [&](const A (&x)[W], int at) {
        const A high = max_of(x);
        if (high > best || best_at < 0) best = high, best_at = at;
        if (__any(high > limit)) {
            if (high > limit) {
                const A d = from - high, f = d < A(-1e4) ? A(0) : expw(d);
                if (limit > ninf(A())) t = f > A(0) ? (t + d * s) * f : t * f, s *= f;
                from = high;
                limit = high + LAG;
            }
        }
#pragma unroll
        for (int e = 0; e < W; e++) {
            const A d = x[e] - from, w = expw(d);
            s += w;
            if (ENTROPY) t += w * floor_of(d);       // 0 * inf is not wanted
        }
    };
    int i = tid;
    for (; i + (U - 1) * NT < loads; i += U * NT) {
        Pack<T, W> p[U];
#pragma unroll
        for (int u = 0; u < U; u++) p[u] = load_pack<W>(row + (long)(i + u * NT) * W);
#pragma unroll
        for (int u = 0; u < U; u++) {
            A x[W];
#pragma unroll
            for (int e = 0; e < W; e++) x[e] = widen(p[u].v[e]);
            take(x, i + u * NT);
        }
    }
    for (; i < loads; i += NT) {
        const Pack<T, W> p = load_pack<W>(row + (long)i * W);
        A x[W];
#pragma unroll
        for (int e = 0; e < W; e++) x[e] = widen(p.v[e]);
        take(x, i);
    }
    const int rest = n - loads * W;
    // the last, partial load belongs to the thread whose turn it is
    if (rest > 0 && tid == loads % NT) {
        A x[W];
#pragma unroll
        for (int e = 0; e < W; e++) x[e] = e < rest ? (A)widen(row[(long)loads * W + e]) : ninf(A());
        take(x, loads);
    }

    Sums<A> sums = {limit > ninf(A()) ? from : ninf(A()), s, t};
    shift(sums, best);
    sums = over_wave(sums);
    if (lane == 0) lds.m[wave] = sums.m, lds.s[wave] = sums.s, lds.t[wave] = sums.t;
    if (o.top) lds.key[tid] = best_at < 0 ? Key<A>(0) : key_of(best, best_at);
    if (tid == 0) lds.n_owners = lds.n_found = 0;
    __syncthreads();
    A all = lds.m[0];
#pragma unroll
    for (int w = 1; w < NT / 64; w++) all = lds.m[w] > all ? lds.m[w] : all;
    sums = {all, A(0), A(0)};
#pragma unroll
    for (int w = 0; w < NT / 64; w++) {
        Sums<A> one = {lds.m[w], lds.s[w], lds.t[w]};
        shift(one, all);
        sums.s += one.s;
        sums.t += one.t;
    }
    if (tid == 0) {
        if (part.sums) part.sums[r * part.slices + slice] = sums;
        else finish_row(sums, r, given, y, classes, o);
    }
    if (!o.top) return;
    const A l = sums.m == ninf(A()) && sums.s == A(0) ? ninf(A()) : logw(sums.s);
    if (l != l) {      // a NaN is no number's largest, so what follows may find nothing
        if (!part.sums)                                     // else the row's join says so, from the sums
            for (int place = tid; place < o.top; place += NT) put_top(o, r, place, sums.m, -1, sums.m, l);
        return;
    }
    auto put = [&](int place, Key<A> k) {
        if (part.sums) part.keys[(r * part.slices + slice) * o.top + place] = k;
        else put_top(o, r, place, key_value(k), (int)key_index(k), sums.m, l);
    };
    const int turns = (loads + (rest > 0) + NT - 1) / NT;
    for (int rank = min(o.top, BAR_RANK);; rank = o.top) {
        if (wave == 0) {
            // groups of every 64th thread: what lies together in the row, as in one that is in order, is in different ones
            Key<A> high = lds.key[lane];
#pragma unroll
            for (int w = 1; w < NT / 64; w++) high = lds.key[w * 64 + lane] > high ? lds.key[w * 64 + lane] : high;
            const Key<A> bar = wave_kth(high, rank, lds.high);
            if (lane == 0) lds.bar = bar;
        }
        __syncthreads();
        const Key<A> bar = lds.bar;
        if (best_at >= 0 && key_of(best, best_at) >= bar) lds.owners[atomicAdd(&lds.n_owners, 1)] = tid;
        __syncthreads();
        for (int task = tid; task < lds.n_owners * turns; task += NT) {
            const int at = lds.owners[task / turns] + (task % turns) * NT;
            const int count = at < loads ? W : at == loads ? rest : 0;
            Pack<T, W> p;
            if (count == W) p = load_pack<W>(row + (long)at * W);
            else {
#pragma unroll
                for (int e = 0; e < W; e++)
                    if (e < count) p.v[e] = row[(long)at * W + e];
            }
#pragma unroll
            for (int e = 0; e < W; e++) {
                const A x = widen(p.v[e]);
                if (e < count && key_of(x, at) >= bar) {
                    const int place = atomicAdd(&lds.n_found, 1);
                    if (place < MOST) lds.found[place] = key_of(x, (unsigned)(begin + (long)at * W + e));
                }
            }
        }
        __syncthreads();
        if (lds.n_found >= o.top || rank == o.top) break;
        __syncthreads();
        if (tid == 0) lds.n_owners = lds.n_found = 0;
    }
    if (lds.n_found <= MOST) {
        in_order(lds.found, lds.n_found, o.top, put);
        if (part.sums)     // a last slice shorter than the list: nothing behind its elements
            for (int place = lds.n_found + tid; place < o.top; place += NT) put(place, Key<A>(0));
    } else   // too many elements of a few threads reach the bar: a row ordered on their stride
        in_rounds([&](int j) { return key_of((A)widen(row[j]), (unsigned)(begin + j)); }, n, o.top, lds.key, put);
}

// Joins a row's slices: their sums, and their lists of alternatives through the same bar.
constexpr int JOIN_KEYS = 2048;   // slices x top, see slices_of

template <typename T>
__global__ __launch_bounds__(256) void log_probs_join(const T *__restrict__ logits, int classes, long stride, Targets targets,
                                                      ScoreOut<Wide<T>> o, SliceOut<Wide<T>> part)
{
    typedef Wide<T> A;
    __shared__ Key<A> keys[JOIN_KEYS + CCNN_MAX_TOP], found[CANDIDATES], high_of[4];
    __shared__ decltype(key_high(Key<A>())) order[64];
    __shared__ Key<A> bar;
    __shared__ int n_found;
    const long r = blockIdx.x;
    const int tid = threadIdx.x, lane = tid & 63;
    const int pitch = part.slices | 1, n = pitch * o.top;
    long y = -1;
    A given = A(0);
    if (tid == 0) {
        y = targets.at(r);
        if (y >= 0 && y < classes) given = widen(logits[r * stride + y]);
        n_found = 0;
    }
    // Place by place of all slices, an odd number to a place: among groups of every 64th key both a row's first
    // alternatives and those of one slice, which may be all, are in different ones.
    for (int k = tid; k < n; k += 256) {
        const int place = k / pitch, slice = k - place * pitch;
        keys[k] = slice < part.slices ? part.keys[(r * part.slices + slice) * o.top + place] : Key<A>(0);
    }
    const Sums<A> *in = part.sums + r * part.slices;
    Sums<A> sums = {ninf(A()), A(0), A(0)};
    for (int k = lane; k < part.slices; k += 64) sums = join(sums, in[k]);
    sums = over_wave(sums);
    if (tid == 0) finish_row(sums, r, given, y, classes, o);
    if (!o.top) return;
    const A l = sums.m == ninf(A()) && sums.s == A(0) ? ninf(A()) : logw(sums.s);
    if (l != l) {      // of the slices that hold it there are no keys
        for (int place = tid; place < o.top; place += 256) put_top(o, r, place, sums.m, -1, sums.m, l);
        return;
    }
    __syncthreads();
    if (tid < 64) {
        Key<A> high = 0;
        for (int k = lane; k < n; k += 64) high = keys[k] > high ? keys[k] : high;
        const Key<A> b = n < 64 ? Key<A>(0) : wave_kth(high, o.top, order);
        if (lane == 0) bar = b;
    }
    __syncthreads();
    for (int k = tid; k < n; k += 256)
        if (keys[k] >= bar) {
            const int place = atomicAdd(&n_found, 1);
            if (place < CANDIDATES) found[place] = keys[k];
        }
    __syncthreads();
    auto put = [&](int place, Key<A> k) { put_top(o, r, place, key_value(k), (int)key_index(k), sums.m, l); };
    if (n_found <= CANDIDATES) in_order(found, n_found, o.top, put);
    else in_rounds([&](int j) { return keys[j]; }, n, o.top, high_of, put);
}

// ---------------------------------------------------------------------------- gradient
template <typename A>
struct GradIn {
    const A *entropy, *high, *log_sum, *d_logp, *d_entropy;
    GradIn from(long r) const
    {
        return {entropy + r, high + r, log_sum + r, d_logp ? d_logp + r : nullptr, d_entropy ? d_entropy + r : nullptr};
    }
};

// What one row's elements have in common.
template <typename A>
struct GradRow {
    A m, l, dl, dh, h;
    long y;
    bool empty, bad;
    __device__ GradRow(const GradIn<A> &in, const Targets &targets, long r, int classes)
    {
        y = targets.at(r);
        m = in.high[r], l = in.log_sum[r];
        dl = in.d_logp && y >= 0 ? in.d_logp[r] : A(0);
        dh = in.d_entropy ? in.d_entropy[r] : A(0);
        h = in.d_entropy ? in.entropy[r] : A(0);
        empty = m == ninf(A());
        bad = y >= classes;
    }
    __device__ __forceinline__ A at(A x, long j) const
    {
        const A lp = (x - m) - l, p = expw(lp);
        A g = (y == j ? dl : A(0)) - dl * p;
        if (p > A(0)) g -= dh * p * (lp + h);
        return bad ? nan_of(A()) : empty ? A(0) : g;
    }
};

// A thread to each 16 bytes of a row, rows one after the other: 200000 x 1000 bf16 in 190 us, 4.2 TB/s read and written; 20000 x
// 1000 fp64 in 66 us, 4.9 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void log_probs_grad_packs(const T *logits, unsigned rows, int classes, long stride,
                                                            Targets targets, GradIn<Wide<T>> in, T *d_logits, long d_stride,
                                                            unsigned packs)
{
    typedef Wide<T> A;
    constexpr int W = 16 / sizeof(T);
    const unsigned q = blockIdx.x * 256 + threadIdx.x, r = q / packs;
    const int j = (int)(q - r * packs) * W;
    if (r >= rows) return;
    Pack<T, W> p = load_some<W>(logits + r * stride, j, classes);
    const GradRow<A> row(in, targets, r, classes);
#pragma unroll
    for (int e = 0; e < W; e++) narrow(row.at((A)widen(p.v[e]), j + e), p.v[e]);
    store_some<W>(d_logits + r * d_stride, j, classes, p);
}

constexpr int GRAD_LOADS = 2;   // 1 and 4 are a few per cent slower over 1 GB of logits

// A tile of a row to a workgroup, two loads to a thread, under way while the row's values come.  4096 x 128000 bf16 in 345 us,
// 6.1 TB/s read and written, with the vector units busy for 95 % of the CUs' cycles (19 operations an element): both bounds at
// once.  fp32 is bound by the memory (42 %): 3001 x 32003 in 128 us, 6.0 TB/s; fp64 too (52 %): 1024 x 128000 in 328 us, 6.4 TB/s.
template <typename T>
__global__ __launch_bounds__(256) void log_probs_grad_wide(const T *logits, int classes, long stride, Targets targets,
                                                           GradIn<Wide<T>> in, T *d_logits, long d_stride)
{
    typedef Wide<T> A;
    constexpr int W = 16 / sizeof(T);
    const long r = blockIdx.y;
    const T *x = logits + r * stride;
    T *d = d_logits + r * d_stride;
    const int first = blockIdx.x * (256 * GRAD_LOADS * W) + threadIdx.x * W;
    Pack<T, W> p[GRAD_LOADS];
#pragma unroll
    for (int u = 0; u < GRAD_LOADS; u++) {
        const int j = first + u * 256 * W;
        if (j + W <= classes) p[u] = load_pack<W>(x + j);
    }
    const GradRow<A> row(in, targets, r, classes);
#pragma unroll
    for (int u = 0; u < GRAD_LOADS; u++) {
        const int j = first + u * 256 * W;
        if (j + W <= classes) {
#pragma unroll
            for (int e = 0; e < W; e++) narrow(row.at((A)widen(p[u].v[e]), j + e), p[u].v[e]);
            store_pack<W>(d + j, p[u]);
        } else {
            for (int e = j; e < classes; e++) narrow(row.at((A)widen(x[e]), e), d[e]);
        }
    }
}

// ---------------------------------------------------------------------------- host
constexpr int SMALL_CLASSES = 1024;
constexpr int PACKED_CLASSES = 1024;    // gradient: 16 bytes a thread up to here, tiles of a row beyond (65536 x 2048 bf16:
                                        // 126 and 90 us; 200000 x 200: 43 us, a wave to a row took 96)
constexpr long ROWS_AT_ONCE = 1 << 24, SLICED_AT_ONCE = 1 << 22;   // 64 or 512 threads each stay below a launch's 2^32

// A wave to a row, in place of a workgroup, for short rows if there are enough of them, the more the longer they are: 100000 x
// 1025 bf16 takes 68 us instead of 303, 16384 x 16384 94 instead of 115, 1024 x 4096 with 5 alternatives 7.2 instead of 9.4,
// 1024 x 8192 9.6 instead of 10.4; 512 x 8192 would take 9.3 instead of 7.9, 1024 x 16384 15.4 instead of 12.5, and of fp32
// 1024 x 8192 12.3 instead of 10.3, 3001 x 32003 100 instead of 73.
inline bool wave_rows(long rows, int classes, int size)
{
    return rows >= 512 && classes <= 16384 && (long)classes * size <= 16 * rows;
}

// Slices of a row: one up to UNSPLIT classes, where a workgroup ends with the row before a second launch could join
// slices (one row of 50000 bf16 with 20 alternatives: 9.4 us whole, 10.7 in slices; of 65536: 10.2 and 11.0;
// 61 rows of 50251 fp16: 9.9 and 12.8).  Beyond, enough of them to give every CU two workgroups, none shorter
// than a load per thread, and their lists short enough for the LDS of the workgroup that joins them.
constexpr int UNSPLIT = 65536;

inline int slices_of(long rows, int classes, int top, int size, long *length)
{
    const long width = 16 / size, turn = width * SLICE_THREADS;
    long want = (512 + rows - 1) / rows;
    const long most = (classes + turn - 1) / turn;
    if (want > most) want = most;
    if (top > 0 && want > JOIN_KEYS / top) want = JOIN_KEYS / top;
    if (classes <= UNSPLIT) want = 1;
    if (want < 1) want = 1;
    *length = ((classes + want - 1) / want + width - 1) / width * width;
    return (int)((classes + *length - 1) / *length);
}

template <typename A>
size_t slice_bytes(long rows, int classes, int top, int size)
{
    long length;
    if (classes <= SMALL_CLASSES) return 0;
    const int slices = slices_of(rows, classes, top, size, &length);
    if (slices == 1) return 0;
    return align_up(rows * slices * sizeof(Sums<A>)) + align_up(rows * slices * (size_t)top * sizeof(Key<A>));
}

template <typename T>
int score_impl(const void *logits, long rows, int classes, long stride, Targets targets, int top, int want_entropy,
               void *stats, void *top_logp, int *top_index, void *workspace, hipStream_t st)
{
    typedef Wide<T> A;
    A *s = (A *)stats;
    const ScoreOut<A> o = {s, s + rows, s + 2 * rows, s + 3 * rows, (A *)top_logp, top_index, top, want_entropy};
    const T *x = (const T *)logits;
    if (classes <= SMALL_CLASSES) {
        typedef void (*Kern)(const T *, long, int, long, Targets, ScoreOut<A>);
        // Few lanes to a row while there are rows enough for the device, more where latency counts: 100000 x 50
        // bf16 with 5 alternatives takes 13.8 us with 8 lanes, 30 with 32, 8000 x 50 4.8 and 5.2, 1000 x 50 5.0 and
        // 3.9; 100000 x 250 takes 37.6 us with 16, 68.7 with 64, 8000 x 250 7.0 and 8.6, 1000 x 250 6.9 and 4.4.
        const bool many = rows >= 8192;
        const int group = classes <= 16 ? 2 : classes <= 64 ? (many ? 8 : 32) : classes <= 256 ? (many ? 16 : 64) : 64;
        const Kern kern = classes <= 16    ? log_probs_small<T, 2, 8>
                          : classes <= 64  ? (many ? log_probs_small<T, 8, 8> : log_probs_small<T, 32, 2>)
                          : classes <= 256 ? (many ? log_probs_small<T, 16, 16> : log_probs_small<T, 64, 4>)
                                           : log_probs_small<T, 64, 16>;
        const long per = 256 / group;
        for (long r0 = 0; r0 < rows; r0 += ROWS_AT_ONCE) {
            const long nr = rows - r0 < ROWS_AT_ONCE ? rows - r0 : ROWS_AT_ONCE;
            launch("log_probs_small", kern, dim3((unsigned)((nr + per - 1) / per)), dim3(256), 0, st, x + r0 * stride, nr,
                   classes, stride, targets.from(r0), o.from(r0));
            CCNN_LAUNCH_CHECK();
        }
        return 0;
    }
    SliceOut<A> part = {};
    part.slices = slices_of(rows, classes, top, sizeof(T), &part.length);
    if (part.slices > 1) {
        Carver c(workspace);
        part.sums = c.take<Sums<A>>(rows * part.slices);
        part.keys = c.take<Key<A>>(rows * part.slices * (size_t)top);
    }
    const bool waves = wave_rows(rows, classes, sizeof(T));
    const auto kern = waves ? (want_entropy ? log_probs_slice<T, true, 64> : log_probs_slice<T, false, 64>)
                            : (want_entropy ? log_probs_slice<T, true, SLICE_THREADS> : log_probs_slice<T, false, SLICE_THREADS>);
    const int threads = waves ? 64 : SLICE_THREADS;
    for (long r0 = 0; r0 < rows; r0 += SLICED_AT_ONCE) {
        const long nr = rows - r0 < SLICED_AT_ONCE ? rows - r0 : SLICED_AT_ONCE;
        launch("log_probs_slice", kern, dim3((unsigned)(nr * part.slices)), dim3(threads), 0, st, x + r0 * stride, classes, stride,
               targets.from(r0), o.from(r0), part);
        CCNN_LAUNCH_CHECK();
    }
    if (part.slices > 1) {
        launch("log_probs_join", log_probs_join<T>, dim3((unsigned)rows), dim3(256), 0, st, x, classes, stride, targets, o, part);
        CCNN_LAUNCH_CHECK();
    }
    return 0;
}

template <typename T>
int score_grad_impl(const void *logits, long rows, int classes, long stride, Targets targets, const void *stats,
                    const void *d_logp, const void *d_entropy, void *d_logits, long d_stride,
                    hipStream_t st)
{
    typedef Wide<T> A;
    const T *x = (const T *)logits;
    T *d = (T *)d_logits;
    const A *s = (const A *)stats;
    const GradIn<A> in = {s + rows, s + 2 * rows, s + 3 * rows, (const A *)d_logp, (const A *)d_entropy};
    if (classes <= PACKED_CLASSES) {
        const unsigned packs = (unsigned)((classes * sizeof(T) + 15) / 16);
        const long most = (1L << 31) / packs;             // rows of a launch: their packs are counted in 32 bits
        for (long r0 = 0; r0 < rows; r0 += most) {
            const long nr = rows - r0 < most ? rows - r0 : most;
            launch("log_probs_grad_packs", log_probs_grad_packs<T>, dim3((unsigned)((nr * packs + 255) / 256)), dim3(256), 0, st,
                   x + r0 * stride, (unsigned)nr, classes, stride, targets.from(r0), in.from(r0), d + r0 * d_stride, d_stride,
                   packs);
            CCNN_LAUNCH_CHECK();
        }
        return 0;
    }
    const long tile = 256 * GRAD_LOADS * (16 / sizeof(T));
    for (long r0 = 0; r0 < rows; r0 += 65535) {
        const long nr = rows - r0 < 65535 ? rows - r0 : 65535;
        launch("log_probs_grad_wide", log_probs_grad_wide<T>, dim3((unsigned)((classes + tile - 1) / tile), (unsigned)nr),
               dim3(256), 0, st, x + r0 * stride, classes, stride, targets.from(r0), in.from(r0), d + r0 * d_stride, d_stride);
        CCNN_LAUNCH_CHECK();
    }
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
    if (!type_bytes(type) || rows <= 0 || classes < 1 || top < 0) return 0;
    return type == CCNN_TYPE_F64 ? slice_bytes<double>(rows, classes, top, 8) : slice_bytes<float>(rows, classes, top, type_bytes(type));
}

int ccnn_log_probs(const void *logits, int type, long rows, int classes, long stride, const void *targets, int target_bytes,
                   int top, int want_entropy, void *stats, void *top_logp, int *top_index, void *workspace,
                   size_t workspace_bytes, void *stream)
{
    if (int e = score_args(logits, type, rows, classes, stride, targets, target_bytes)) return e;
    if (top < 0 || top > CCNN_MAX_TOP || top > classes) return CCNN_E_INVALID;
    if (rows == 0) return 0;
    if (!stats || (top > 0 && (!top_logp || !top_index))) return CCNN_E_INVALID;
    const size_t need = ccnn_log_probs_workspace_bytes(rows, classes, top, type);
    if (workspace_bytes < need || (need && !workspace)) return CCNN_E_WORKSPACE;
    const Targets t = {targets, target_bytes};
    switch (type) {
    case CCNN_TYPE_F32: return score_impl<float>(logits, rows, classes, stride, t, top, want_entropy, stats, top_logp, top_index, workspace, (hipStream_t)stream);
    case CCNN_TYPE_F64: return score_impl<double>(logits, rows, classes, stride, t, top, want_entropy, stats, top_logp, top_index, workspace, (hipStream_t)stream);
    case CCNN_TYPE_BF16: return score_impl<Bf16>(logits, rows, classes, stride, t, top, want_entropy, stats, top_logp, top_index, workspace, (hipStream_t)stream);
    default: return score_impl<F16>(logits, rows, classes, stride, t, top, want_entropy, stats, top_logp, top_index, workspace, (hipStream_t)stream);
    }
}

int ccnn_log_probs_grad(const void *logits, int type, long rows, int classes, long stride, const void *targets,
                        int target_bytes, const void *stats, const void *d_logp, const void *d_entropy,
                        void *d_logits, long d_stride, void *stream)
{
    if (int e = score_args(logits, type, rows, classes, stride, targets, target_bytes)) return e;
    if (d_stride < classes) return CCNN_E_INVALID;
    if (rows == 0) return 0;
    if (!stats || !d_logits || (!d_logp && !d_entropy)) return CCNN_E_INVALID;
    if (d_logits == logits && d_stride != stride) return CCNN_E_INVALID;
    const Targets t = {targets, target_bytes};
    switch (type) {
    case CCNN_TYPE_F32: return score_grad_impl<float>(logits, rows, classes, stride, t, stats, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    case CCNN_TYPE_F64: return score_grad_impl<double>(logits, rows, classes, stride, t, stats, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    case CCNN_TYPE_BF16: return score_grad_impl<Bf16>(logits, rows, classes, stride, t, stats, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    default: return score_grad_impl<F16>(logits, rows, classes, stride, t, stats, d_logp, d_entropy, d_logits, d_stride, (hipStream_t)stream);
    }
}

}  // extern "C"
