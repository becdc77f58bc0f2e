// Losses of a softmax policy over a catalogue's scores, with their gradient: preferences between lists, and the clipped policy
// loss with a KL term.
//
//   log p[t][j] = scale (s[t][j] - m_t) - log l_t,   m_t = max_j s[t][j],   l_t = sum_j exp(scale (s[t][j] - m_t))
//   dscores[t][j] = scale c_t (1[j = item_t] - p[t][j]),   c_t = d(weighted loss) / d(log p of row t's item)
//
// One exp and a few flop per score: bound by memory.  A block reads a row (or, where rows are few, a part of one) once, with
// the running maximum and sum in registers; a row's parts are joined by whoever needs the row's loss.  Everything that is one number
// per row is computed in 64 bits - a list's log-ratio is a small difference of sums of log-probabilities - and
// rounded once when it is stored.
#include "operators.h"
#include <float.h>

namespace {

struct LossArgs {
    const void* scores;
    const int32_t* item;
    const int64_t* off;                       // preference only
    const float *ref_logp, *old_logp, *advantage, *grad_weight;
    float *loss, *margin, *kl, *logp;
    void* dscores;
    float4* part;                             // [rows][splits] statistics of a row's parts
    float2* stat;                             // [rows] (maximum, sum) of a row
    float* coef;                              // [rows] c_t, 0 where a row takes no part
    int64_t rows, n_items, scores_stride, dscores_stride;
    float scale, scale2;                      // scale2 = scale * log2(e), rounded
    double scale_rest;                        // scale - scale2 / log2(e)
    int n_seq, splits, zero_rest;
    double beta, smoothing, clip_low, clip_high, kl_coef;
};

// What is known of a set of scores: its maximum m, l = sum of 2^(c (x - m)), c being scale * log2(e) rounded to f32, and of a
// sample of it ls = sum of 2^(c (x - m)) and qs = sum of (x - m) 2^(c (x - m)).  The rounding of c is the same for every score: it would
// move log l of all rows the same way (by 6e-8 for scores of deviation 2), and the log-ratio of lists of different lengths by
// that times their difference.  qs / ls, the derivative of log l by c, takes it out again; one score of each 16 bytes is
// sample enough for a factor of a rounding.  (Where a few scores that are not in the sample hold nearly all of l, the mean is near
// 0 and the sample's own is not: it counts for no more than its share of l.)  m is -inf for a set with nothing in it.
struct Stat { float m, l, ls, qs; };

__device__ __forceinline__ Stat join(Stat a, Stat b, float c)
{
    const float m = fmaxf(a.m, b.m), base = m == -INFINITY ? 0.0f : m;
    // a set without a finite maximum has sums of 0, or NaN
    const float da = a.m == -INFINITY ? 0.0f : a.m - base, db = b.m == -INFINITY ? 0.0f : b.m - base;
    const float fa = fast_exp2(da * c), fb = fast_exp2(db * c);
    return {m, a.l * fa + b.l * fb, a.ls * fa + b.ls * fb, (fa > 0.0f ? fmaf(da, a.ls, a.qs) * fa : 0.0f) + (fb > 0.0f ? fmaf(db, b.ls, b.qs) * fb : 0.0f)};
}

// over a wavefront, in every lane: everyone moves to the common maximum first, so that plain sums are left
__device__ __forceinline__ Stat join_lanes(Stat st, float c)
{
    const float m = wave_max(st.m), base = m == -INFINITY ? 0.0f : m, d = st.m == -INFINITY ? 0.0f : st.m - base, f = fast_exp2(d * c);
    return {m, group_sum_dpp<64>(st.l * f), group_sum_dpp<64>(st.ls * f), group_sum_dpp<64>(f > 0.0f ? fmaf(d, st.ls, st.qs) * f : 0.0f)};
}

// N vectors of V scores into a thread's statistics
template <int V, int N>
__device__ __forceinline__ void add_scores(Stat& st, const float (&x)[N][V], float c)
{
    float m = x[0][0];
#pragma unroll
    for (int n = 0; n < N; n++)
#pragma unroll
        for (int v = 0; v < V; v++) m = fmaxf(m, x[n][v]);
    if (m > st.m) {   // rarely, after the first few
        const float d = st.m == -INFINITY ? 0.0f : st.m - m, f = fast_exp2(d * c);
        st.qs = f > 0.0f ? fmaf(d, st.ls, st.qs) * f : 0.0f;
        st.ls *= f;
        st.l *= f;
        st.m = m;
    }
    const float base = st.m == -INFINITY ? 0.0f : st.m;
#pragma unroll
    for (int n = 0; n < N; n++) {
        float l = 0.0f;
#pragma unroll
        for (int v = 0; v < V; v++) {
            const float d = x[n][v] - base, e = fast_exp2(d * c);
            l += e;
            if (v == 0) {
                st.ls += e;
                st.qs = fmaf(fmaxf(d, -FLT_MAX), e, st.qs);   // a masked score adds 0, not -inf * 0
            }
        }
        st.l += l;
    }
}

template <class T, int V> __device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&x)[V])
{
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = to_f32(p.v[v]);
}

// Where a row's 16-byte vectors begin and how many there are; what is in front and behind is taken singly
struct Vectors { int64_t lead, n, tail; };
template <class T> __device__ __forceinline__ Vectors vectors_of(const T* row, int64_t j0, int64_t j1)
{
    constexpr int V = 16 / sizeof(T);
    const int64_t a0 = j0 + (int64_t)(((16 - ((uintptr_t)(row + j0) & 15)) & 15) / sizeof(T));
    Vectors r;
    r.lead = a0 < j1 ? a0 : j1;
    r.n = (j1 - r.lead) / V;
    r.tail = r.lead + r.n * V;
    return r;
}

// what thread `tid` of `step` finds in the scores [j0, j1) of a row.  NaN scores give a NaN sum.
template <class T>
__device__ __forceinline__ Stat thread_statistics(const T* __restrict__ row, int64_t j0, int64_t j1, float c, int tid, int step)
{
    constexpr int V = 16 / sizeof(T), N = 4;   // four loads in flight per thread
    Stat st = {-INFINITY, 0.0f, 0.0f, 0.0f};
    const Vectors w = vectors_of(row, j0, j1);
    const Pack<T, V>* p = reinterpret_cast<const Pack<T, V>*>(row + w.lead);
    int64_t i = tid;
    for (; i + (N - 1) * step < w.n; i += N * step) {
        Pack<T, V> raw[N];
#pragma unroll
        for (int n = 0; n < N; n++) raw[n] = p[i + n * step];
        float x[N][V];
#pragma unroll
        for (int n = 0; n < N; n++) unpack<T, V>(raw[n], x[n]);
        add_scores<V, N>(st, x, c);
    }
    for (; i < w.n; i += step) {
        float x[1][V];
        unpack<T, V>(p[i], x[0]);
        add_scores<V, 1>(st, x, c);
    }
    const int64_t n = (w.lead - j0) + (j1 - w.tail);   // at most 2 V - 2
    if (tid < n) {
        const int64_t j = tid < w.lead - j0 ? j0 + tid : w.tail + (tid - (w.lead - j0));
        const float x[1][1] = {{to_f32(row[j])}};
        add_scores<1, 1>(st, x, c);
    }
    return st;
}

// over the block, valid in every thread
template <class T>
__device__ __forceinline__ Stat row_statistics(const T* __restrict__ row, int64_t j0, int64_t j1, float c, Stat* red)
{
    Stat st = join_lanes(thread_statistics(row, j0, j1, c, threadIdx.x, blockDim.x), c);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) red[threadIdx.x >> 6] = st;
    __syncthreads();
    const int waves = blockDim.x / 64, lane = threadIdx.x & 63;   // at most 16: every wavefront joins them for itself
    st = lane < waves ? red[lane] : Stat{-INFINITY, 0.0f, 0.0f, 0.0f};
    return join_lanes(st, c);
}

__device__ __forceinline__ bool row_counts(const LossArgs& a, int64_t row)
{
    return a.item[row] >= 0 && a.item[row] < a.n_items;
}

template <class T>
__global__ __launch_bounds__(512) void row_statistics_kernel(LossArgs a)
{
    __shared__ Stat red[8];
    const int64_t row = blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    if (!row_counts(a, row)) return;
    if (a.off && (row < a.off[0] || row >= a.off[a.n_seq])) return;
    const int64_t per = (a.n_items + a.splits - 1) / a.splits, j0 = split * per, j1 = j0 + per < a.n_items ? j0 + per : a.n_items;
    const Stat st = row_statistics((const T*)a.scores + row * a.scores_stride, j0 < j1 ? j0 : j1, j1, a.scale2, red);
    if (threadIdx.x == 0) a.part[blockIdx.x] = make_float4(st.m, st.l, st.ls, st.qs);
}

__device__ __forceinline__ Stat part_of(const LossArgs& a, int64_t row, int k)
{
    const float4 p = a.part[row * a.splits + k];
    return {p.x, p.y, p.z, p.w};
}

// log p of a row's item from the row's statistics; false: the row takes no part
template <class T>
__device__ __forceinline__ bool row_log_probability(const LossArgs& a, int64_t row, const Stat& st, double& logp)
{
    logp = 0.0;
    if (st.m == -INFINITY && st.l == 0.0f) return false;
    const double of = fmax((double)st.ls, (double)st.l * (sizeof(T) / 16.0));   // a sample with less than its share speaks for its share
    const double l = log((double)st.l), mean = of > 0.0 ? (double)st.qs / of : 0.0;
    logp = (double)a.scale * ((double)to_f32(((const T*)a.scores)[row * a.scores_stride + a.item[row]]) - (double)st.m) - l - a.scale_rest * mean;
    return true;
}

__device__ __forceinline__ double softplus64(double v) { return fmax(v, 0.0) + log1p(exp(-fabs(v))); }

__device__ __forceinline__ void pair_loss(const LossArgs& a, int64_t p, double m)
{
    a.margin[p] = (float)m;
    double loss = 0.0;   // a term with weight 0 adds nothing, be it infinite
    if (a.smoothing < 1.0) loss += (1.0 - a.smoothing) * softplus64(-m);
    if (a.smoothing > 0.0) loss += a.smoothing * softplus64(m);
    a.loss[p] = (float)loss;
}
// d(weighted loss) / d(log p) of the preferred list's rows; the other list's have the opposite
__device__ __forceinline__ float pair_coef(const LossArgs& a, int64_t p, double m)
{
    return (float)(a.beta * (a.smoothing - 1.0 / (1.0 + exp(m))) * (double)a.grad_weight[p]);
}

// A block per pair adds up its two lists' rows in a fixed order: a thread per row, or a wavefront where a row has several parts.
template <class T>
__global__ __launch_bounds__(256) void preference_kernel(LossArgs a)
{
    __shared__ double red[256];
    const int64_t p = blockIdx.x;
    double sum = 0.0;
    int64_t begin[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {   // offsets that break the rules stay within the rows
        const int64_t o = a.off[2 * p + k];
        begin[k] = o < 0 ? 0 : o > a.rows ? a.rows : o;
    }
    const bool wide = a.splits > 1;
    const int lane = wide ? threadIdx.x & 63 : 0, at = wide ? threadIdx.x >> 6 : threadIdx.x, step = wide ? 4 : 256;
#pragma unroll
    for (int side = 0; side < 2; side++)
        for (int64_t row = begin[side] + at; row < begin[side + 1]; row += step) {
            double logp = 0.0;
            bool on = row_counts(a, row);
            Stat st = {-INFINITY, 0.0f, 0.0f, 0.0f};
            if (on) {
                if (wide) {
                    for (int k = lane; k < a.splits; k += 64) st = join(st, part_of(a, row, k), a.scale2);
                    st = join_lanes(st, a.scale2);
                } else {
                    st = part_of(a, row, 0);
                }
            }
            if (lane) continue;
            on = on && row_log_probability<T>(a, row, st, logp);
            a.logp[row] = (float)logp;
            a.stat[row] = make_float2(st.m, st.l);
            if (on && a.ref_logp) logp -= (double)a.ref_logp[row];
            sum += side ? -logp : logp;
            a.coef[row] = on ? (side ? -1.0f : 1.0f) : 0.0f;
        }
    red[threadIdx.x] = sum;
    __syncthreads();
    for (int n = 128; n > 0; n >>= 1) {
        if ((int)threadIdx.x < n) red[threadIdx.x] += red[threadIdx.x + n];
        __syncthreads();
    }
    const double m = a.beta * red[0];
    if (threadIdx.x == 0) pair_loss(a, p, m);
    if (!a.grad_weight) return;
    const float c = pair_coef(a, p, m);
    for (int64_t row = begin[0] + threadIdx.x; row < begin[2]; row += 256) a.coef[row] = a.coef[row] == 0.0f ? 0.0f : a.coef[row] * c;
}

// loss, KL and c_t of one row
__device__ __forceinline__ void policy_row(const LossArgs& a, int64_t row, double logp, bool on, float& coef)
{
    double loss = 0.0, kl = 0.0, c = 0.0;
    if (on) {
        const double adv = a.advantage[row], r = exp(logp - (double)a.old_logp[row]);
        // an advantage of 0 asks for nothing, however far the ratio went
        const double open = adv == 0.0 ? 0.0 : r * adv, held = adv == 0.0 ? 0.0 : fmin(fmax(r, 1.0 - a.clip_low), 1.0 + a.clip_high) * adv;
        const bool nan = r != r || open != open || held != held;   // (0 times infinity too; fmin would take the other term)
        loss = nan ? (double)NAN : -fmin(open, held);
        c = nan ? (double)NAN : open <= held ? -open : 0.0;
        if (a.ref_logp) {
            const double x = (double)a.ref_logp[row] - logp, e = expm1(x);
            kl = x == (double)INFINITY ? x : e - x;
            if (a.kl_coef != 0.0) { loss += a.kl_coef * kl; c -= a.kl_coef * e; }
        }
    }
    a.loss[row] = (float)loss;
    if (a.kl) a.kl[row] = (float)kl;
    a.logp[row] = (float)logp;
    coef = a.grad_weight ? (float)(c * (double)a.grad_weight[row]) : 0.0f;
    if (!on) coef = 0.0f;
}

// a wavefront per row joins its parts
template <class T>
__global__ __launch_bounds__(256) void policy_kernel(LossArgs a)
{
    const int64_t row = (int64_t)blockIdx.x * 4 + (threadIdx.x >> 6);
    const int lane = threadIdx.x & 63;
    if (row >= a.rows) return;
    Stat st = {-INFINITY, 0.0f, 0.0f, 0.0f};
    const bool counts = row_counts(a, row);
    if (counts)
        for (int k = lane; k < a.splits; k += 64) st = join(st, part_of(a, row, k), a.scale2);
    st = join_lanes(st, a.scale2);
    if (lane) return;
    double logp = 0.0;
    const bool on = counts && row_log_probability<T>(a, row, st, logp);
    a.stat[row] = make_float2(st.m, st.l);
    policy_row(a, row, logp, on, a.coef[row]);
}

// 16 bytes that are not needed again: the gradient, and the scores it is made of, leave the Infinity Cache to the rows that are
// yet to be read a second time (2000 rows of 200 000 bf16 scores: 355 us without, 332 so; 1536 rows of preferences 365 and 321 us)
typedef unsigned int Quad __attribute__((ext_vector_type(4)));
template <class P> __device__ __forceinline__ P load_once(const P* p)
{
    static_assert(sizeof(P) == 16);
    return __builtin_bit_cast(P, __builtin_nontemporal_load(reinterpret_cast<const Quad*>(p)));
}
template <class P> __device__ __forceinline__ void store_once(P* p, const P& v)
{
    static_assert(sizeof(P) == 16);
    __builtin_nontemporal_store(__builtin_bit_cast(Quad, v), reinterpret_cast<Quad*>(p));
}

// The gradient's elements [j0, j1) of a row, from its end to its beginning: where the same block has just read the row, what it
// read last is still in the cache.
template <class T>
__device__ __forceinline__ void write_gradient(const LossArgs& a, int64_t row, int64_t j0, int64_t j1, float coef, float m, float l, int tid, int step)
{
    constexpr int V = 16 / sizeof(T), N = 4;
    const T* in = (const T*)a.scores + row * a.scores_stride;
    T* out = (T*)a.dscores + row * a.dscores_stride;
    const float c = coef * a.scale, cl = -c / l;   // c (1[item] - 2^(c2 (x - m)) / l)
    const int64_t item = a.item[row];
    auto of = [&](float x, int64_t j) {
        const float e = cl * fast_exp2((x - m) * a.scale2);
        return j == item ? c + e : e;
    };
    const bool same = (((uintptr_t)(in + j0) ^ (uintptr_t)(out + j0)) & 15) == 0;   // rows of equal alignment move in 16-byte pieces
    Vectors w = vectors_of(out, j0, j1);
    if (!same) w = {j1, 0, j1};
    const Pack<T, V>* p = reinterpret_cast<const Pack<T, V>*>(in + w.lead);
    Pack<T, V>* q = reinterpret_cast<Pack<T, V>*>(out + w.lead);
    auto vector_of = [&](const Pack<T, V>& raw, int64_t i) {
        const int64_t j = w.lead + i * V;
        float x[V];
        unpack<T, V>(raw, x);
        Pack<T, V> o;
        if (item >= j && item < j + V) {
#pragma unroll
            for (int v = 0; v < V; v++) o.v[v] = from_f32<T>(of(x[v], j + v));
        } else {
#pragma unroll
            for (int v = 0; v < V; v++) o.v[v] = from_f32<T>(cl * fast_exp2((x[v] - m) * a.scale2));
        }
        return o;
    };
    const int64_t whole = w.n / (N * step) * (N * step);
    for (int64_t i = whole + tid; i < w.n; i += step) store_once(q + i, vector_of(load_once(p + i), i));
    for (int64_t i = whole - N * step + tid; i >= 0; i -= N * step) {
        Pack<T, V> raw[N];
#pragma unroll
        for (int n = 0; n < N; n++) raw[n] = load_once(p + i + n * step);
#pragma unroll
        for (int n = 0; n < N; n++) store_once(q + i + n * step, vector_of(raw[n], i + n * step));
    }
    for (int64_t j = j0 + tid; j < w.lead; j += step) out[j] = from_f32<T>(of(to_f32(in[j]), j));
    for (int64_t j = w.tail + tid; j < j1; j += step) out[j] = from_f32<T>(of(to_f32(in[j]), j));
}

template <class T>
__device__ __forceinline__ void write_zeros(const LossArgs& a, int64_t row, int64_t j0, int64_t j1, int tid, int step)
{
    constexpr int V = 16 / sizeof(T);
    T* out = (T*)a.dscores + row * a.dscores_stride;
    const Vectors w = vectors_of(out, j0, j1);
    Pack<T, V> zero;
#pragma unroll
    for (int v = 0; v < V; v++) zero.v[v] = from_f32<T>(0.0f);
    for (int64_t i = tid; i < w.n; i += step) reinterpret_cast<Pack<T, V>*>(out + w.lead)[i] = zero;
    for (int64_t j = j0 + tid; j < w.lead; j += step) out[j] = zero.v[0];
    for (int64_t j = w.tail + tid; j < j1; j += step) out[j] = zero.v[0];
}

// Rows in falling order: the last ones that the statistics read are the ones still in the Infinity Cache.  1536 rows of 200 000 bf16
// scores: statistics 107 us, 5.7 TB/s; gradient 208 us, 5.9 TB/s of scores and gradient.
template <class T>
__global__ __launch_bounds__(512) void gradient_kernel(LossArgs a)
{
    const int64_t row = a.rows - 1 - blockIdx.x / a.splits;
    const int split = blockIdx.x % a.splits;
    const int64_t per = (a.n_items + a.splits - 1) / a.splits, j1 = (split + 1) * per < a.n_items ? (split + 1) * per : a.n_items, j0 = split * per < j1 ? split * per : j1;
    if (a.off && (row < a.off[0] || row >= a.off[a.n_seq])) {
        if (!a.zero_rest) return;
        write_zeros<T>(a, row, j0, j1, threadIdx.x, blockDim.x);
        if (split == 0 && threadIdx.x == 0) a.logp[row] = 0.0f;
        return;
    }
    const float coef = a.coef[row];
    if (coef == 0.0f) write_zeros<T>(a, row, j0, j1, threadIdx.x, blockDim.x);   // p is finite or the row's coefficient is NaN: nothing to read
    else write_gradient<T>(a, row, j0, j1, coef, a.stat[row].x, a.stat[row].y, threadIdx.x, blockDim.x);
}

// The policy loss where a block takes whole rows: it reads a row twice, but the second time from the cache (two blocks of a
// compute unit hold 2 x 400 KB of bf16 rows of 200 000 items at a time, 200 MB over the chip, within the 256 MB of Infinity
// Cache), and one launch does it all (2000 rows: 332 us, 4.8 TB/s of scores and gradient, counted once).
template <class T>
__global__ __launch_bounds__(1024) void policy_fused_kernel(LossArgs a)
{
    __shared__ Stat red[16];
    __shared__ float coef_s;
    const int64_t row = blockIdx.x;
    const bool counts = row_counts(a, row);
    Stat st = {-INFINITY, 0.0f, 0.0f, 0.0f};
    if (counts) st = row_statistics((const T*)a.scores + row * a.scores_stride, 0, a.n_items, a.scale2, red);
    if (threadIdx.x == 0) {
        double logp = 0.0;
        const bool on = counts && row_log_probability<T>(a, row, st, logp);
        policy_row(a, row, logp, on, coef_s);
    }
    if (!a.dscores) return;
    __syncthreads();
    const float coef = coef_s;
    if (coef == 0.0f) write_zeros<T>(a, row, 0, a.n_items, threadIdx.x, blockDim.x);
    else write_gradient<T>(a, row, 0, a.n_items, coef, st.m, st.l, threadIdx.x, blockDim.x);
}

// Few rows of few items: one launch, a block per pair, a wavefront per row (at most kSmallRows rows in the call, so in a pair).
constexpr int kSmallRows = 64;
template <class T>
__global__ __launch_bounds__(1024) void preference_small_kernel(LossArgs a)
{
    __shared__ double gain[kSmallRows];
    __shared__ float m_s[kSmallRows], l_s[kSmallRows];
    __shared__ bool on_s[kSmallRows];
    __shared__ float coef_s;
    const int64_t p = blockIdx.x;
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63, rows = (int)a.rows;
    int begin[3];
#pragma unroll
    for (int k = 0; k < 3; k++) {   // offsets that break the rules stay within the rows
        const int64_t o = a.n_seq ? a.off[2 * p + k] : rows;
        begin[k] = o < 0 ? 0 : o > rows ? rows : (int)o;
    }
    if (threadIdx.x < kSmallRows) gain[threadIdx.x] = 0.0;
    __syncthreads();
    for (int row = begin[0] + wave; row < begin[2]; row += 16) {
        bool on = row_counts(a, row);
        Stat st = {-INFINITY, 0.0f, 0.0f, 0.0f};
        if (on) st = join_lanes(thread_statistics((const T*)a.scores + row * a.scores_stride, 0, a.n_items, a.scale2, lane, 64), a.scale2);
        if (lane) continue;
        double logp = 0.0;
        on = on && row_log_probability<T>(a, row, st, logp);
        a.logp[row] = (float)logp;
        if (on && a.ref_logp) logp -= (double)a.ref_logp[row];
        gain[row] = row < begin[1] ? logp : -logp;
        m_s[row] = st.m;
        l_s[row] = st.l;
        on_s[row] = on;
    }
    __syncthreads();
    if (wave == 0 && a.n_seq) {
        const double m = a.beta * group_sum<64>(gain[lane]);
        if (lane == 0) {
            pair_loss(a, p, m);
            coef_s = a.grad_weight ? pair_coef(a, p, m) : 0.0f;
        }
    }
    if (blockIdx.x == 0 && a.zero_rest)   // rows of no list
        for (int row = wave; row < rows; row += 16)
            if (row < a.off[0] || row >= a.off[a.n_seq]) {
                if (lane == 0) a.logp[row] = 0.0f;
                if (a.dscores) write_zeros<T>(a, row, 0, a.n_items, lane, 64);
            }
    __syncthreads();
    if (!a.dscores) return;
    for (int row = begin[0] + wave; row < begin[2]; row += 16) {
        const float coef = !on_s[row] ? 0.0f : row < begin[1] ? coef_s : -coef_s;
        if (coef == 0.0f) write_zeros<T>(a, row, 0, a.n_items, lane, 64);
        else write_gradient<T>(a, row, 0, a.n_items, coef, m_s[row], l_s[row], lane, 64);
    }
}

// rows of no list, where no gradient pass comes by
__global__ __launch_bounds__(256) void rest_kernel(LossArgs a)
{
    const int64_t row = (int64_t)blockIdx.x * 256 + threadIdx.x;
    if (row < a.rows && (row < a.off[0] || row >= a.off[a.n_seq])) a.logp[row] = 0.0f;
}

int check_desc(const rec_loss_desc* d)
{
    REC_REFUSE(!d, "null argument");
    REC_REFUSE(d->type < REC_TYPE_F32 || d->type > REC_TYPE_BF16, "unknown type");
    REC_REFUSE(d->rows < 0 || d->rows > (1 << 22) - 1, "rows must be in 0..2^22-1");   // a launch holds fewer than 2^32 threads
    REC_REFUSE(d->n_items < 1 || d->n_items > INT32_MAX, "n_items must be in 1..2^31-1");
    REC_REFUSE(!(d->scale > 0.0f) || !isfinite((float)(d->scale * 1.4426950408889634)), "scale must be positive, and scale * log2(e) finite");
    return 0;
}

// Parts a row is cut into: one where the rows alone fill the chip (4 blocks of 512 threads per compute unit), else as many as
// that takes, of at least 8192 items each.
constexpr int kThreads = 512;
int splits_of(const rec_loss_desc* d)
{
    const int64_t want = d->rows > 0 ? (1024 + d->rows - 1) / d->rows : 1, most = (d->n_items + 8191) / 8192;
    const int64_t s = want < most ? want : most;
    return (int)(s < 1 ? 1 : s > 256 ? 256 : s);
}

int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }
// One launch does it all, and nothing passes between launches: a wavefront reads a row by itself, a pair's block 16 at a time, so rows
// are short, and few to a pair (how they are spread over the pairs the host does not know).  One launch against three, us in a graph:
// 2 rows of 4000, 8000, 16 000, 65 536 f32 items 9.5 / 12.5, 13.0 / 12.7, 19 / 13, 60 / 12; 6 of 4000 and 8000 11 / 13, 15 / 13; 16 of
// 2000 and 4000 11 / 13, 15 / 13; a second round pays below 25 rows: 24 of 300 and 1000 9.0 / 11.0, 11.6 / 11.7; 32 of 500 11.4 / 10.9; 64
// of 2000 34 / 13 in one pair, 12 / 13 in four, 8 / 13 in 32.
bool small_preference(const rec_loss_desc* d, int n_pairs)
{
    if (d->rows > kSmallRows || d->rows * d->n_items > 131072) return false;
    if (d->rows > 16 * (int64_t)n_pairs) return d->rows <= 24 * (int64_t)n_pairs && d->n_items <= 1000;
    return d->n_items <= 8000 && d->rows * d->n_items <= 32768 * (int64_t)n_pairs;
}
// (64, 256 and 900 rows of 20 000 bf16 items: calls of 13, 14 and 20 us, 20, 21 and 36 by three launches over parts of rows; 900 of
// 200 000 items 158 and 194)
bool whole_policy(const rec_loss_desc* d) { return splits_of(d) == 1 || d->rows >= 512 || d->n_items * rec_type_size(d->type) < 65536; }
// Threads for a row that a block reads and then turns into its gradient.  Small blocks keep more rows in flight, and a row's loads
// over the waits of another's sums; the rows in flight, 2048 threads' worth on each of 256 compute units, should stay within 210 MB
// of the Infinity Cache.  Few rows take more, down to two or three 16-byte loads a thread, until a quarter of the lanes are
// busy.  (bf16: 20 000 rows of 20 000 items 599 us with 1024 threads, 356 with 256, 350 with the rule's 128; 4000 of 60 000 items 234, 206
// with 1024, 256, 198 with the rule's 512; 300 of 8000 items 12, 10 with 64, 128, 7.6 with the rule's 512; f32, 50 000 of 4000 items 579,
// 311 with 512, 128, 326 with the rule's 64.)
int row_threads(const rec_loss_desc* d)
{
    const int64_t bytes = d->n_items * rec_type_size(d->type);
    int threads = 64;
    while (threads < 1024 && (threads * 400 < bytes || (d->rows * threads < 131072 && bytes / 16 >= 3 * threads))) threads *= 2;
    return threads;
}
// Threads for a row, or a part of one, where one launch reads the scores and another makes the gradient: four 16-byte loads each at
// least (500 000 rows of 300 bf16 items 3734 us with 512 threads, 677 with 64; 8000 of 2000 items 70 and 37).
int part_threads(const rec_loss_desc* d)
{
    const int64_t vectors = d->n_items * rec_type_size(d->type) / 16;
    int threads = 64;
    while (threads < kThreads && (splits_of(d) > 1 || vectors >= 8 * threads)) threads *= 2;
    return threads;
}
int64_t workspace_of(const rec_loss_desc* d) { return d->rows * splits_of(d) * 16 + round16(d->rows * 8) + round16(d->rows * 4); }

int check_call(const rec_loss_desc* d, const void* scores, int64_t scores_stride, const float* grad_weight, int64_t weights, const void* dscores,
               int64_t dscores_stride, const void* workspace, int64_t workspace_bytes, int64_t needs)
{
    const int64_t size = rec_type_size(d->type);
    REC_REFUSE(scores_stride < d->n_items || scores_stride > INT32_MAX, "the scores' row stride is smaller than n_items, or beyond 2^31-1");
    REC_REFUSE(weights > 0 && d->rows > 0 && !grad_weight != !dscores, "grad_weight and dscores come together");   // an empty array may be null
    if (dscores) {
        REC_REFUSE(dscores_stride < d->n_items || dscores_stride > INT32_MAX, "the gradient's row stride is smaller than n_items, or beyond 2^31-1");
        const bool in_place = dscores == scores && dscores_stride == scores_stride;
        REC_REFUSE(!in_place && rec_overlap(RowsOf{scores, d->rows, scores_stride * size, d->n_items * size}, RowsOf{dscores, d->rows, dscores_stride * size, d->n_items * size}), "dscores overlaps the scores");
    }
    REC_REFUSE(workspace_bytes < needs, "the workspace is too small");
    REC_REFUSE(needs > 0 && (!workspace || !rec_aligned(workspace, 16)), "the workspace is null or not aligned to 16 bytes");
    return rec_check_device(d->device);
}

void fill(LossArgs& a, const rec_loss_desc* d, const void* scores, int64_t scores_stride, const int32_t* item, const float* ref_logp, const float* grad_weight,
          float* loss, float* logp, void* dscores, int64_t dscores_stride, void* workspace)
{
    a.scores = scores; a.scores_stride = scores_stride; a.item = item; a.ref_logp = ref_logp; a.grad_weight = grad_weight;
    a.loss = loss; a.logp = logp; a.dscores = dscores; a.dscores_stride = dscores_stride;
    a.rows = d->rows; a.n_items = d->n_items; a.scale = d->scale; a.scale2 = (float)((double)d->scale * 1.4426950408889634);
    a.scale_rest = (double)d->scale - (double)a.scale2 * 0.6931471805599453;
    a.zero_rest = d->zero_rest; a.splits = splits_of(d);
    char* ws = (char*)workspace;
    a.part = (float4*)ws;
    a.stat = (float2*)(ws + d->rows * a.splits * 16);
    a.coef = (float*)(ws + d->rows * a.splits * 16 + round16(d->rows * 8));
}

#define LOSS_DISPATCH(CALL)                                                                         \
    if (d->type == REC_TYPE_F32) { CALL(float); }                                                   \
    else if (d->type == REC_TYPE_F16) { CALL(_Float16); }                                           \
    else { CALL(__bf16); }

}  // namespace

extern "C" int64_t rec_preference_loss_workspace(const rec_loss_desc* d, int32_t n_pairs)
{
    return rec_guarded([&]() -> int64_t {
        if (check_desc(d)) return -1;
        REC_REFUSE(n_pairs < 0 || n_pairs > (1 << 22) - 1, "n_pairs must be in 0..2^22-1");
        return small_preference(d, n_pairs) ? 0 : workspace_of(d);
    });
}

extern "C" int rec_preference_loss(const rec_loss_desc* d, const void* scores, int64_t scores_stride, const int32_t* item,
                                   const int64_t* seq_off, int32_t n_pairs, const float* ref_logp, float beta, float smoothing,
                                   const float* grad_weight, float* loss, float* margin, float* logp, void* dscores, int64_t dscores_stride,
                                   void* workspace, int64_t workspace_bytes, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        REC_REFUSE(n_pairs < 0 || n_pairs > (1 << 22) - 1, "n_pairs must be in 0..2^22-1");
        REC_REFUSE(!seq_off || (d->rows > 0 && (!scores || !item || !logp)) || (n_pairs > 0 && (!loss || !margin)), "null argument");
        REC_REFUSE(!isfinite(beta), "beta must be finite");
        REC_REFUSE(!(smoothing >= 0.0f && smoothing <= 1.0f), "smoothing must be in 0..1");
        if (int rc = check_call(d, scores, scores_stride, grad_weight, n_pairs, dscores, dscores_stride, workspace, workspace_bytes, small_preference(d, n_pairs) ? 0 : workspace_of(d))) return rc;
        LossArgs a = {};
        fill(a, d, scores, scores_stride, item, ref_logp, grad_weight, loss, logp, dscores, dscores_stride, workspace);
        a.off = seq_off; a.n_seq = 2 * n_pairs; a.margin = margin; a.beta = beta; a.smoothing = smoothing;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        hipStream_t st = (hipStream_t)stream;
        // (one pair of 6 x 2848 f32: 9.5 us, three launches of 4.8, 4.0 and 3.4 us otherwise)
        if (d->rows > 0 && small_preference(d, n_pairs)) {
#define CALL(T) preference_small_kernel<T><<<n_pairs ? (unsigned)n_pairs : 1u, 1024, 0, st>>>(a)
            LOSS_DISPATCH(CALL)
#undef CALL
            HIP_TRY(hipGetLastError());
            return 0;
        }
        const unsigned blocks = (unsigned)(d->rows * a.splits);
#define CALL(T)                                                                                     \
        if (blocks) row_statistics_kernel<T><<<blocks, part_threads(d), 0, st>>>(a);                       \
        if (n_pairs) preference_kernel<T><<<(unsigned)n_pairs, 256, 0, st>>>(a);                    \
        if (blocks && dscores) gradient_kernel<T><<<blocks, part_threads(d), 0, st>>>(a)
        LOSS_DISPATCH(CALL)
#undef CALL
        if (d->zero_rest && !dscores && d->rows > 0) rest_kernel<<<(unsigned)((d->rows + 255) / 256), 256, 0, st>>>(a);
        HIP_TRY(hipGetLastError());
        return 0;
    });
}

extern "C" int64_t rec_policy_loss_workspace(const rec_loss_desc* d)
{
    return rec_guarded([&]() -> int64_t {
        if (check_desc(d)) return -1;
        return whole_policy(d) ? 0 : workspace_of(d);
    });
}

extern "C" int rec_policy_loss(const rec_loss_desc* d, const void* scores, int64_t scores_stride, const int32_t* item,
                               const float* old_logp, const float* advantage, const float* ref_logp, float clip_low, float clip_high,
                               float kl_coef, const float* grad_weight, float* loss, float* kl, float* logp, void* dscores,
                               int64_t dscores_stride, void* workspace, int64_t workspace_bytes, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        REC_REFUSE(d->rows > 0 && (!scores || !item || !old_logp || !advantage || !loss || !logp), "null argument");
        REC_REFUSE(!(clip_low >= 0.0f && clip_low <= 1.0f) || !(clip_high >= 0.0f) || !isfinite(clip_high), "clip_low must be in 0..1 and clip_high at least 0");
        REC_REFUSE(!isfinite(kl_coef) || (!ref_logp && kl_coef != 0.0f), "kl_coef must be finite, and 0 without ref_logp");
        if (int rc = check_call(d, scores, scores_stride, grad_weight, d->rows, dscores, dscores_stride, workspace, workspace_bytes, whole_policy(d) ? 0 : workspace_of(d))) return rc;
        LossArgs a = {};
        fill(a, d, scores, scores_stride, item, ref_logp, grad_weight, loss, logp, dscores, dscores_stride, workspace);
        a.old_logp = old_logp; a.advantage = advantage; a.kl = kl;
        a.clip_low = clip_low; a.clip_high = clip_high; a.kl_coef = kl_coef;
        if (d->rows == 0) return 0;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        hipStream_t st = (hipStream_t)stream;
        if (whole_policy(d)) {
#define CALL(T) policy_fused_kernel<T><<<(unsigned)d->rows, row_threads(d), 0, st>>>(a)
            LOSS_DISPATCH(CALL)
#undef CALL
            HIP_TRY(hipGetLastError());
            return 0;
        }
        const unsigned blocks = (unsigned)(d->rows * a.splits);
#define CALL(T)                                                                                     \
        row_statistics_kernel<T><<<blocks, part_threads(d), 0, st>>>(a);                                   \
        policy_kernel<T><<<(unsigned)((d->rows + 3) / 4), 256, 0, st>>>(a);                         \
        if (dscores) gradient_kernel<T><<<blocks, part_threads(d), 0, st>>>(a)
        LOSS_DISPATCH(CALL)
#undef CALL
        HIP_TRY(hipGetLastError());
        return 0;
    });
}
