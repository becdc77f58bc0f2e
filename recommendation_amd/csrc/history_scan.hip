// Selective state space scan over packed histories: y, its gradient, and the form for single clicks.
//
//   delta = softplus(raw + bias)    h_t[n] = exp(delta_t A[n]) h_{t-1}[n] + delta_t u_t B_t[n]    y_t = (sum_n C_t[n] h_t[n] + D u_t) silu(z_t)
//
// per channel; h starts at each history's initial state.  A lane holds four states of one channel, LN neighbouring lanes all of
// them, so a block of 256 lanes walks 256 / LN channels of one group through time; what a step needs per channel (delta and
// delta * u) and per group (B, C) is staged in LDS 16 rows at a time, in f32.
//
// The packed rows are cut into chunks that ignore where histories begin, so ragged lengths leave no block idle.  A history that
// crosses from one chunk into the next hands its state over: the first pass computes what each chunk adds on its own
// (only from the last history's beginning on, and only if it goes on), the second links the chunks of each history, the third
// walks again from the linked states and writes y.  With one chunk the first two are not launched.
//
// Bound by vector instructions: per row and state one exp and three multiply-adds forwards, one exp and some ten backwards, and
// the sums over states and channels.  100 000 rows of 128 bf16 channels with 16 states (1000 histories): 45 + 17 + 80 us for
// the three passes, 48 + 22 + 244 and 12 + 9 for sums backwards, where the arrays alone would take 42 us in all at the rate of a copy.
#include "operators.h"
#include <type_traits>

namespace {

constexpr int TT = REC_SCAN_CHECKPOINT;   // rows staged at a time
constexpr int HALF = 8;                   // rows whose states the gradient keeps

struct ScanArgs {
    const void *u, *delta, *z, *B, *C, *dy;
    const float *A, *D, *delta_bias, *initial, *dfinal, *checkpoints_in;
    const int64_t* off;
    void *y, *du, *ddelta, *dz, *dB, *dC;
    float *final_state, *checkpoints, *dinitial;
    float *link, *span;          // [chunks][channels][states] state handed into a chunk (backward: gradient handed out of it), [chunks][channels] sum of delta
    int* kind;                   // [chunks] what a chunk hands on: 0 nothing, 1 what it adds itself, 2 what it is handed as well
    float *part_bc;              // backward: [channel tiles of a group][rows][groups][2][states]
    float *part_a;               // backward: [chunks][channels * states + 2 * channels]: dA, dD, ddelta_bias
    int64_t u_stride, delta_stride, z_stride, B_stride, C_stride, y_stride, dy_stride;
    int64_t rows;
    int main_blocks, n_seq, channels, groups, per, states, chunk, chunks, tiles, tiles_per_group, softplus, zero_rest;
};

// the block's place: a chunk of rows, a run of channels of one group
template <int LN> struct Place {
    static constexpr int CH = 256 / LN;
    int64_t r0, r1;
    int chunk, g, part, ch0, nch, ch, lane_n, d;
    bool on;
    __device__ __forceinline__ Place(const ScanArgs& a)
    {
        const int tile = blockIdx.x % a.tiles;
        chunk = blockIdx.x / a.tiles;
        r0 = (int64_t)chunk * a.chunk;
        r1 = r0 + a.chunk < a.rows ? r0 + a.chunk : a.rows;
        g = tile / a.tiles_per_group;
        part = tile % a.tiles_per_group;
        ch0 = g * a.per + part * CH;
        nch = min(CH, (g + 1) * a.per - ch0);
        ch = threadIdx.x / LN;
        lane_n = threadIdx.x % LN * 4;
        on = ch < nch;
        d = ch0 + (on ? ch : 0);
    }
};

// Four of a channel's states, of an f32 array [...][channels][states].  The array's leading index is the same for the whole
// block, so an address is a scalar base and a 32-bit offset of the lane (channels * states * 4 < 2^29).
template <int LN>
__device__ __forceinline__ void load_states(const float* p, int64_t lead, const ScanArgs& a, int d, int n0, bool on, float (&h)[4])
{
    struct alignas(4) Four { float v[4]; };
    const float* base = p + lead * ((int64_t)a.channels * a.states);
    const int at = d * a.states + n0;
    if (!p) {
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = 0.0f;
    } else if (a.states == 4 * LN) {
        const Four f = *reinterpret_cast<const Four*>(base + at);
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = on ? f.v[e] : 0.0f;
    } else {
#pragma unroll
        for (int e = 0; e < 4; e++) h[e] = on && n0 + e < a.states ? base[at + e] : 0.0f;
    }
}
template <int LN>
__device__ __forceinline__ void store_states(float* p, int64_t lead, const ScanArgs& a, int d, int n0, bool on, const float (&h)[4])
{
    struct alignas(4) Four { float v[4]; };
    float* base = p + lead * ((int64_t)a.channels * a.states);
    const int at = d * a.states + n0;
    if (!on) return;
    if (a.states == 4 * LN) {
        *reinterpret_cast<Four*>(base + at) = Four{{h[0], h[1], h[2], h[3]}};
        return;
    }
#pragma unroll
    for (int e = 0; e < 4; e++)
        if (n0 + e < a.states) base[at + e] = h[e];
}

// `v`, computed whether or not the choice that follows wants it: a choice that is the same for the whole launch would otherwise
// become a branch for each of a thread's values, and keep their loads and exps from overlapping.
__device__ __forceinline__ float computed(float v)
{
    asm volatile("" : "+v"(v));
    return v;
}

// What a thread stages of a tile: PT (row, channel) pairs, 256 apart, all of one channel, and NB values each of B and C.
// Loads come first and unconditionally (a row or channel outside the chunk takes the nearest inside), so that all of a tile's are
// in flight together; what does not count is set to zero when it is staged.
template <class T, int LN, bool U, bool Z, bool DY, bool GB, bool GC> struct Tile {
    static constexpr int CH = 256 / LN, NP = 4 * LN, PT = TT * CH / 256, NB = TT * NP > 256 ? TT * NP / 256 : 1;
    T d[PT], u[U ? PT : 1], z[Z ? PT : 1], g[DY ? PT : 1], b[GB ? NB : 1], c[GC ? NB : 1];
    // the row of pair k: where a wavefront's pairs are of one row, a scalar
    static __device__ __forceinline__ int row(int k)
    {
        const int t = CH >= 64 ? __builtin_amdgcn_readfirstlane(threadIdx.x & ~63u) : (int)threadIdx.x;
        return (t + 256 * k) / CH;
    }
    static __device__ __forceinline__ int channel() { return threadIdx.x % CH; }
    __device__ __forceinline__ void fetch(const ScanArgs& a, const Place<LN>& p, int64_t t0)
    {
        const int dd = p.ch0 + min(channel(), p.nch - 1);
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int64_t at = t0 + row(k) < p.r1 ? t0 + row(k) : p.r1 - 1;
            d[k] = ((const T*)a.delta + at * a.delta_stride)[dd];
            if (U) u[k] = ((const T*)a.u + at * a.u_stride)[dd];
            if (Z) z[k] = ((const T*)(a.z ? a.z : a.u) + at * (a.z ? a.z_stride : a.u_stride))[dd];
            if (DY) g[k] = ((const T*)a.dy + at * a.dy_stride)[dd];
        }
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const int i = threadIdx.x + 256 * k, n = i % NP < a.states ? i % NP : a.states - 1;
            const int64_t r = t0 + i / NP % TT, at = r < p.r1 ? r : p.r1 - 1;
            if (GB) b[k] = ((const T*)a.B + at * a.B_stride)[p.g * a.states + n];
            if (GC) c[k] = ((const T*)a.C + at * a.C_stride)[p.g * a.states + n];
        }
    }
    // B and C of rows [lo, hi)
    __device__ __forceinline__ void stage_groups(const ScanArgs& a, int64_t t0, int64_t lo, int64_t hi, float (*sB)[NP], float (*sC)[NP])
    {
#pragma unroll
        for (int k = 0; k < NB; k++) {
            const int i = threadIdx.x + 256 * k, r = i / NP, n = i % NP;
            const bool counts = n < a.states && t0 + r >= lo && t0 + r < hi;
            if (TT * NP < 256 && r >= TT) continue;
            if (GB) sB[r][n] = counts ? to_f32(b[k]) : 0.0f;
            if (GC) sC[r][n] = counts ? to_f32(c[k]) : 0.0f;
        }
    }
};

// first pass: the state a chunk's last history has at the chunk's end, for a state of zero in front of the chunk.  (One history of
// 20 000 rows x 256 f16 channels: 22 us, the link 14, the third pass 32.)
template <class T, int LN>
__global__ __launch_bounds__(256) void scan_local_kernel(ScanArgs a)
{
    using P = Place<LN>;
    constexpr int CH = P::CH, NP = 4 * LN;
    __shared__ float2 sd[TT][CH];
    __shared__ alignas(16) float sB[TT][NP];
    const P p(a);
    if (p.chunk + 1 >= a.chunks) return;
    const int s = sequence_of(a.off, a.n_seq, p.r1 - 1);
    const bool goes_on = s >= 0 && s < a.n_seq && a.off[s + 1] > p.r1;
    const int64_t begin = goes_on ? a.off[s] : p.r1;
    if (blockIdx.x % a.tiles == 0 && threadIdx.x == 0) a.kind[p.chunk] = !goes_on ? 0 : begin < p.r0 ? 2 : 1;
    if (!goes_on) return;
    const int64_t from = begin > p.r0 ? begin : p.r0;
    float A2[4], h[4], span = 0.0f;
    load_states<LN>(a.A, 0, a, p.d, p.lane_n, p.on, A2);
#pragma unroll
    for (int e = 0; e < 4; e++) A2[e] *= REC_LOG2E;
    load_states<LN>(begin >= p.r0 ? a.initial : nullptr, s, a, p.d, p.lane_n, p.on, h);
    Tile<T, LN, true, false, false, true, false> t;
    const int ch = t.channel();
    const bool mine = ch < p.nch;
    const float bias = mine && a.delta_bias ? a.delta_bias[p.ch0 + ch] : 0.0f;
    t.fetch(a, p, from);
    for (int64_t t0 = from; t0 < p.r1; t0 += TT) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < t.PT; k++) {
            const bool counts = mine && t0 + t.row(k) < p.r1;
            const float raw = to_f32(t.d[k]) + bias, sp = computed(softplus_f32(raw)), delta = a.softplus ? sp : raw;
            sd[t.row(k)][ch] = counts ? make_float2(delta, delta * to_f32(t.u[k])) : make_float2(0.0f, 0.0f);
        }
        t.stage_groups(a, t0, t0, p.r1, sB, nullptr);
        __syncthreads();
        if (t0 + TT < p.r1) t.fetch(a, p, t0 + TT);
#pragma unroll
        for (int r = 0; r < TT; r++) {   // rows behind the chunk's last move nothing: exp(0) and 0
            const float2 v = sd[r][p.ch];
            span += v.x;
#pragma unroll
            for (int e = 0; e < 4; e++) h[e] = fmaf(fast_exp2(v.x * A2[e]), h[e], v.y * sB[r][p.lane_n + e]);
        }
    }
    store_states<LN>(a.link, p.chunk + 1, a, p.d, p.lane_n, p.on, h);
    if (p.on && p.lane_n == 0) a.span[(int64_t)p.chunk * a.channels + p.d] = span;
}

// The state behind rows whose decays multiply to 2^(2 x), and what those rows add to it.  The factor may be beyond f32 where the
// state is not - nothing is there to grow yet, or it is far from the end of the range - so its root is taken twice.  It is cut at
// 2^254, which leaves nothing of f32's normal range but infinity, so that 0 stays 0.
__device__ __forceinline__ float carried(float h, float x, float own)
{
    const float e = fast_exp2(x), root = x > 127.0f ? 0x1p127f : e;
    return fmaf(h * root, root, own);
}

// second pass: the state handed into chunk c + 1 is exp(A span) times what was handed into c (where c's history came from there), plus
// what c adds.  Such steps compose, so 64 threads share the chunks of a channel's state: each composes a run of them, then
// walks it again from what the runs in front of it lead to.  The exponents are added, not the factors multiplied.  A run in which
// a history begins takes nothing over: `cut`, and not a factor of 0, says so, for a factor that underflows still makes NaN of NaN.
// The gradient takes the same steps from the back.
constexpr int LINK_COLS = 16, LINK_RUNS = 64;
template <bool BACK>
__global__ __launch_bounds__(LINK_COLS * LINK_RUNS) void scan_link_kernel(ScanArgs a)
{
    __shared__ float sX[LINK_RUNS][LINK_COLS], sH[LINK_RUNS][LINK_COLS];
    __shared__ bool s_cut[LINK_RUNS][LINK_COLS];
    const int col = threadIdx.x % LINK_COLS, run = threadIdx.x / LINK_COLS;
    const int64_t i = (int64_t)blockIdx.x * LINK_COLS + col, n = (int64_t)a.channels * a.states;
    const bool on = i < n;
    const int d = on ? (int)(i / a.states) : 0;
    const float A2 = on ? a.A[i] * (0.5f * REC_LOG2E) : 0.0f;   // halves of the exponents, as carried() wants them
    const int steps = a.chunks - 1, per = (steps + LINK_RUNS - 1) / LINK_RUNS;
    const int k0 = min(run * per, steps), k1 = min(k0 + per, steps);
    // step k: forwards from chunk k, whose state goes to slot k + 1; backwards from chunk `steps - k`, whose gradient is in its own slot
    auto chunk_of = [&](int k) { return BACK ? steps - k : k; };
    auto slot_of = [&](int k) { return (int64_t)(BACK ? steps - k : k + 1) * n + i; };
    // four steps' loads at a time: the stores in between keep the compiler from running ahead
    constexpr int AHEAD = 4;
    auto walk = [&](auto&& step) {
        for (int k = k0; k < k1; k += AHEAD) {
            int kind[AHEAD];
            float own[AHEAD], span[AHEAD];
#pragma unroll
            for (int e = 0; e < AHEAD; e++) {
                const int at = min(k + e, k1 - 1), c = chunk_of(at);
                kind[e] = a.kind[c];
                own[e] = a.link[slot_of(at)];
                span[e] = a.span[(int64_t)c * a.channels + d];
            }
#pragma unroll
            for (int e = 0; e < AHEAD; e++)
                if (k + e < k1) step(k + e, kind[e], own[e], A2 * span[e]);
        }
    };
    float X = 0.0f, H = 0.0f;
    bool cut = false;
    if (on)
        walk([&](int, int kind, float own, float x) {
            cut |= kind != 2;
            X += x;
            H = kind == 2 ? carried(H, x, own) : kind == 1 ? own : 0.0f;
        });
    // what the runs up to each one lead to, by doubling
    for (int o = 1; o < LINK_RUNS; o *= 2) {
        sX[run][col] = X;
        sH[run][col] = H;
        s_cut[run][col] = cut;
        __syncthreads();
        if (run >= o && !cut) {
            H = carried(sH[run - o][col], X, H);
            X += sX[run - o][col];
            cut = s_cut[run - o][col];
        }
        __syncthreads();
    }
    sH[run][col] = H;
    __syncthreads();
    float h = run > 0 ? sH[run - 1][col] : 0.0f;
    if (!on) return;
    walk([&](int k, int kind, float own, float x) {
        h = kind == 2 ? carried(h, x, own) : kind == 1 ? own : 0.0f;
        a.link[slot_of(k)] = h;
    });
}

// Sums over a channel's lanes are taken for GR rows together: lane j < GR of the channel keeps, and writes, row j's.
template <int LN> constexpr int rows_together() { return LN < 4 ? LN : 4; }
template <int LN, int GR> __device__ __forceinline__ void write_sums(float (*to)[256 / LN + 16], int r, int ch, const float (&v)[GR])
{
    const int j = threadIdx.x % LN;
    float mine = group_sum_dpp<LN>(v[0]);
#pragma unroll
    for (int k = 1; k < GR; k++) {
        const float s = group_sum_dpp<LN>(v[k]);
        mine = j == k ? s : mine;
    }
    if (GR == LN || j < GR) to[r + j][ch] = mine;
}

// Empty histories: their state passes through (forwards initial -> final_state, backwards dfinal -> dinitial).  Blocks behind
// the walk's take them, a value per thread; so many that they alone would make a launch too large have one of their own, whose
// threads go around (a loop in the walk's kernels costs the gradient 3 % where it goes around once).
__device__ __forceinline__ void pass_value(const ScanArgs& a, const float* from, float* to, int64_t i)
{
    const int64_t s = i / ((int64_t)a.channels * a.states);
    if (a.off[s + 1] <= a.off[s]) to[i] = from ? from[i] : 0.0f;
}
__device__ __forceinline__ void pass_empty(const ScanArgs& a, const float* from, float* to)
{
    const int64_t i = (int64_t)(blockIdx.x - a.main_blocks) * 256 + threadIdx.x;
    if (i < (int64_t)a.channels * a.states * a.n_seq) pass_value(a, from, to, i);
}
__global__ __launch_bounds__(256) void scan_pass_empty_kernel(ScanArgs a, const float* from, float* to)
{
    const int64_t n = (int64_t)a.channels * a.states * a.n_seq;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) pass_value(a, from, to, i);
}
constexpr int64_t kManyStates = 1 << 28;

// third pass: y, the states that histories end with, and the checkpoints
template <class T, int LN>
__global__ __launch_bounds__(256) void scan_forward_kernel(ScanArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {
        pass_empty(a, a.initial, a.final_state);
        return;
    }
    using P = Place<LN>;
    constexpr int CH = P::CH, NP = 4 * LN, GR = rows_together<LN>();
    __shared__ float2 sd[TT][CH];
    __shared__ alignas(16) float sB[TT][NP], sC[TT][NP], sy[TT][CH + 16];   // rows of sy 16 banks apart: GR rows are written at once
    const P p(a);
    const int64_t lo = a.off[0], hi = a.off[a.n_seq];
    SeqCursor c;
    c.begin(a.off, a.n_seq, p.r0);
    float A2[4], h[4] = {0.0f, 0.0f, 0.0f, 0.0f};
    load_states<LN>(a.A, 0, a, p.d, p.lane_n, p.on, A2);
#pragma unroll
    for (int e = 0; e < 4; e++) A2[e] *= REC_LOG2E;
    if (c.inside(a.n_seq)) {
        if (a.off[c.s] >= p.r0) load_states<LN>(a.initial, c.s, a, p.d, p.lane_n, p.on, h);
        else if (p.chunk > 0) load_states<LN>(a.link, p.chunk, a, p.d, p.lane_n, p.on, h);
    }
    Tile<T, LN, true, true, false, true, true> t;
    constexpr int PT = decltype(t)::PT;
    const int ch = t.channel(), d = p.ch0 + ch;
    const bool mine = ch < p.nch;
    const float bias = mine && a.delta_bias ? a.delta_bias[d] : 0.0f, Dd = mine && a.D ? a.D[d] : 0.0f;
    t.fetch(a, p, p.r0);
    for (int64_t t0 = p.r0; t0 < p.r1; t0 += TT) {
        const int nt = (int)(p.r1 - t0 < TT ? p.r1 - t0 : TT);
        const int64_t blo = lo > t0 ? lo : t0, bhi = hi < t0 + nt ? hi : t0 + nt;   // a row of no history moves nothing
        float u[PT], gate[PT];
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int64_t row = t0 + t.row(k);
            u[k] = to_f32(t.u[k]);
            gate[k] = computed(silu_f32(to_f32(t.z[k])));
            gate[k] = a.z ? gate[k] : 1.0f;
            const float raw = to_f32(t.d[k]) + bias, sp = computed(softplus_f32(raw)), delta = a.softplus ? sp : raw;
            sd[t.row(k)][ch] = mine && row >= blo && row < bhi ? make_float2(delta, delta * u[k]) : make_float2(0.0f, 0.0f);
        }
        t.stage_groups(a, t0, blo, bhi, sB, sC);
        __syncthreads();
        if (t0 + TT < p.r1) t.fetch(a, p, t0 + TT);
        if (a.checkpoints) store_states<LN>(a.checkpoints, t0 / TT, a, p.d, p.lane_n, p.on, h);
        auto step = [&](int r) {
            const float2 v = sd[r][p.ch];
            float y = 0.0f;
#pragma unroll
            for (int e = 0; e < 4; e++) {
                h[e] = fmaf(fast_exp2(v.x * A2[e]), h[e], v.y * sB[r][p.lane_n + e]);
                y = fmaf(h[e], sC[r][p.lane_n + e], y);
            }
            return y;
        };
        if (nt == TT && t0 + TT < c.next) {   // no history begins or ends here
#pragma unroll
            for (int r = 0; r < TT; r += GR) {
                float y[GR];
#pragma unroll
                for (int k = 0; k < GR; k++) y[k] = step(r + k);
                write_sums<LN, GR>(sy, r, p.ch, y);
            }
        } else {
            for (int r = 0; r < nt; r++) {
                const int64_t row = t0 + r;
                if (row >= c.next) {
                    c.advance(a.off, a.n_seq, row);
                    load_states<LN>(c.inside(a.n_seq) ? a.initial : nullptr, c.s, a, p.d, p.lane_n, p.on, h);
                }
                const float y = group_sum_dpp<LN>(step(r));
                if (p.lane_n == 0) sy[r][p.ch] = y;
                if (a.final_state && row + 1 == c.next && c.inside(a.n_seq)) store_states<LN>(a.final_state, c.s, a, p.d, p.lane_n, p.on, h);
            }
        }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int r = t.row(k);
            const int64_t row = t0 + r;
            if (r >= nt || !mine) continue;
            T* y = (T*)a.y + row * a.y_stride + d;
            if (row < lo || row >= hi) {
                if (a.zero_rest) *y = from_f32<T>(0.0f);
                continue;
            }
            float v = sy[r][ch];
            if (a.D) v = fmaf(Dd, u[k], v);
            *y = from_f32<T>(v * gate[k]);
        }
    }
}

// ---- gradient.  With G_t = dL/dh_t:   G_t = C_t dys_t + exp(delta_{t+1} A) G_{t+1}   (dfinal in place of the second term at a
// history's last row), dys = dy silu(z).  The chunks are linked as above, from the back.

// first pass: what a chunk hands to the rows in front of it, exp(delta A) G at its first row, for nothing handed in from behind
template <class T, int LN>
__global__ __launch_bounds__(256) void scan_local_backward_kernel(ScanArgs a)
{
    using P = Place<LN>;
    constexpr int CH = P::CH, NP = 4 * LN;
    __shared__ float2 sd[TT][CH];
    __shared__ alignas(16) float sC[TT][NP];
    const P p(a);
    if (p.chunk == 0) return;
    const int s = sequence_of(a.off, a.n_seq, p.r0);
    const bool came = s >= 0 && s < a.n_seq && a.off[s] < p.r0;
    const int64_t end = came ? a.off[s + 1] : p.r0;
    if (blockIdx.x % a.tiles == 0 && threadIdx.x == 0) a.kind[p.chunk] = !came ? 0 : end > p.r1 && p.chunk + 1 < a.chunks ? 2 : 1;
    if (!came) return;
    const int64_t to = end < p.r1 ? end : p.r1;
    float A2[4], g[4], span = 0.0f;
    load_states<LN>(a.A, 0, a, p.d, p.lane_n, p.on, A2);
#pragma unroll
    for (int e = 0; e < 4; e++) A2[e] *= REC_LOG2E;
    load_states<LN>(end <= p.r1 ? a.dfinal : nullptr, s, a, p.d, p.lane_n, p.on, g);
    Tile<T, LN, false, true, true, false, true> t;
    const int ch = t.channel();
    const bool mine = ch < p.nch;
    const float bias = mine && a.delta_bias ? a.delta_bias[p.ch0 + ch] : 0.0f;
    int64_t t0 = p.r0 + (to - 1 - p.r0) / TT * TT;
    t.fetch(a, p, t0);
    for (; t0 >= p.r0; t0 -= TT) {
        __syncthreads();
#pragma unroll
        for (int k = 0; k < t.PT; k++) {
            const bool counts = mine && t0 + t.row(k) < to;
            const float raw = to_f32(t.d[k]) + bias, sp = computed(softplus_f32(raw)), delta = a.softplus ? sp : raw, gy = to_f32(t.g[k]), gate = computed(silu_f32(to_f32(t.z[k])));
            sd[t.row(k)][ch] = counts ? make_float2(delta, a.z ? gy * gate : gy) : make_float2(0.0f, 0.0f);
        }
        t.stage_groups(a, t0, t0, to, nullptr, sC);
        __syncthreads();
        if (t0 > p.r0) t.fetch(a, p, t0 - TT);
#pragma unroll
        for (int r = TT - 1; r >= 0; r--) {   // rows behind the history's last move nothing
            const float2 v = sd[r][p.ch];
            span += v.x;
#pragma unroll
            for (int e = 0; e < 4; e++) g[e] = fast_exp2(v.x * A2[e]) * fmaf(sC[r][p.lane_n + e], v.y, g[e]);
        }
    }
    store_states<LN>(a.link, p.chunk, a, p.d, p.lane_n, p.on, g);
    if (p.on && p.lane_n == 0) a.span[(int64_t)p.chunk * a.channels + p.d] = span;
}

// zeros instead of h, without a branch
__device__ __forceinline__ void clear_if(float (&h)[4], bool clear)
{
    unsigned keep = __builtin_amdgcn_readfirstlane(clear ? 0u : ~0u);
    asm volatile("" : "+s"(keep));   // or the cleared states of the walk forwards would be kept, next to the states, for the one backwards
#pragma unroll
    for (int e = 0; e < 4; e++) h[e] = __uint_as_float(__float_as_uint(h[e]) & keep);
}

// What is staged in LDS is read again behind this line: without it the compiler keeps all that the walk forwards has read
// (160 registers) for the walk backwards.
#define REC_READ_AGAIN()                          \
    do {                                          \
        asm volatile("" ::: "memory");            \
        __builtin_amdgcn_sched_barrier(0);        \
    } while (0)

// third pass of the gradient: per 16 rows, the states again from the checkpoint in front of them, then the gradient backwards.  A lane keeps the
// tile's states in registers (64 of them).  Keeping the decays as well left room for one wavefront per SIMD instead of three.  (Two
// with 128 channels: their LDS leaves room for two blocks.)
// With states handed in or out (STATES) the lookups and loads at each history's beginning, in all three walks, take 182 to 227 registers,
// some hundred scalars beyond those there are, and two wavefronts: 400 to 414 us for 40 000 rows of 128 bf16 channels in 8000 histories,
// vector instructions issued in 28 % of the cycles.
template <class T, int LN, bool STATES>
__global__ __launch_bounds__(256, STATES || LN == 2 ? 2 : 3) void scan_backward_kernel(ScanArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {
        pass_empty(a, a.dfinal, a.dinitial);
        return;
    }
    using P = Place<LN>;
    using Q = Tile<T, LN, true, true, true, true, true>;
    constexpr int CH = P::CH, NP = 4 * LN, PT = Q::PT, ROW = CH + 16, GR = rows_together<LN>();
    __shared__ float2 sd[TT][CH];                  // delta, delta * u
    __shared__ float sg[TT][CH];                   // dys
    __shared__ alignas(16) float sB[TT][NP], sC[TT][NP];
    __shared__ float s_in[TT][ROW], s_gB[TT][ROW], s_qA[TT][ROW];
    __shared__ alignas(16) float s_bc[4][TT][2][NP];           // dB, dC of each wavefront's channels
    __shared__ float s_own[3][PT][256];            // what a thread wants back after the walk: u, the derivative of softplus, dy times the derivative of the gate
    const P p(a);
    const int64_t lo = a.off[0], hi = a.off[a.n_seq];
    float A2[4], G[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dA[4] = {0.0f, 0.0f, 0.0f, 0.0f}, dD = 0.0f, dbias = 0.0f;
    load_states<LN>(a.A, 0, a, p.d, p.lane_n, p.on, A2);
#pragma unroll
    for (int e = 0; e < 4; e++) A2[e] *= REC_LOG2E;
    // the sequence (n_seq: none) of the row at hand, walking backwards, and its first row
    int s = sequence_of(a.off, a.n_seq, p.r1 - 1);
    int64_t begin = s >= 0 ? a.off[s] : -1;
    if (s >= 0 && s < a.n_seq) {
        if (a.off[s + 1] <= p.r1) load_states<LN>(a.dfinal, s, a, p.d, p.lane_n, p.on, G);
        else if (p.chunk + 1 < a.chunks) load_states<LN>(a.link, p.chunk + 1, a, p.d, p.lane_n, p.on, G);
    }
    auto step_back = [&](int& q, int64_t& b) {   // to the sequence in front, past empty ones
        const int64_t at = b;
        q--;
        if (q >= 0 && a.off[q] >= at) {
            int low = -1, high = q - 1;
            while (low < high) {
                const int mid = low + ((high - low + 1) >> 1);
                if (a.off[mid] < at) low = mid; else high = mid - 1;
            }
            q = low;
        }
        b = q >= 0 ? a.off[q] : -1;
    };
    const int wave = threadIdx.x >> 6, lane = threadIdx.x & 63;
    const int ch = Q::channel(), d = p.ch0 + ch;
    const bool mine = ch < p.nch;
    const float bias = mine && a.delta_bias ? a.delta_bias[d] : 0.0f, Dd = mine && a.D ? a.D[d] : 0.0f;
    for (int64_t t0 = (p.r1 - 1) / TT * TT; t0 >= p.r0; t0 -= TT) {
        const int nt = (int)(p.r1 - t0 < TT ? p.r1 - t0 : TT);
        unsigned bounds = 0;   // the tile's rows that begin a sequence, or the rows behind the last one
        int q = s;
        for (int64_t b = begin; b >= t0;) {
            if (b < t0 + nt) bounds |= 1u << (b - t0);
            if (b == t0) break;
            step_back(q, b);
        }
        bounds = __builtin_amdgcn_readfirstlane(bounds);   // the same in every lane
        Q t;
        t.fetch(a, p, t0);
        float h0[4];   // the state in front of the tile
        load_states<LN>(a.checkpoints_in, t0 / TT, a, p.d, p.lane_n, p.on, h0);
        const int64_t blo = lo > t0 ? lo : t0, bhi = hi < t0 + nt ? hi : t0 + nt;
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int r = Q::row(k);
            const bool counts = mine && t0 + r >= blo && t0 + r < bhi;
            const float raw = to_f32(t.d[k]) + bias, gy = to_f32(t.g[k]), z = to_f32(t.z[k]);
            const float sp = computed(softplus_f32(raw)), ss = computed(sigmoid_f32(raw)), sz = computed(sigmoid_f32(z));
            const float delta = a.softplus ? sp : raw;
            const float u = to_f32(t.u[k]);
            s_own[0][k][threadIdx.x] = u;
            s_own[1][k][threadIdx.x] = a.softplus ? ss : 1.0f;
            s_own[2][k][threadIdx.x] = gy * (sz * fmaf(z, 1.0f - sz, 1.0f));
            sd[r][ch] = counts ? make_float2(delta, delta * u) : make_float2(0.0f, 0.0f);
            sg[r][ch] = counts ? (a.z ? gy * (z * sz) : gy) : 0.0f;
        }
        t.stage_groups(a, t0, blo, bhi, sB, sC);
        __syncthreads();
        // Half a tile at a time, the later half first, so that only eight rows' states are kept (with sixteen there is room for two
        // wavefronts per SIMD instead of three).  A tile in which no history begins is walked without a look at the bounds.
        auto walk = [&](auto bounded) {
            constexpr bool BOUNDED = decltype(bounded)::value;
            // the state of row r from the one in front of it
            auto enter = [&](int r, float (&h)[4]) {
                if (!BOUNDED) return;
                const bool bound = (bounds >> r) & 1;
                if (!STATES) {
                    clear_if(h, bound);
                } else if (bound) {
                    const int at = sequence_of(a.off, a.n_seq, t0 + r);
                    load_states<LN>(at >= 0 && at < a.n_seq ? a.initial : nullptr, at, a, p.d, p.lane_n, p.on, h);
                }
            };
#pragma unroll 1
            for (int half = TT - HALF; half >= 0; half -= HALF) {
                float h[4], first[4], hs[HALF][4];   // the state in front of the half, and behind each of its rows
#pragma unroll
                for (int e = 0; e < 4; e++) h[e] = h0[e];
                if (half > 0) {
#pragma unroll
                    for (int r = 0; r < HALF; r++) {
                        enter(r, h);
                        const float2 v = sd[r][p.ch];
#pragma unroll
                        for (int e = 0; e < 4; e++) h[e] = fmaf(fast_exp2(v.x * A2[e]), h[e], v.y * sB[r][p.lane_n + e]);
                    }
                }
#pragma unroll
                for (int e = 0; e < 4; e++) first[e] = h[e];
#pragma unroll
                for (int r0 = 0; r0 < HALF; r0 += GR) {
                    float y[GR];
#pragma unroll
                    for (int k = 0; k < GR; k++) {
                        const int i = r0 + k, r = half + i;
                        if (i % 4 == 0) REC_READ_AGAIN();
#pragma unroll
                        for (int e = 0; e < 4; e++) h[e] = i == 0 ? first[e] : hs[i > 0 ? i - 1 : 0][e];
                        enter(r, h);
                        const float2 v = sd[r][p.ch];
                        y[k] = 0.0f;
#pragma unroll
                        for (int e = 0; e < 4; e++) {
                            hs[i][e] = fmaf(fast_exp2(v.x * A2[e]), h[e], v.y * sB[r][p.lane_n + e]);
                            y[k] = fmaf(hs[i][e], sC[r][p.lane_n + e], y[k]);
                        }
                    }
                    if (a.z) write_sums<LN, GR>(s_in, half + r0, p.ch, y);
                }
                float vB[2][4], vC[2][4], gB[GR], qA[GR];
#pragma unroll
                for (int i = HALF - 1; i >= 0; i--) {
                    const int r = half + i;
                    if (i % 2 == 1) REC_READ_AGAIN();
                    const float2 v = sd[r][p.ch];
                    const float ys = sg[r][p.ch];
                    float hb[4];
#pragma unroll
                    for (int e = 0; e < 4; e++) hb[e] = i == 0 ? first[e] : hs[i > 0 ? i - 1 : 0][e];
                    enter(r, hb);
                    gB[i % GR] = qA[i % GR] = 0.0f;
#pragma unroll
                    for (int e = 0; e < 4; e++) {
                        const float b = sB[r][p.lane_n + e];
                        const float g = fmaf(sC[r][p.lane_n + e], ys, G[e]);
                        vB[i % 2][e] = g * v.y;
                        vC[i % 2][e] = hs[i][e] * ys;
                        gB[i % GR] = fmaf(g, b, gB[i % GR]);
                        G[e] = fast_exp2(v.x * A2[e]) * g;
                        const float q = G[e] * hb[e];
                        qA[i % GR] = fmaf(q, A2[e], qA[i % GR]);   // (A, times ln 2 below)
                        dA[e] = fmaf(q, v.x, dA[e]);
                    }
                    if (BOUNDED) {
                        const bool bound = (bounds >> r) & 1;
                        if (!STATES) {
                            clear_if(G, bound);
                        } else if (bound) {   // in front of this row another sequence ends, or none does
                            if (s >= 0 && s < a.n_seq && a.dinitial) store_states<LN>(a.dinitial, s, a, p.d, p.lane_n, p.on, G);
                            step_back(s, begin);
                            load_states<LN>(s >= 0 ? a.dfinal : nullptr, s, a, p.d, p.lane_n, p.on, G);
                        }
                    }
                    if (i % GR == 0) {
                        write_sums<LN, GR>(s_gB, r, p.ch, gB);
                        write_sums<LN, GR>(s_qA, r, p.ch, qA);
                    }
                    if (i % 2 == 0) {
                        // Two rows' 16 values, over the wavefront's channels: each fold halves the values and leaves the halves of the
                        // lanes with different ones (bit 5 of the lane: the row, bit 4: dB or dC); what is left is summed inside 16 lanes.
                        float w[4];
#pragma unroll
                        for (int e = 0; e < 4; e++) w[e] = row_sum_strided<LN>(fold16(fold32(vB[0][e], vB[1][e]), fold32(vC[0][e], vC[1][e])));
                        float* to = s_bc[wave][r + (lane >> 5)][(lane >> 4) & 1] + p.lane_n;
                        const int copy = lane % 16 / LN;   // lanes with the same sums
                        if constexpr (LN <= 4) {
                            const float mine4 = copy == 0 ? w[0] : copy == 1 ? w[1] : copy == 2 ? w[2] : w[3];
                            if (copy < 4) to[copy] = mine4;
                        } else if constexpr (LN == 8) {
                            *reinterpret_cast<float2*>(to + 2 * copy) = copy ? make_float2(w[2], w[3]) : make_float2(w[0], w[1]);
                        } else {
                            *reinterpret_cast<float4*>(to) = make_float4(w[0], w[1], w[2], w[3]);
                        }
                    }
                }
            }
        };
        if (bounds == 0) walk(std::false_type{});
        else walk(std::true_type{});
        if (!STATES)
            while (begin >= t0) { if (begin == 0) break; step_back(s, begin); }
        __syncthreads();
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int r = Q::row(k);
            const int64_t row = t0 + r, at = row * a.channels + d;
            if (r >= nt || !mine) continue;
            if (row < lo || row >= hi) {
                if (a.zero_rest) {
                    ((T*)a.du)[at] = ((T*)a.ddelta)[at] = from_f32<T>(0.0f);
                    if (a.z) ((T*)a.dz)[at] = from_f32<T>(0.0f);
                }
                continue;
            }
            const float2 v = sd[r][ch];
            const float ys = sg[r][ch], g = s_gB[r][ch];
            const float u = s_own[0][k][threadIdx.x];
            const float dd = fmaf(u, g, s_qA[r][ch] * 0.69314718055994530942f) * s_own[1][k][threadIdx.x];
            ((T*)a.du)[at] = from_f32<T>(a.D ? fmaf(v.x, g, Dd * ys) : v.x * g);
            ((T*)a.ddelta)[at] = from_f32<T>(dd);
            if (a.z) ((T*)a.dz)[at] = from_f32<T>(s_own[2][k][threadIdx.x] * (a.D ? fmaf(Dd, u, s_in[r][ch]) : s_in[r][ch]));
            dD = fmaf(ys, u, dD);
            dbias += dd;
        }
        // dB and dC of the block's channels: the four wavefronts in order
        for (int i = threadIdx.x; i < TT * 2 * NP; i += 256) {
            const int r = i / (2 * NP), w = i / NP % 2, n = i % NP;
            const int64_t row = t0 + r;
            if (r >= nt || n >= a.states) continue;
            const float v = (s_bc[0][r][w][n] + s_bc[1][r][w][n]) + (s_bc[2][r][w][n] + s_bc[3][r][w][n]);
            if (a.tiles_per_group > 1) {
                a.part_bc[((((int64_t)p.part * a.rows + row) * a.groups + p.g) * 2 + w) * a.states + n] = v;
            } else if ((row >= lo && row < hi) || a.zero_rest) {
                ((T*)(w ? a.dC : a.dB))[(row * a.groups + p.g) * a.states + n] = from_f32<T>(v);
            }
        }
    }
    if (!a.part_a) return;
    float* part = a.part_a + (int64_t)p.chunk * (a.channels * a.states + 2 * a.channels);
    store_states<LN>(part, 0, a, p.d, p.lane_n, p.on, dA);
    // a thread's pairs are of one channel: the threads of a channel in order
    __syncthreads();
    float *red_D = &s_in[0][0], *red_b = &s_gB[0][0];   // 16 * CH >= 256 each
    red_D[threadIdx.x] = dD;
    red_b[threadIdx.x] = dbias;
    __syncthreads();
    if ((int)threadIdx.x < p.nch) {
        float x = 0.0f, y = 0.0f;
        for (int k = threadIdx.x; k < 256; k += CH) { x += red_D[k]; y += red_b[k]; }
        part[a.channels * a.states + p.ch0 + threadIdx.x] = x;
        part[a.channels * a.states + a.channels + p.ch0 + threadIdx.x] = y;
    }
}

// dB and dC where a group's channels are spread over blocks: 32 rows a block, a row's values on neighbouring threads
constexpr int SUM_ROWS = 32;
template <class T>
__global__ __launch_bounds__(256) void scan_sum_groups_kernel(ScanArgs a)
{
    const int per_row = a.groups * 2 * a.states, n = per_row * SUM_ROWS;
    const int64_t row0 = (int64_t)blockIdx.x * SUM_ROWS, lo = a.off[0], hi = a.off[a.n_seq];
    const float* part = a.part_bc + row0 * per_row;
    for (int i = threadIdx.x; i < n; i += 256) {
        const int r = i / per_row, at = i - r * per_row, pair = at / a.states, v = at - pair * a.states;   // pair: group * 2 + (B or C)
        const int64_t row = row0 + r;
        if (row >= a.rows || ((row < lo || row >= hi) && !a.zero_rest)) continue;
        float sum = 0.0f;
        for (int k = 0; k < a.tiles_per_group; k++) sum += part[k * (a.rows * per_row) + i];
        ((T*)(pair & 1 ? a.dC : a.dB))[(row * a.groups + pair / 2) * a.states + v] = from_f32<T>(sum);
    }
}

// ---- single clicks: a block per row; bound by the state, which is read and written once (4 bytes a value each way), and by
// the waits in between (1000 rows of 256 channels with 16 states: 10 us, 3.4 TB/s).  Four pieces of 256 / LN channels at a time: a thread prepares whole channels (delta, delta * u, the gate), then
// takes four states of one channel of each piece, and everything a row needs is asked for at once, before the block looks for
// other rows of its slot.
// The code is kept short (one copy of everything; WHOLE: all 4 LN states of a lane group exist and lie on boundaries of four): a
// launch this small waits for its instructions, too.
constexpr int PIECES = 4;
template <class T, int LN, bool WHOLE>
__global__ __launch_bounds__(256) void scan_step_kernel(ScanArgs a, const int32_t* __restrict__ slots, float* state)
{
    struct alignas(4) Four { float v[4]; };
    constexpr int CH = 256 / LN, ALL = PIECES * CH, PT = ALL > 256 ? ALL / 256 : 1;
    __shared__ float2 sd[ALL];
    __shared__ float sy[ALL];
    __shared__ unsigned seen[4];
    const int row = blockIdx.x, rows = (int)a.rows;
    const int ch = threadIdx.x / LN, n0 = threadIdx.x % LN * 4;
    const int slot = slots[row];
    const bool valid = slot >= 0 && slot < a.n_seq;
    // (a row without a slot reads A in the state's place - a pool may be empty - and stores nothing)
    float* pool = valid ? state + (int64_t)slot * a.channels * a.states : const_cast<float*>(a.A);
    auto states = [&](const float* p, int d, float (&v)[4]) {   // of a channel that exists
        if (WHOLE) {
            const Four f = *reinterpret_cast<const Four*>(p + d * a.states + n0);
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = f.v[e];
        } else {
#pragma unroll
            for (int e = 0; e < 4; e++) v[e] = p[d * a.states + min(n0 + e, a.states - 1)];
        }
    };
    for (int tile0 = 0; tile0 < a.tiles; tile0 += PIECES) {
        int group[PIECES], first[PIECES], count[PIECES];   // a piece's group, first channel and channels: scalars
#pragma unroll
        for (int k = 0; k < PIECES; k++) {
            const int tile = min(tile0 + k, a.tiles - 1);
            group[k] = a.groups == 1 ? 0 : tile / a.tiles_per_group;
            const int part = (tile - group[k] * a.tiles_per_group) * CH;
            first[k] = group[k] * a.per + part;
            count[k] = tile0 + k < a.tiles ? min(CH, a.per - part) : 0;
        }
        int mine[PT];
#pragma unroll
        for (int k = 0; k < PT; k++) {
            const int v = threadIdx.x + 256 * k, q = v / CH;
            mine[k] = -1;
#pragma unroll
            for (int i = 0; i < PIECES; i++)
                if (q == i && v % CH < count[i]) mine[k] = first[i] + v % CH;
        }
        for (int r = row;;) {
            T rd[PT], ru[PT], rz[PT];
            Pack<T, 4> rb[PIECES], rc[PIECES];
            float bias[PT], D[PT], h[PIECES][4], A[PIECES][4];
#pragma unroll
            for (int k = 0; k < PT; k++) {
                const int at = mine[k] < 0 ? 0 : mine[k];
                rd[k] = ((const T*)a.delta + r * a.delta_stride)[at];
                ru[k] = ((const T*)a.u + r * a.u_stride)[at];
                rz[k] = ((const T*)(a.z ? a.z : a.u) + r * (a.z ? a.z_stride : a.u_stride))[at];
                bias[k] = a.delta_bias ? a.delta_bias[at] : 0.0f;
                D[k] = a.D ? a.D[at] : 0.0f;
            }
#pragma unroll
            for (int k = 0; k < PIECES; k++) {   // (a row of a shared slot finds the state as the one before it has left it: in memory)
                const int d = first[k] + min(ch, max(count[k], 1) - 1);
                states(a.A, d, A[k]);
                states(pool, d, h[k]);
                const T *b = (const T*)a.B + r * a.B_stride + group[k] * a.states, *c = (const T*)a.C + r * a.C_stride + group[k] * a.states;
                if (WHOLE) {
                    rb[k] = *reinterpret_cast<const Pack<T, 4>*>(b + n0);
                    rc[k] = *reinterpret_cast<const Pack<T, 4>*>(c + n0);
                } else {
#pragma unroll
                    for (int e = 0; e < 4; e++) { rb[k].v[e] = b[min(n0 + e, a.states - 1)]; rc[k].v[e] = c[min(n0 + e, a.states - 1)]; }
                }
            }
            if (r == row && tile0 == 0) look_for_slot(slots, a.rows, row, slot, seen);
            float gate[PT], u[PT];
#pragma unroll
            for (int k = 0; k < PT; k++) {
                const float raw = to_f32(rd[k]) + bias[k], sp = computed(softplus_f32(raw)), delta = a.softplus ? sp : raw;
                u[k] = to_f32(ru[k]);
                gate[k] = computed(silu_f32(to_f32(rz[k])));
                if (PT > 1 || (int)threadIdx.x < ALL) sd[threadIdx.x + 256 * k] = make_float2(delta, delta * u[k]);
            }
            __syncthreads();
            const unsigned shared = slots_seen(seen);
            if (valid && (shared & 1)) return;   // the first row of a slot takes the others along
#pragma unroll
            for (int k = 0; k < PIECES; k++) {
                const float2 v = sd[k * CH + ch];
                float y = 0.0f;
#pragma unroll
                for (int e = 0; e < 4; e++) {
                    h[k][e] = fmaf(fast_exp2(v.x * (A[k][e] * REC_LOG2E)), h[k][e], v.y * to_f32(rb[k].v[e]));
                    if (WHOLE || n0 + e < a.states) y = fmaf(h[k][e], to_f32(rc[k].v[e]), y);
                }
                if (valid && ch < count[k]) {
                    float* p = pool + (first[k] + ch) * a.states + n0;
                    if (WHOLE) *reinterpret_cast<Four*>(p) = Four{{h[k][0], h[k][1], h[k][2], h[k][3]}};
                    else
#pragma unroll
                        for (int e = 0; e < 4; e++)
                            if (n0 + e < a.states) p[e] = h[k][e];
                }
                y = group_sum_dpp<LN>(y);
                if (n0 == 0) sy[k * CH + ch] = y;
            }
            __syncthreads();
#pragma unroll
            for (int k = 0; k < PT; k++) {
                if (mine[k] < 0) continue;
                float y = sy[threadIdx.x + 256 * k];
                if (a.D) y = fmaf(D[k], u[k], y);
                if (a.z) y *= gate[k];
                ((T*)a.y)[r * a.y_stride + mine[k]] = from_f32<T>(valid ? y : 0.0f);
            }
            if (!valid || !(shared & 2)) break;
            r = next_row_of(slots, rows, r, slot);
            if (r >= rows) break;
        }
    }
}

// ---- host
int check_desc(const rec_scan_desc* d)
{
    REC_REFUSE(!d, "null argument");
    REC_REFUSE(d->type < REC_TYPE_F32 || d->type > REC_TYPE_BF16, "unknown type");
    REC_REFUSE(d->rows < 0 || d->rows > INT32_MAX, "rows must be in 0..2^31-1");
    REC_REFUSE(d->n_seq < 0 || d->n_seq == INT32_MAX, "n_seq must be in 0..2^31-2");
    REC_REFUSE(d->channels < 1 || d->channels > 1 << 20, "channels must be in 1..2^20");
    REC_REFUSE(d->groups < 1 || d->channels % d->groups, "groups must divide the channels");
    REC_REFUSE(d->states < 1 || d->states > 64, "states must be in 1..64");
    return 0;
}

int check_inputs(const rec_scan_desc* d, const rec_scan_inputs* in)
{
    REC_REFUSE(!in || !in->A || (d->rows > 0 && (!in->u || !in->delta || !in->B || !in->C)), "null argument");
    const int64_t n = (int64_t)d->groups * d->states;
    REC_REFUSE(in->u_stride < d->channels || in->delta_stride < d->channels || (in->z && in->z_stride < d->channels), "a row stride is smaller than the channels");
    REC_REFUSE(in->B_stride < n || in->C_stride < n, "a row stride is smaller than groups x states");
    REC_REFUSE(in->u_stride > INT32_MAX || in->delta_stride > INT32_MAX || in->z_stride > INT32_MAX || in->B_stride > INT32_MAX || in->C_stride > INT32_MAX,
               "a row stride is beyond 2^31-1");
    return 0;
}

bool overlaps_inputs(const rec_scan_desc* d, const rec_scan_inputs* in, const RowsOf& out)
{
    const int64_t e = rec_type_size(d->type), w = d->channels * e, n = (int64_t)d->groups * d->states * e;
    const RowsOf ins[5] = {{in->u, d->rows, in->u_stride * e, w}, {in->delta, d->rows, in->delta_stride * e, w}, {in->z, d->rows, in->z_stride * e, w},
                           {in->B, d->rows, in->B_stride * e, n}, {in->C, d->rows, in->C_stride * e, n}};
    for (const RowsOf& i : ins)
        if (rec_overlap(i, out)) return true;
    return false;
}

RowsOf channel_rows(const rec_scan_desc* d, const void* p, int64_t stride)
{
    const int64_t e = rec_type_size(d->type);
    return {p, d->rows, stride * e, d->channels * e};
}

int64_t state_bytes(const rec_scan_desc* d) { return (int64_t)d->n_seq * d->channels * d->states * 4; }

int lanes_of(const rec_scan_desc* d) { return d->states <= 4 ? 1 : d->states <= 8 ? 2 : d->states <= 16 ? 4 : d->states <= 32 ? 8 : 16; }
// The passes over histories take two lanes at least, and more, idle ones too, where the group's channels fill half a block or less: a
// block with fewer channels stages and keeps less.  (The gradient's last pass, bf16, 4 states: 50 000 rows of 256 channels 230 us with
// one lane, whose LDS leaves room for one block on a compute unit, 187 with two, 240 with four; 100 000 rows of 100 channels 404 and
// 186 us with one and two; f32, 16 575 rows of 31 channels 86 and 32 us with one and eight.)
int pass_lanes(const rec_scan_desc* d)
{
    int lanes = d->states <= 4 ? 2 : lanes_of(d);
    while (lanes < 16 && 256 / (2 * lanes) >= d->channels / d->groups) lanes *= 2;
    return lanes;
}

// How the rows are cut.  A chunk more costs its first pass (two thirds of the third, over the chunk's last history) and a state
// handed over, so chunks are as long as they can be while the launch still fills the chip: `blocks` of them, between 16 and
// 512 rows.
struct Cut { int tiles_per_group, tiles, chunk, chunks; };
constexpr int kForwardBlocks = 2048, kBackwardBlocks = 3000;
Cut cut_of(const rec_scan_desc* d, int blocks, int lanes)
{
    Cut c;
    const int ch = 256 / lanes, per = d->channels / d->groups;
    c.tiles_per_group = (per + ch - 1) / ch;
    c.tiles = c.tiles_per_group * d->groups;
    int64_t rows = d->rows * c.tiles / blocks / TT * TT;
    if (rows < 16) rows = 16;
    if (rows > 512) rows = 512;
    c.chunk = (int)rows;
    c.chunks = (int)((d->rows + rows - 1) / rows);
    return c;
}

int64_t link_bytes(const rec_scan_desc* d, const Cut& c)
{
    return c.chunks > 1 ? (int64_t)c.chunks * ((int64_t)d->channels * d->states + d->channels + 1) * 4 : 0;
}

void fill(ScanArgs& a, const rec_scan_desc* d, const rec_scan_inputs* in, const Cut& c)
{
    a.u = in->u; a.delta = in->delta; a.z = in->z; a.B = in->B; a.C = in->C; a.A = in->A; a.D = in->D; a.delta_bias = in->delta_bias; a.initial = in->initial;
    a.u_stride = in->u_stride; a.delta_stride = in->delta_stride; a.z_stride = in->z_stride; a.B_stride = in->B_stride; a.C_stride = in->C_stride;
    a.rows = d->rows; a.n_seq = d->n_seq; a.channels = d->channels; a.groups = d->groups; a.per = d->channels / d->groups; a.states = d->states;
    a.chunk = c.chunk; a.chunks = c.chunks; a.tiles = c.tiles; a.tiles_per_group = c.tiles_per_group; a.softplus = d->softplus; a.zero_rest = d->zero_rest;
}

int check_blocks(int64_t blocks)
{
    REC_REFUSE(blocks > (1ll << 24) - 1, "too many rows, channels or sequences for one call");   // a launch holds fewer than 2^32 threads
    return 0;
}

// a launch for n columns, `cols` to a block, `times` threads a column: as many blocks of 256 threads as that would be
int64_t in_blocks(int64_t n, int64_t cols, int64_t times) { return (n + cols - 1) / cols * (cols * times / 256); }

int check_workspace(const void* p, int64_t has, int64_t needs)
{
    REC_REFUSE(has < needs, "the workspace is too small");
    REC_REFUSE(needs > 0 && (!p || !rec_aligned(p, 16)), "the workspace is null or not aligned to 16 bytes");
    return 0;
}

#define SCAN_TYPES(LANES, CALL)                                                                             \
    if (d->type == REC_TYPE_F32) { LANES(float, CALL) }                                                     \
    else if (d->type == REC_TYPE_F16) { LANES(_Float16, CALL) }                                             \
    else { LANES(__bf16, CALL) }
#define SCAN_PASS_LANES(T, CALL)                                                                            \
    switch (pass_lanes(d)) {                                                                                \
    case 2: CALL(T, 2); break; case 4: CALL(T, 4); break; case 8: CALL(T, 8); break; default: CALL(T, 16); break; \
    }
#define SCAN_STEP_LANES(T, CALL)                                                                            \
    switch (lanes_of(d)) {                                                                                  \
    case 1: CALL(T, 1); break; case 2: CALL(T, 2); break; case 4: CALL(T, 4); break;                        \
    case 8: CALL(T, 8); break; default: CALL(T, 16); break;                                                 \
    }

}  // namespace

extern "C" int64_t rec_history_scan_workspace(const rec_scan_desc* d)
{
    return rec_guarded([&]() -> int64_t {
        if (check_desc(d)) return -1;
        return link_bytes(d, cut_of(d, kForwardBlocks, pass_lanes(d)));
    });
}

extern "C" int rec_history_scan(const rec_scan_desc* d, const rec_scan_inputs* in, const int64_t* seq_off, void* y, int64_t y_stride,
                                float* final_state, float* checkpoints, void* workspace, int64_t workspace_bytes, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        if (int rc = check_inputs(d, in)) return rc;
        REC_REFUSE(!seq_off || (d->rows > 0 && !y), "null argument");
        REC_REFUSE(y_stride < d->channels || y_stride > INT32_MAX, "a row stride is smaller than the channels, or beyond 2^31-1");
        REC_REFUSE(overlaps_inputs(d, in, channel_rows(d, y, y_stride)), "the output overlaps an input");
        REC_REFUSE(rec_overlap(in->initial, state_bytes(d), final_state, state_bytes(d)), "final_state overlaps initial");
        const Cut c = cut_of(d, kForwardBlocks, pass_lanes(d));
        if (int rc = check_workspace(workspace, workspace_bytes, link_bytes(d, c))) return rc;
        const int64_t blocks = (int64_t)c.chunks * c.tiles, n = (int64_t)d->channels * d->states;
        const bool many_states = final_state && n * d->n_seq >= kManyStates;
        const int64_t empty_blocks = final_state && !many_states ? (n * d->n_seq + 255) / 256 : 0;
        if (int rc = check_blocks(blocks + empty_blocks)) return rc;
        if (int rc = check_blocks(c.chunks > 1 ? in_blocks(n, LINK_COLS, LINK_RUNS) : 0)) return rc;
        if (int rc = rec_check_device(d->device)) return rc;
        ScanArgs a = {};
        fill(a, d, in, c);
        a.off = seq_off; a.y = y; a.y_stride = y_stride; a.final_state = final_state; a.checkpoints = checkpoints;
        a.main_blocks = (int)blocks;
        a.link = (float*)workspace;
        a.span = a.link + c.chunks * n;
        a.kind = (int*)(a.span + (int64_t)c.chunks * d->channels);
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        hipStream_t st = (hipStream_t)stream;
        if (c.chunks > 1) {
#define CALL(T, LN) scan_local_kernel<T, LN><<<(unsigned)blocks, 256, 0, st>>>(a)
            SCAN_TYPES(SCAN_PASS_LANES, CALL)
#undef CALL
            scan_link_kernel<false><<<(unsigned)((n + LINK_COLS - 1) / LINK_COLS), LINK_COLS * LINK_RUNS, 0, st>>>(a);
        }
        if (blocks + empty_blocks > 0) {
#define CALL(T, LN) scan_forward_kernel<T, LN><<<(unsigned)(blocks + empty_blocks), 256, 0, st>>>(a)
            SCAN_TYPES(SCAN_PASS_LANES, CALL)
#undef CALL
        }
        if (many_states) scan_pass_empty_kernel<<<kManyStates / 256, 256, 0, st>>>(a, a.initial, a.final_state);
        HIP_TRY(hipGetLastError());
        return 0;
    });
}

static int64_t backward_part_a(const rec_scan_desc* d, const Cut& c) { return (int64_t)c.chunks * ((int64_t)d->channels * d->states + 2 * d->channels) * 4; }
static int64_t backward_part_bc(const rec_scan_desc* d, const Cut& c) { return c.tiles_per_group > 1 ? (int64_t)c.tiles_per_group * d->rows * d->groups * 2 * d->states * 4 : 0; }
static int64_t round16(int64_t n) { return (n + 15) / 16 * 16; }

extern "C" int64_t rec_history_scan_backward_workspace(const rec_scan_desc* d)
{
    return rec_guarded([&]() -> int64_t {
        if (check_desc(d)) return -1;
        const Cut c = cut_of(d, kBackwardBlocks, pass_lanes(d));
        return round16(link_bytes(d, c)) + round16(backward_part_a(d, c)) + backward_part_bc(d, c);
    });
}

extern "C" int rec_history_scan_backward(const rec_scan_desc* d, const void* dy, int64_t dy_stride, const rec_scan_inputs* in,
                                         const int64_t* seq_off, const float* checkpoints, const float* dfinal, const rec_scan_gradients* out,
                                         void* workspace, int64_t workspace_bytes, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        if (int rc = check_inputs(d, in)) return rc;
        REC_REFUSE(!seq_off || !out || (d->rows > 0 && (!dy || !checkpoints || !out->du || !out->ddelta || !out->dB || !out->dC || (in->z && !out->dz))), "null argument");
        REC_REFUSE(dy_stride < d->channels || dy_stride > INT32_MAX, "a row stride is smaller than the channels, or beyond 2^31-1");
        const int64_t group = (int64_t)rec_type_size(d->type) * d->groups * d->states;
        const RowsOf outs[5] = {channel_rows(d, out->du, d->channels), channel_rows(d, out->ddelta, d->channels), channel_rows(d, in->z ? out->dz : nullptr, d->channels),
                                {out->dB, d->rows, group, group}, {out->dC, d->rows, group, group}};
        for (int k = 0; k < 5; k++) {
            REC_REFUSE(overlaps_inputs(d, in, outs[k]) || rec_overlap(channel_rows(d, dy, dy_stride), outs[k]), "an output overlaps an input");
            for (int j = 0; j < k; j++) REC_REFUSE(rec_overlap(outs[j], outs[k]), "two outputs overlap");
        }
        REC_REFUSE(rec_overlap(in->initial, state_bytes(d), out->dinitial, state_bytes(d)) || rec_overlap(dfinal, state_bytes(d), out->dinitial, state_bytes(d)),
                   "dinitial overlaps initial or dfinal");
        if (int rc = check_workspace(workspace, workspace_bytes, rec_history_scan_backward_workspace(d))) return rc;
        const Cut c = cut_of(d, kBackwardBlocks, pass_lanes(d));
        const int64_t blocks = (int64_t)c.chunks * c.tiles, n = (int64_t)d->channels * d->states;
        const bool many_states = out->dinitial && n * d->n_seq >= kManyStates;
        const int64_t empty_blocks = out->dinitial && !many_states ? (n * d->n_seq + 255) / 256 : 0;
        const int64_t sum_blocks = c.tiles_per_group > 1 ? (d->rows + SUM_ROWS - 1) / SUM_ROWS : 0;
        const bool params = out->dA || out->dD || out->ddelta_bias;
        for (int64_t launch : {blocks + empty_blocks, sum_blocks, c.chunks > 1 ? in_blocks(n, LINK_COLS, LINK_RUNS) : 0, params ? sum_partials_blocks(n + 2 * d->channels) : 0})
            if (int rc = check_blocks(launch)) return rc;
        if (int rc = rec_check_device(d->device)) return rc;
        ScanArgs a = {};
        fill(a, d, in, c);
        a.off = seq_off; a.dy = dy; a.dy_stride = dy_stride; a.checkpoints_in = checkpoints; a.dfinal = dfinal;
        a.du = out->du; a.ddelta = out->ddelta; a.dz = out->dz; a.dB = out->dB; a.dC = out->dC; a.dinitial = out->dinitial;
        a.main_blocks = (int)blocks;
        char* ws = (char*)workspace;
        a.link = (float*)ws;
        a.span = a.link + c.chunks * n;
        a.kind = (int*)(a.span + (int64_t)c.chunks * d->channels);
        float* part_a = (float*)(ws + round16(link_bytes(d, c)));
        a.part_a = params ? part_a : nullptr;
        a.part_bc = (float*)(ws + round16(link_bytes(d, c)) + round16(backward_part_a(d, c)));
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        hipStream_t st = (hipStream_t)stream;
        if (c.chunks > 1) {
#define CALL(T, LN) scan_local_backward_kernel<T, LN><<<(unsigned)blocks, 256, 0, st>>>(a)
            SCAN_TYPES(SCAN_PASS_LANES, CALL)
#undef CALL
            scan_link_kernel<true><<<(unsigned)((n + LINK_COLS - 1) / LINK_COLS), LINK_COLS * LINK_RUNS, 0, st>>>(a);
        }
        if (blocks + empty_blocks > 0) {
            // without states handed in or out, a history's beginning is a zero
            if (in->initial || dfinal || out->dinitial) {
#define CALL(T, LN) scan_backward_kernel<T, LN, true><<<(unsigned)(blocks + empty_blocks), 256, 0, st>>>(a)
                SCAN_TYPES(SCAN_PASS_LANES, CALL)
#undef CALL
            } else {
#define CALL(T, LN) scan_backward_kernel<T, LN, false><<<(unsigned)(blocks + empty_blocks), 256, 0, st>>>(a)
                SCAN_TYPES(SCAN_PASS_LANES, CALL)
#undef CALL
            }
        }
        if (many_states) scan_pass_empty_kernel<<<kManyStates / 256, 256, 0, st>>>(a, a.dfinal, a.dinitial);
        if (sum_blocks > 0) {
            if (d->type == REC_TYPE_F32) scan_sum_groups_kernel<float><<<(unsigned)sum_blocks, 256, 0, st>>>(a);
            else if (d->type == REC_TYPE_F16) scan_sum_groups_kernel<_Float16><<<(unsigned)sum_blocks, 256, 0, st>>>(a);
            else scan_sum_groups_kernel<__bf16><<<(unsigned)sum_blocks, 256, 0, st>>>(a);
        }
        HIP_TRY(hipGetLastError());
        if (!params) return 0;
        return launch_sum_partials(part_a, c.chunks, n + 2 * d->channels, out->dA, n, out->dD, d->channels, out->ddelta_bias, st);
    });
}

extern "C" int rec_history_scan_step(const rec_scan_desc* d, const rec_scan_inputs* in, const int32_t* slots, float* state, void* y,
                                     int64_t y_stride, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        if (int rc = check_inputs(d, in)) return rc;
        REC_REFUSE(d->rows > 65536, "a step takes at most 65536 rows");
        REC_REFUSE((d->rows > 0 && (!y || !slots)) || (d->n_seq > 0 && !state), "null argument");
        REC_REFUSE(y_stride < d->channels || y_stride > INT32_MAX, "a row stride is smaller than the channels, or beyond 2^31-1");
        const RowsOf yr = channel_rows(d, y, y_stride), pool = {state, 1, INT64_MAX, state_bytes(d)};
        REC_REFUSE(overlaps_inputs(d, in, yr) || overlaps_inputs(d, in, pool) || rec_overlap(pool, yr), "the inputs, y and the state must not overlap");
        if (int rc = rec_check_device(d->device)) return rc;
        if (d->rows == 0) return 0;
        Cut c = cut_of(d, kForwardBlocks, lanes_of(d));
        c.chunk = 0; c.chunks = 0;
        ScanArgs a = {};
        fill(a, d, in, c);
        a.y = y; a.y_stride = y_stride;
        // four states of B and C in one load: no group's last four reach into the next, and all begin on a multiple of four
        const size_t four = 4 * (size_t)rec_type_size(d->type);
        const bool whole = d->states == 4 * lanes_of(d) && rec_aligned(in->B, four) && rec_aligned(in->C, four) && in->B_stride % 4 == 0 && in->C_stride % 4 == 0;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        const int64_t e = rec_type_size(d->type);
        auto behind = [&](const void* p, int64_t r, int64_t stride) -> const void* { return p ? (const char*)p + r * stride * e : nullptr; };
        for (int64_t r = 0; r < d->rows; r += kStepRows) {
            a.rows = d->rows - r < kStepRows ? d->rows - r : kStepRows;
            a.u = behind(in->u, r, a.u_stride); a.delta = behind(in->delta, r, a.delta_stride); a.z = behind(in->z, r, a.z_stride);
            a.B = behind(in->B, r, a.B_stride); a.C = behind(in->C, r, a.C_stride); a.y = (char*)y + r * y_stride * e;
            if (whole) {
#define CALL(T, LN) scan_step_kernel<T, LN, true><<<(unsigned)a.rows, 256, 0, (hipStream_t)stream>>>(a, slots + r, state)
                SCAN_TYPES(SCAN_STEP_LANES, CALL)
#undef CALL
            } else {
#define CALL(T, LN) scan_step_kernel<T, LN, false><<<(unsigned)a.rows, 256, 0, (hipStream_t)stream>>>(a, slots + r, state)
                SCAN_TYPES(SCAN_STEP_LANES, CALL)
#undef CALL
            }
        }
        HIP_TRY(hipGetLastError());
        return 0;
    });
}
