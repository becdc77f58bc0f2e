// Short causal convolution over packed histories: y, its gradient, and the form for single clicks.
//
//   v[t][d] = bias[d] + sum_{j < W} weight[d][j] x[t - (W-1) + j][d],   y = silu(v) or v
//
// About 2 W flop per element read and written, four times that in the gradient: bound by memory, the gradient by its vector
// instructions as much (issued in 68 % of its cycles, while it moves 3.4 TB/s).  A thread owns V neighbouring channels and walks a
// strip of consecutive rows with the window in registers, so a row is read once plus W-1 rows of halo per strip (these come from
// the cache), its loads a few rows ahead.  Where a history begins inside the strip, the window is replaced by that history's own.  A
// wavefront has one strip where the channels allow: what it knows of the histories is scalar then, and the registers hold windows
// (gradient over 598 655 x 128 bf16, W = 4: 88 registers and 134 us against 138 and 165 with a strip per thread).  V = 2: with V = 4
// the gradient takes 205 us, with 8 375, their registers leaving one or two wavefronts per SIMD.  The forward call over the same rows
// takes 69 us, 4.4 TB/s.
#include "operators.h"

namespace {

struct ConvArgs {
    const void *x, *initial, *dy, *dfinal;
    void *y, *final_window, *dx, *dinitial;
    const float *weight, *bias;
    const int64_t* off;
    float* partial;   // backward: [blocks][channels * W + channels] sums of dweight and dbias
    int64_t x_stride, y_stride, dy_stride, dx_stride;
    int64_t rows, strips;
    int n_seq, channels, nvec, ct, tiles, silu, zero_rest, strip_rows, main_blocks;
};

template <class T, int V> __device__ __forceinline__ void load_row(const void* base, int64_t at, float (&out)[V])
{
    const Pack<T, V> p = *reinterpret_cast<const Pack<T, V>*>((const T*)base + at);
#pragma unroll
    for (int v = 0; v < V; v++) out[v] = to_f32(p.v[v]);
}
template <class T, int V> __device__ __forceinline__ void store_row(void* base, int64_t at, const float (&in)[V])
{
    Pack<T, V> p;
#pragma unroll
    for (int v = 0; v < V; v++) p.v[v] = from_f32<T>(in[v]);
    *reinterpret_cast<Pack<T, V>*>((T*)base + at) = p;
}

template <int W, int V>
__device__ __forceinline__ void load_filter(const ConvArgs& a, int d, float (&w)[W][V], float (&b)[V])
{
#pragma unroll
    for (int v = 0; v < V; v++) {
#pragma unroll
        for (int j = 0; j < W; j++) w[j][v] = a.weight[(int64_t)(d + v) * W + j];
        b[v] = a.bias ? a.bias[d + v] : 0.0f;
    }
}

// the window of sequence s in front of row `row` (>= the sequence's first row, or a row of no sequence)
template <class T, int W, int V>
__device__ __forceinline__ void load_window(const ConvArgs& a, int s, int64_t start, int64_t row, int d, float (&win)[W - 1][V])
{
#pragma unroll
    for (int j = 0; j < W - 1; j++) {
        const int64_t at = row - (W - 1) + j;
        if (at >= start && at >= 0) {
            load_row<T, V>(a.x, at * a.x_stride + d, win[j]);
        } else {
            const int64_t q = at - start + (W - 1);
            if (a.initial && s >= 0 && s < a.n_seq && q >= 0 && q < W - 1) {
                load_row<T, V>(a.initial, ((int64_t)s * (W - 1) + q) * a.channels + d, win[j]);
            } else {
#pragma unroll
                for (int v = 0; v < V; v++) win[j][v] = 0.0f;
            }
        }
    }
}

// The windows that histories leave behind: item q of sequence s is its row end - (W-1) + q, or item q + length of its initial
// window where the history is shorter than that.  One thread per (sequence, item, V channels), in blocks behind the strips'.
template <class T, int W, int V>
__device__ __forceinline__ void final_window(const ConvArgs& a, int64_t i)
{
    const int d = (int)(i % a.nvec) * V, q = (int)(i / a.nvec % (W - 1));
    const int s = (int)(i / a.nvec / (W - 1));
    const int64_t b = a.off[s], e = a.off[s + 1], at = e - (W - 1) + q, iq = at - b + (W - 1);
    float v[V];
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = 0.0f;
    if (at >= b) {
        if (at >= 0 && at < a.rows) load_row<T, V>(a.x, at * a.x_stride + d, v);
    } else if (a.initial && iq >= 0 && iq < W - 1) {
        load_row<T, V>(a.initial, ((int64_t)s * (W - 1) + iq) * a.channels + d, v);
    }
    store_row<T, V>(a.final_window, ((int64_t)s * (W - 1) + q) * a.channels + d, v);
}
// dinitial of empty histories: their window passes through
template <class T, int W, int V>
__device__ __forceinline__ void empty_dinitial(const ConvArgs& a, int64_t i)
{
    const int64_t s = i / a.nvec / (W - 1);
    if (a.off[s + 1] > a.off[s]) return;
    const int64_t at = i / a.nvec * a.channels + i % a.nvec * V;
    float v[V];
#pragma unroll
    for (int k = 0; k < V; k++) v[k] = 0.0f;
    if (a.dfinal) load_row<T, V>(a.dfinal, at, v);
    store_row<T, V>(a.dinitial, at, v);
}
// what the blocks behind the strips' do: f(i) for every place i of the windows, one per thread up to 2^28 of them, several where there
// are more, for these alone must not make a launch too large
int64_t window_blocks(const rec_conv_desc* d, int64_t nvec)
{
    const int64_t n = (int64_t)d->n_seq * (d->taps - 1) * nvec;
    return n < (1ll << 28) ? (n + 255) / 256 : 1ll << 20;
}
template <int W, class F> __device__ __forceinline__ void every_window_place(const ConvArgs& a, F&& f)
{
    const int64_t n = (int64_t)a.n_seq * (W - 1) * a.nvec, step = (int64_t)(gridDim.x - a.main_blocks) * 256;
    for (int64_t i = (int64_t)(blockIdx.x - a.main_blocks) * 256 + threadIdx.x; i < n; i += step) f(i);
}

constexpr int kForwardGroup = 4, kBackwardGroup = 2;
// GROUP rows of a strip, loaded together and a group ahead of the walk; a row behind the array's end takes the last one
template <int GROUP, class T, int V>
__device__ __forceinline__ void fetch_rows(const void* base, int64_t stride, int64_t r, int64_t rows, int d, Pack<T, V> (&raw)[GROUP])
{
#pragma unroll
    for (int k = 0; k < GROUP; k++) {
        const int64_t at = r + k < rows ? r + k : rows - 1;
        raw[k] = *reinterpret_cast<const Pack<T, V>*>((const T*)base + at * stride + d);
    }
}
template <class T, int V> __device__ __forceinline__ void unpack(const Pack<T, V>& p, float (&x)[V])
{
#pragma unroll
    for (int v = 0; v < V; v++) x[v] = to_f32(p.v[v]);
}

// The strip and the channels of a thread: `ct` threads share a strip, 256 / ct strips a block.  ONE: a wavefront has one strip, which
// then is a scalar, and with it all that is known of the histories in it.
template <int V, bool ONE> struct Place {
    int64_t strip;
    int cv, d;
    bool on;
    __device__ __forceinline__ Place(const ConvArgs& a)
    {
        const int ct = ONE ? 64 : a.ct, part = threadIdx.x / ct;
        strip = (int64_t)(blockIdx.x / a.tiles) * (256 / ct) + (ONE ? __builtin_amdgcn_readfirstlane(part) : part);
        cv = blockIdx.x % a.tiles * ct + threadIdx.x % ct;
        on = cv < a.nvec;
        d = on ? cv * V : 0;
    }
};

template <class T, int W, int V, bool ONE>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {
        every_window_place<W>(a, [&](int64_t i) { final_window<T, W, V>(a, i); });
        return;
    }
    constexpr int GROUP = kForwardGroup;
    const Place<V, ONE> p(a);
    if (p.strip >= a.strips || !p.on) return;
    const int d = p.d;
    const int64_t strip = p.strip, r0 = strip * a.strip_rows, r1 = r0 + a.strip_rows < a.rows ? r0 + a.strip_rows : a.rows;
    Pack<T, V> ahead[GROUP];
    fetch_rows<GROUP, T, V>(a.x, a.x_stride, r0, a.rows, d, ahead);
    float w[W][V], b[V], win[W - 1][V];
    load_filter<W, V>(a, d, w, b);
    SeqCursor c;
    c.begin(a.off, a.n_seq, r0);
    load_window<T, W, V>(a, c.s, c.inside(a.n_seq) ? a.off[c.s] : r0, r0, d, win);
    auto step = [&](const float (&x)[V], float (&y)[V]) {
#pragma unroll
        for (int v = 0; v < V; v++) {
            float s = b[v];
#pragma unroll
            for (int j = 0; j < W - 1; j++) s = fmaf(w[j][v], win[j][v], s);
            s = fmaf(w[W - 1][v], x[v], s);
            y[v] = a.silu ? silu_f32(s) : s;
#pragma unroll
            for (int j = 0; j + 1 < W - 1; j++) win[j][v] = win[j + 1][v];
            win[W - 2][v] = x[v];
        }
    };
    for (int64_t r = r0; r < r1; r += GROUP) {
        float x[GROUP][V], y[V];
#pragma unroll
        for (int k = 0; k < GROUP; k++) unpack<T, V>(ahead[k], x[k]);
        if (r + GROUP < r1) fetch_rows<GROUP, T, V>(a.x, a.x_stride, r + GROUP, a.rows, d, ahead);
        if (r + GROUP <= r1 && r + GROUP <= c.next && c.inside(a.n_seq)) {   // all of one history
#pragma unroll
            for (int k = 0; k < GROUP; k++) {
                step(x[k], y);
                store_row<T, V>(a.y, (r + k) * a.y_stride + d, y);
            }
            continue;
        }
#pragma unroll
        for (int k = 0; k < GROUP; k++) {
            const int64_t row = r + k;
            if (row >= r1) continue;
            if (row >= c.next) {
                c.advance(a.off, a.n_seq, row);
                load_window<T, W, V>(a, c.s, row, row, d, win);
            }
            step(x[k], y);
            if (c.inside(a.n_seq)) {
                store_row<T, V>(a.y, row * a.y_stride + d, y);
            } else if (a.zero_rest) {
#pragma unroll
                for (int v = 0; v < V; v++) y[v] = 0.0f;
                store_row<T, V>(a.y, row * a.y_stride + d, y);
            }
        }
    }
}

// The gradient walks the same strips.  acc[i] collects dx of the W rows up to the current one; the oldest is complete W-1 rows
// later, so a strip reads W-1 rows past its end.  The window in front of a history's first row is W-1 rows like any other
// to the walk: what arrives there is dinitial, and dfinal enters at the last W-1 rows, of the window too if the history is shorter.
template <class T, int W, int V, bool ONE>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {
        every_window_place<W>(a, [&](int64_t i) { empty_dinitial<T, W, V>(a, i); });
        return;
    }
    constexpr int GROUP = kBackwardGroup;
    const Place<V, ONE> p(a);
    const int ct = ONE ? 64 : a.ct, lane_c = threadIdx.x % ct, d = p.d;
    const bool on = p.on;
    const int per = 256 / ct;   // strips a block walks at a time
    const int blocks_r = a.main_blocks / a.tiles;
    float w[W][V], b[V], dw[W][V], db[V];
    load_filter<W, V>(a, d, w, b);
#pragma unroll
    for (int v = 0; v < V; v++) {
        db[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) dw[j][v] = 0.0f;
    }
    for (int64_t strip = p.strip; on && strip < a.strips; strip += (int64_t)blocks_r * per) {
        const int64_t r0 = strip * a.strip_rows, r1 = r0 + a.strip_rows < a.rows ? r0 + a.strip_rows : a.rows, r2 = r1 + (W - 1);
        Pack<T, V> ahead_x[GROUP], ahead_g[GROUP];
        fetch_rows<GROUP, T, V>(a.x, a.x_stride, r0, a.rows, d, ahead_x);
        fetch_rows<GROUP, T, V>(a.dy, a.dy_stride, r0, a.rows, d, ahead_g);
        SeqCursor c;
        c.begin(a.off, a.n_seq, r0);
        int64_t start = c.inside(a.n_seq) ? a.off[c.s] : r0;
        float win[W - 1][V], acc[W][V];
        load_window<T, W, V>(a, c.s, start, r0, d, win);
#pragma unroll
        for (int i = 0; i < W; i++)
#pragma unroll
            for (int v = 0; v < V; v++) acc[i][v] = 0.0f;
        // a finished row of the walk: one of this strip's, or one of the window of a history that begins in this strip
        auto emit = [&](int64_t e, const float (&g)[V]) {
            if (e >= start) {
                if (e >= r0 && e < r1) store_row<T, V>(a.dx, e * a.dx_stride + d, g);
            } else if (a.dinitial && start >= r0 && c.inside(a.n_seq)) {
                const int64_t q = e - start + (W - 1);
                if (q >= 0) store_row<T, V>(a.dinitial, ((int64_t)c.s * (W - 1) + q) * a.channels + d, g);
            }
        };
        // one row; `done` receives the row W-1 in front of it
        auto step = [&](const float (&x)[V], const float (&g)[V], bool own, float (&done)[V]) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float s = b[v];
#pragma unroll
                for (int j = 0; j < W - 1; j++) s = fmaf(w[j][v], win[j][v], s);
                s = fmaf(w[W - 1][v], x[v], s);
                const float dv = a.silu ? g[v] * dsilu_f32(s) : g[v], mine = own ? dv : 0.0f;
#pragma unroll
                for (int i = 0; i < W; i++) acc[i][v] = fmaf(w[i][v], dv, acc[i][v]);
#pragma unroll
                for (int j = 0; j < W - 1; j++) dw[j][v] = own ? fmaf(dv, win[j][v], dw[j][v]) : dw[j][v];
                dw[W - 1][v] = own ? fmaf(dv, x[v], dw[W - 1][v]) : dw[W - 1][v];
                db[v] += mine;
#pragma unroll
                for (int j = 0; j + 1 < W - 1; j++) win[j][v] = win[j + 1][v];
                win[W - 2][v] = x[v];
                done[v] = acc[0][v];
#pragma unroll
                for (int i = 0; i + 1 < W; i++) acc[i][v] = acc[i + 1][v];
                acc[W - 1][v] = 0.0f;
            }
        };
        bool over = false;
        for (int64_t r = r0; r < r2 && !over; r += GROUP) {
            float x[GROUP][V], g[GROUP][V], done[V];
#pragma unroll
            for (int k = 0; k < GROUP; k++) {
                unpack<T, V>(ahead_x[k], x[k]);
                unpack<T, V>(ahead_g[k], g[k]);
            }
            if (r + GROUP < r2) {
                fetch_rows<GROUP, T, V>(a.x, a.x_stride, r + GROUP, a.rows, d, ahead_x);
                fetch_rows<GROUP, T, V>(a.dy, a.dy_stride, r + GROUP, a.rows, d, ahead_g);
            }
            const int64_t first = (start > r0 ? start : r0) + (W - 1);
            if (r >= first && r + GROUP <= r1 && r + GROUP <= c.next && c.inside(a.n_seq)) {   // all of one history, and so are the rows finished
#pragma unroll
                for (int k = 0; k < GROUP; k++) {
                    step(x[k], g[k], true, done);
                    store_row<T, V>(a.dx, (r + k - (W - 1)) * a.dx_stride + d, done);
                }
                continue;
            }
#pragma unroll
            for (int k = 0; k < GROUP; k++) {
                const int64_t row = r + k;
                if (over || row >= r2) continue;
                if (row >= c.next || row >= a.rows) {
                    if (c.inside(a.n_seq)) {   // the history ended with the row in front
#pragma unroll
                        for (int i = 0; i < W - 1; i++) {
                            float f[V];
#pragma unroll
                            for (int v = 0; v < V; v++) f[v] = 0.0f;
                            if (a.dfinal) load_row<T, V>(a.dfinal, ((int64_t)c.s * (W - 1) + i) * a.channels + d, f);
#pragma unroll
                            for (int v = 0; v < V; v++) f[v] += acc[i][v];
                            emit(row - (W - 1) + i, f);
                        }
                    }
                    if (row >= r1) { over = true; continue; }
                    c.advance(a.off, a.n_seq, row);
                    start = row;
                    load_window<T, W, V>(a, c.s, start, row, d, win);
#pragma unroll
                    for (int i = 0; i < W; i++)
#pragma unroll
                        for (int v = 0; v < V; v++) acc[i][v] = 0.0f;
                }
                if (!c.inside(a.n_seq)) {
                    if (row >= r1) { over = true; continue; }
                    if (a.zero_rest) store_row<T, V>(a.dx, row * a.dx_stride + d, acc[0]);   // zeros
                    continue;
                }
                step(x[k], g[k], row < r1, done);
                emit(row - (W - 1), done);
            }
        }
    }
    if (!a.partial) return;
    // the block's sums, over its strips in a fixed order
    __shared__ float red[256][V + 1];
    float* part = a.partial + (int64_t)(blockIdx.x / a.tiles) * a.channels * (W + 1);
#pragma unroll
    for (int j = 0; j <= W; j++) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; v++) red[threadIdx.x][v] = j < W ? dw[j < W ? j : 0][v] : db[v];
        __syncthreads();
        if ((int)threadIdx.x < ct && on) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float s = 0.0f;
                for (int k = 0; k < per; k++) s += red[k * ct + lane_c][v];
                part[j < W ? (int64_t)(d + v) * W + j : (int64_t)a.channels * W + d + v] = s;
            }
        }
    }
}

// A block takes one row and up to 256 V of its channels.  The first row that names a slot takes the later ones along.
template <class T, int W, int V>
__global__ __launch_bounds__(256) void conv_step_kernel(ConvArgs a, const int32_t* __restrict__ slots, T* window)
{
    const int64_t row = blockIdx.x / a.tiles;
    const int cv = (int)(blockIdx.x % a.tiles) * (int)blockDim.x + threadIdx.x;
    const bool on = cv < a.nvec;
    const int d = on ? cv * V : 0, slot = slots[row];
    __shared__ unsigned seen[4];
    look_for_slot(slots, a.rows, row, slot, seen);
    __syncthreads();
    const unsigned shared = slots_seen(seen);
    const bool earlier = shared & 1, later = shared & 2;
    float y[V];
    if (slot < 0 || slot >= a.n_seq) {
#pragma unroll
        for (int v = 0; v < V; v++) y[v] = 0.0f;
        if (on) store_row<T, V>(a.y, row * a.y_stride + d, y);
        return;
    }
    if (earlier) return;
    float w[W][V], b[V];
    load_filter<W, V>(a, d, w, b);
    const int64_t at = (int64_t)slot * (W - 1) * a.channels + d;
    auto click = [&](int64_t r) {   // the window goes through memory, so that rows of a shared slot are steps like any other
        float win[W][V];
        if (!on) return;
#pragma unroll
        for (int j = 0; j < W - 1; j++) load_row<T, V>(window, at + (int64_t)j * a.channels, win[j]);
        load_row<T, V>(a.x, r * a.x_stride + d, win[W - 1]);
#pragma unroll
        for (int v = 0; v < V; v++) {
            float s = b[v];
#pragma unroll
            for (int j = 0; j < W; j++) s = fmaf(w[j][v], win[j][v], s);
            y[v] = a.silu ? silu_f32(s) : s;
        }
        store_row<T, V>(a.y, r * a.y_stride + d, y);
#pragma unroll
        for (int j = 0; j < W - 1; j++) store_row<T, V>(window, at + (int64_t)j * a.channels, win[j + 1]);
    };
    click(row);
    if (later)
        for (int r = next_row_of(slots, (int)a.rows, (int)row, slot); r < (int)a.rows; r = next_row_of(slots, (int)a.rows, r, slot)) click(r);
}

// Rows of a strip: long strips read fewer rows twice (gradient above: 163, 142, 134 us at 32, 64, 128 rows), short ones give a small
// call more threads (2048 x 128 f32 forward: 15 us at 32 rows, 5 at 4).  262 144 threads, half of what the chip holds, are enough
// (100 000 x 128 bf16, forward and gradient: 25 and 56 us with strips for 65 536 threads, 19 and 40 for 131 072, 16 and 36 for 262 144,
// 19 and 43 for 524 288).
int strip_rows_of(int64_t rows, int64_t nvec, int longest)
{
    const int64_t s = rows * nvec / 262144 / 4 * 4;
    return (int)(s < 4 ? 4 : s > longest ? longest : s);
}
constexpr int kForwardVec = 2, kBackwardVec = 2;
constexpr int kForwardStrip = 128, kBackwardStrip = 128;
constexpr int kBackwardBlocks = 2048;   // at most, per tile of channels: bounds the partial sums

int check_desc(const rec_conv_desc* d)
{
    REC_REFUSE(!d, "null argument");
    REC_REFUSE(d->type < REC_TYPE_F32 || d->type > REC_TYPE_BF16, "unknown type");
    REC_REFUSE(d->rows < 0 || d->rows > INT32_MAX, "rows must be in 0..2^31-1");
    REC_REFUSE(d->n_seq < 0 || d->n_seq == INT32_MAX, "n_seq must be in 0..2^31-2");
    REC_REFUSE(d->channels < 1 || d->channels > 1 << 20, "channels must be in 1..2^20");
    REC_REFUSE(d->taps < 2 || d->taps > 8, "taps must be in 2..8");
    return 0;
}

int check_stride(int64_t stride, const rec_conv_desc* d)
{
    REC_REFUSE(stride < d->channels || stride > INT32_MAX, "a row stride is smaller than the channels, or beyond 2^31-1");
    return 0;
}

RowsOf rows_of(const rec_conv_desc* d, const void* p, int64_t stride)
{
    const int size = rec_type_size(d->type);
    return {p, d->rows, stride * size, (int64_t)d->channels * size};
}

int64_t window_bytes(const rec_conv_desc* d) { return (int64_t)d->n_seq * (d->taps - 1) * d->channels * rec_type_size(d->type); }

struct Layout { int vec, nvec; };

// V channels per thread where every row of every array starts on a V-element boundary
Layout layout_of(const rec_conv_desc* d, int widest, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides)
{
    const int size = rec_type_size(d->type);
    bool wide = d->channels % widest == 0;
    for (const void* p : ptrs) wide = wide && rec_aligned(p, (size_t)widest * size);
    for (int64_t s : strides) wide = wide && s % widest == 0;
    // 33 to 64 channels are one wavefront's at V = 1 and half of one's at V = 2 (gradient over 598 655 x 64 bf16: 90 us against 118)
    const int v = wide && (widest > 2 || d->channels > 64 || d->channels <= 32) ? widest : 1;
    return {v, d->channels / v};
}

struct Grid { int ct, tiles, per, blocks_r, strip_rows; int64_t strips; };
Grid grid_of(const rec_conv_desc* d, int nvec, int longest, int64_t most_blocks)
{
    Grid g;
    g.ct = 64;
    while (g.ct > 1 && g.ct / 2 >= nvec) g.ct /= 2;
    g.tiles = (nvec + g.ct - 1) / g.ct;
    g.per = 256 / g.ct;
    g.strip_rows = strip_rows_of(d->rows, nvec, longest);
    g.strips = (d->rows + g.strip_rows - 1) / g.strip_rows;
    const int64_t all = (g.strips + g.per - 1) / g.per, rounds = (all + most_blocks - 1) / most_blocks;
    g.blocks_r = rounds ? (int)((all + rounds - 1) / rounds) : 0;   // each block as many strips as any other
    return g;
}

#define CONV_TAPS(T, V, ONE, CALL)                                                                                    \
    switch (d->taps) {                                                                                                \
    case 2: CALL(T, 2, V, ONE); break; case 3: CALL(T, 3, V, ONE); break; case 4: CALL(T, 4, V, ONE); break;          \
    case 5: CALL(T, 5, V, ONE); break; case 6: CALL(T, 6, V, ONE); break; case 7: CALL(T, 7, V, ONE); break;          \
    default: CALL(T, 8, V, ONE); break;                                                                               \
    }
#define CONV_TYPE(T, WIDE, vec, one, CALL)                                                                            \
    {                                                                                                                 \
        if (vec == 1) { if (one) { CONV_TAPS(T, 1, true, CALL) } else { CONV_TAPS(T, 1, false, CALL) } }              \
        else if (one) { CONV_TAPS(T, WIDE, true, CALL) }                                                              \
        else { CONV_TAPS(T, WIDE, false, CALL) }                                                                      \
    }
#define CONV_DISPATCH(WIDE32, WIDE16, vec, one, CALL)                                                                 \
    if (d->type == REC_TYPE_F32) CONV_TYPE(float, WIDE32, vec, one, CALL)                                             \
    else if (d->type == REC_TYPE_F16) CONV_TYPE(_Float16, WIDE16, vec, one, CALL)                                     \
    else CONV_TYPE(__bf16, WIDE16, vec, one, CALL)

int check_blocks(int64_t blocks)
{
    REC_REFUSE(blocks > (1ll << 24) - 1, "too many rows, channels or sequences for one call");   // a launch holds fewer than 2^32 threads
    return 0;
}

}  // namespace

extern "C" int rec_history_conv(const rec_conv_desc* d, const void* x, int64_t x_stride, const float* weight, const float* bias,
                                const int64_t* seq_off, const void* initial, void* y, int64_t y_stride, void* final_window, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        REC_REFUSE(!weight || !seq_off || (d->rows > 0 && (!x || !y)), "null argument");
        if (int rc = check_stride(x_stride, d)) return rc;
        if (int rc = check_stride(y_stride, d)) return rc;
        const int wide = kForwardVec;
        REC_REFUSE(rec_overlap(rows_of(d, x, x_stride), rows_of(d, y, y_stride)), "the output overlaps the input");
        REC_REFUSE(rec_overlap(initial, window_bytes(d), final_window, window_bytes(d)), "final_window overlaps initial");
        if (int rc = rec_check_device(d->device)) return rc;
        const Layout l = layout_of(d, wide, {x, y, initial, final_window}, {x_stride, y_stride});
        const Grid g = grid_of(d, l.nvec, kForwardStrip, INT32_MAX);
        ConvArgs a = {};
        a.x = x; a.initial = initial; a.y = y; a.final_window = final_window; a.weight = weight; a.bias = bias; a.off = seq_off;
        a.x_stride = x_stride; a.y_stride = y_stride; a.rows = d->rows; a.n_seq = d->n_seq; a.channels = d->channels; a.nvec = l.nvec;
        a.silu = d->silu; a.zero_rest = d->zero_rest; a.strip_rows = g.strip_rows; a.strips = g.strips;
        a.ct = g.ct; a.tiles = g.tiles;
        const int64_t main_blocks = (int64_t)g.blocks_r * g.tiles;
        const int64_t more = final_window ? window_blocks(d, l.nvec) : 0;
        if (int rc = check_blocks(main_blocks + more)) return rc;
        if (main_blocks + more == 0) return 0;
        a.main_blocks = (int)main_blocks;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
#define CALL(T, W, V, ONE) conv_forward_kernel<T, W, V, ONE><<<(unsigned)(main_blocks + more), 256, 0, (hipStream_t)stream>>>(a)
        CONV_DISPATCH(kForwardVec, kForwardVec, l.vec, g.ct == 64, CALL)
#undef CALL
        HIP_TRY(hipGetLastError());
        return 0;
    });
}

extern "C" int64_t rec_history_conv_backward_workspace(const rec_conv_desc* d)
{
    return rec_guarded([&]() -> int64_t {
        if (check_desc(d)) return -1;
        // as much as the layout that takes the most blocks needs, whatever the alignment of the arrays turns out to be
        const int narrow = grid_of(d, d->channels, kBackwardStrip, kBackwardBlocks).blocks_r;
        const int wide = d->channels % kBackwardVec == 0 ? grid_of(d, d->channels / kBackwardVec, kBackwardStrip, kBackwardBlocks).blocks_r : 0;
        return (int64_t)(narrow > wide ? narrow : wide) * d->channels * (d->taps + 1) * 4;
    });
}

extern "C" int rec_history_conv_backward(const rec_conv_desc* d, const void* dy, int64_t dy_stride, const void* x, int64_t x_stride,
                                         const float* weight, const float* bias, const int64_t* seq_off, const void* initial,
                                         const void* dfinal, void* dx, int64_t dx_stride, float* dweight, float* dbias, void* dinitial,
                                         void* workspace, int64_t workspace_bytes, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        REC_REFUSE(!weight || !seq_off || (d->rows > 0 && (!x || !dy || !dx)), "null argument");
        if (int rc = check_stride(x_stride, d)) return rc;
        if (int rc = check_stride(dy_stride, d)) return rc;
        if (int rc = check_stride(dx_stride, d)) return rc;
        REC_REFUSE(rec_overlap(rows_of(d, x, x_stride), rows_of(d, dx, dx_stride)) || rec_overlap(rows_of(d, dy, dy_stride), rows_of(d, dx, dx_stride)),
                   "the output overlaps the input");
        REC_REFUSE(rec_overlap(initial, window_bytes(d), dinitial, window_bytes(d)) || rec_overlap(dfinal, window_bytes(d), dinitial, window_bytes(d)),
                   "dinitial overlaps initial or dfinal");
        const bool sums = dweight || dbias;
        REC_REFUSE(sums && workspace_bytes < rec_history_conv_backward_workspace(d), "the workspace is too small");
        REC_REFUSE(sums && rec_history_conv_backward_workspace(d) > 0 && (!workspace || !rec_aligned(workspace, 16)), "the workspace is null or not aligned to 16 bytes");
        if (int rc = rec_check_device(d->device)) return rc;
        const Layout l = layout_of(d, kBackwardVec, {x, dy, dx, initial, dfinal, dinitial}, {x_stride, dy_stride, dx_stride});
        const Grid g = grid_of(d, l.nvec, kBackwardStrip, kBackwardBlocks);
        ConvArgs a = {};
        a.x = x; a.initial = initial; a.dy = dy; a.dfinal = dfinal; a.dx = dx; a.dinitial = dinitial; a.weight = weight; a.bias = bias;
        a.off = seq_off; a.x_stride = x_stride; a.dy_stride = dy_stride; a.dx_stride = dx_stride; a.rows = d->rows; a.n_seq = d->n_seq;
        a.channels = d->channels; a.nvec = l.nvec; a.silu = d->silu; a.zero_rest = d->zero_rest; a.strip_rows = g.strip_rows;
        a.strips = g.strips; a.ct = g.ct; a.tiles = g.tiles;
        a.partial = sums ? (float*)workspace : nullptr;
        const int64_t main_blocks = (int64_t)g.blocks_r * g.tiles;
        const int64_t more = dinitial ? window_blocks(d, l.nvec) : 0;
        if (int rc = check_blocks(main_blocks + more)) return rc;
        a.main_blocks = (int)main_blocks;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        if (main_blocks + more > 0) {
#define CALL(T, W, V, ONE) conv_backward_kernel<T, W, V, ONE><<<(unsigned)(main_blocks + more), 256, 0, (hipStream_t)stream>>>(a)
            CONV_DISPATCH(kBackwardVec, kBackwardVec, l.vec, g.ct == 64, CALL)
#undef CALL
            HIP_TRY(hipGetLastError());
        }
        if (!sums) return 0;
        return launch_sum_partials(a.partial, g.blocks_r, (int64_t)d->channels * (d->taps + 1), dweight, (int64_t)d->channels * d->taps, dbias,
                                   d->channels, nullptr, (hipStream_t)stream);
    });
}

extern "C" int rec_history_conv_step(const rec_conv_desc* d, const void* x, int64_t x_stride, const float* weight, const float* bias,
                                     const int32_t* slots, void* window, void* y, int64_t y_stride, void* stream)
{
    return rec_guarded([&]() -> int {
        if (int rc = check_desc(d)) return rc;
        REC_REFUSE(d->rows > 65536, "a step takes at most 65536 rows");
        REC_REFUSE(!weight || (d->rows > 0 && (!x || !y || !slots)) || (d->n_seq > 0 && !window), "null argument");
        if (int rc = check_stride(x_stride, d)) return rc;
        if (int rc = check_stride(y_stride, d)) return rc;
        const int size = rec_type_size(d->type), wide = 16 / size;
        const RowsOf xr = rows_of(d, x, x_stride), yr = rows_of(d, y, y_stride);
        const RowsOf pool = {window, 1, INT64_MAX, window_bytes(d)};
        REC_REFUSE(rec_overlap(xr, yr) || rec_overlap(pool, yr) || rec_overlap(pool, xr), "x, y and the window must not overlap");
        if (int rc = rec_check_device(d->device)) return rc;
        if (d->rows == 0) return 0;
        const Layout l = layout_of(d, wide, {x, y, window}, {x_stride, y_stride});
        ConvArgs a = {};
        a.x = x; a.y = y; a.weight = weight; a.bias = bias; a.x_stride = x_stride; a.y_stride = y_stride; a.rows = d->rows;
        a.n_seq = d->n_seq; a.channels = d->channels; a.nvec = l.nvec; a.silu = d->silu;
        const int threads = l.nvec >= 256 ? 256 : (l.nvec + 63) / 64 * 64;
        a.tiles = (l.nvec + threads - 1) / threads;
        if (int rc = check_blocks((d->rows < kStepRows ? d->rows : kStepRows) * a.tiles)) return rc;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        for (int64_t r = 0; r < d->rows; r += kStepRows) {
            a.rows = d->rows - r < kStepRows ? d->rows - r : kStepRows;
            a.x = (const char*)x + r * x_stride * size;
            a.y = (char*)y + r * y_stride * size;
#define CALL(T, W, V, ONE) conv_step_kernel<T, W, V><<<(unsigned)(a.rows * a.tiles), threads, 0, (hipStream_t)stream>>>(a, slots + r, (T*)window)
            CONV_DISPATCH(4, 8, l.vec, false, CALL)
#undef CALL
        }
        HIP_TRY(hipGetLastError());
        return 0;
    });
}
