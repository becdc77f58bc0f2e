// Short causal convolution over packed histories: y, its gradient, and the form for single clicks.
//
//   v[t][d] = bias[d] + sum_{j < W} weight[d][j] x[t - (W-1) + j][d],   y = silu(v) or v
//
// 2 W flop per element read and written: bound by memory.  A thread owns V neighbouring channels (one 16-byte access per row
// where alignment allows) and walks a strip of consecutive rows with the window in registers, so a row is read once plus W-1
// rows of halo per strip (these come from the cache).  Where a history begins inside the strip, the window is replaced by that history's own.
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
__device__ __forceinline__ void final_windows(const ConvArgs& a, int64_t i)
{
    const int64_t n = (int64_t)a.n_seq * (W - 1) * a.nvec;
    if (i >= n) return;
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

template <class T, int W, int V>
__global__ __launch_bounds__(256) void conv_forward_kernel(ConvArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {
        final_windows<T, W, V>(a, (int64_t)(blockIdx.x - a.main_blocks) * 256 + threadIdx.x);
        return;
    }
    const int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x;
    const int64_t strip = i / a.nvec;
    if (strip >= a.strips) return;
    const int d = (int)(i - strip * a.nvec) * V;
    const int64_t r0 = strip * a.strip_rows, r1 = r0 + a.strip_rows < a.rows ? r0 + a.strip_rows : a.rows;
    float w[W][V], b[V], win[W - 1][V];
    load_filter<W, V>(a, d, w, b);
    SeqCursor c;
    c.begin(a.off, a.n_seq, r0);
    load_window<T, W, V>(a, c.s, c.inside(a.n_seq) ? a.off[c.s] : r0, r0, d, win);
    for (int64_t r = r0; r < r1; r++) {
        float x[V], y[V];
        load_row<T, V>(a.x, r * a.x_stride + d, x);
        if (r >= c.next) {
            c.advance(a.off, a.n_seq, r);
            load_window<T, W, V>(a, c.s, r, r, d, win);
        }
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
        if (c.inside(a.n_seq)) {
            store_row<T, V>(a.y, r * a.y_stride + d, y);
        } else if (a.zero_rest) {
#pragma unroll
            for (int v = 0; v < V; v++) y[v] = 0.0f;
            store_row<T, V>(a.y, r * a.y_stride + d, y);
        }
    }
}

// The gradient walks the same strips.  acc[i] collects dx of the W rows up to the current one; the oldest is complete W-1 rows
// later, so a strip reads W-1 rows past its end.  The window in front of a history's first row is W-1 rows like any other
// to the walk: what arrives there is dinitial, and dfinal enters at the last W-1 rows, of the window too if the history is shorter.
template <class T, int W, int V>
__global__ __launch_bounds__(256) void conv_backward_kernel(ConvArgs a)
{
    if ((int)blockIdx.x >= a.main_blocks) {   // dinitial of empty histories: their window passes through
        const int64_t i = (int64_t)(blockIdx.x - a.main_blocks) * 256 + threadIdx.x;
        if (i >= (int64_t)a.n_seq * (W - 1) * a.nvec) return;
        const int64_t s = i / a.nvec / (W - 1);
        if (a.off[s + 1] > a.off[s]) return;
        const int64_t at = i / a.nvec * a.channels + i % a.nvec * V;
        float v[V];
#pragma unroll
        for (int k = 0; k < V; k++) v[k] = 0.0f;
        if (a.dfinal) load_row<T, V>(a.dfinal, at, v);
        store_row<T, V>(a.dinitial, at, v);
        return;
    }
    const int tile = blockIdx.x % a.tiles, lane_c = threadIdx.x % a.ct;
    const int cv = tile * a.ct + lane_c;
    const bool on = cv < a.nvec;
    const int d = on ? cv * V : 0;
    const int per = 256 / a.ct;   // strips a block walks at a time
    const int blocks_r = a.main_blocks / a.tiles;
    float w[W][V], b[V], dw[W][V], db[V];
    load_filter<W, V>(a, d, w, b);
#pragma unroll
    for (int v = 0; v < V; v++) {
        db[v] = 0.0f;
#pragma unroll
        for (int j = 0; j < W; j++) dw[j][v] = 0.0f;
    }
    for (int64_t strip = (int64_t)(blockIdx.x / a.tiles) * per + threadIdx.x / a.ct; on && strip < a.strips; strip += (int64_t)blocks_r * per) {
        const int64_t r0 = strip * a.strip_rows, r1 = r0 + a.strip_rows < a.rows ? r0 + a.strip_rows : a.rows;
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
        for (int64_t r = r0; r < r1 + (W - 1); r++) {
            if (r >= c.next || r >= a.rows) {
                if (c.inside(a.n_seq)) {   // the history ended with row r - 1
#pragma unroll
                    for (int i = 0; i < W - 1; i++) {
                        float g[V], f[V];
#pragma unroll
                        for (int v = 0; v < V; v++) f[v] = 0.0f;
                        if (a.dfinal) load_row<T, V>(a.dfinal, ((int64_t)c.s * (W - 1) + i) * a.channels + d, f);
#pragma unroll
                        for (int v = 0; v < V; v++) g[v] = acc[i][v] + f[v];
                        emit(r - (W - 1) + i, g);
                    }
                }
                if (r >= r1) break;
                c.advance(a.off, a.n_seq, r);
                start = r;
                load_window<T, W, V>(a, c.s, start, r, d, win);
#pragma unroll
                for (int i = 0; i < W; i++)
#pragma unroll
                    for (int v = 0; v < V; v++) acc[i][v] = 0.0f;
            }
            if (!c.inside(a.n_seq)) {
                if (r >= r1) break;
                if (a.zero_rest) store_row<T, V>(a.dx, r * a.dx_stride + d, acc[0]);   // zeros
                continue;
            }
            float x[V], g[V];
            load_row<T, V>(a.x, r * a.x_stride + d, x);
            load_row<T, V>(a.dy, r * a.dy_stride + d, g);
            const bool own = r < r1;
#pragma unroll
            for (int v = 0; v < V; v++) {
                float s = b[v];
#pragma unroll
                for (int j = 0; j < W - 1; j++) s = fmaf(w[j][v], win[j][v], s);
                s = fmaf(w[W - 1][v], x[v], s);
                const float dv = a.silu ? g[v] * dsilu_f32(s) : g[v];
#pragma unroll
                for (int i = 0; i < W; i++) acc[i][v] = fmaf(w[i][v], dv, acc[i][v]);
                if (own) {
#pragma unroll
                    for (int j = 0; j < W - 1; j++) dw[j][v] = fmaf(dv, win[j][v], dw[j][v]);
                    dw[W - 1][v] = fmaf(dv, x[v], dw[W - 1][v]);
                    db[v] += dv;
                }
#pragma unroll
                for (int j = 0; j + 1 < W - 1; j++) win[j][v] = win[j + 1][v];
                win[W - 2][v] = x[v];
            }
            emit(r - (W - 1), acc[0]);
#pragma unroll
            for (int v = 0; v < V; v++) {
#pragma unroll
                for (int i = 0; i + 1 < W; i++) acc[i][v] = acc[i + 1][v];
                acc[W - 1][v] = 0.0f;
            }
        }
    }
    if (!a.partial) return;
    // the block's sums, over its strips in a fixed order
    __shared__ float red[256][V + 1];
    float* part = a.partial + (int64_t)(blockIdx.x / a.tiles) * a.channels * (W + 1);
    for (int j = 0; j <= W; j++) {
        __syncthreads();
#pragma unroll
        for (int v = 0; v < V; v++) {
            float s = db[v];
#pragma unroll
            for (int k = 0; k < W; k++) s = j == k ? dw[k][v] : s;
            red[threadIdx.x][v] = s;
        }
        __syncthreads();
        if ((int)threadIdx.x < a.ct && on) {
#pragma unroll
            for (int v = 0; v < V; v++) {
                float s = 0.0f;
                for (int k = 0; k < per; k++) s += red[k * a.ct + lane_c][v];
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
    const int cv = (int)(blockIdx.x % a.tiles) * (int)blockDim.x + threadIdx.x, d = cv * V;
    const int slot = slots[row];
    bool earlier, later;
    slot_is_shared(slots, a.rows, row, slot, earlier, later);
    if (cv >= a.nvec) return;
    float y[V];
    if (slot < 0 || slot >= a.n_seq) {
#pragma unroll
        for (int v = 0; v < V; v++) y[v] = 0.0f;
        store_row<T, V>(a.y, row * a.y_stride + d, y);
        return;
    }
    if (earlier) return;
    float w[W][V], b[V];
    load_filter<W, V>(a, d, w, b);
    const int64_t at = (int64_t)slot * (W - 1) * a.channels + d;
    auto click = [&](int64_t r) {   // the window goes through memory, so that rows of a shared slot are steps like any other
        float win[W][V];
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
        for (int64_t r = row + 1; r < a.rows; r++)
            if (slots[r] == slot) click(r);
}

constexpr int kStripRows = 32;
constexpr int kBackwardBlocks = 2048;   // at most, per tile of channels: bounds the partial sums

int check_desc(const rec_conv_desc* d)
{
    REC_REFUSE(!d, "null argument");
    REC_REFUSE(d->type < REC_TYPE_F32 || d->type > REC_TYPE_BF16, "unknown type");
    REC_REFUSE(d->rows < 0 || d->rows > INT32_MAX, "rows must be in 0..2^31-1");
    REC_REFUSE(d->n_seq < 0, "n_seq must not be negative");
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

struct Layout { int vec, nvec; };

// V channels per thread where every row of every array starts on a V-element boundary
Layout layout_of(const rec_conv_desc* d, int widest, std::initializer_list<const void*> ptrs, std::initializer_list<int64_t> strides)
{
    const int size = rec_type_size(d->type);
    bool wide = d->channels % widest == 0;
    for (const void* p : ptrs) wide = wide && rec_aligned(p, (size_t)widest * size);
    for (int64_t s : strides) wide = wide && s % widest == 0;
    const int v = wide ? widest : 1;
    return {v, d->channels / v};
}

struct BackwardGrid { int ct, tiles, per, blocks_r; int64_t strips; };
BackwardGrid backward_grid(const rec_conv_desc* d, int nvec)
{
    BackwardGrid g;
    g.ct = 64;
    while (g.ct > 1 && g.ct / 2 >= nvec) g.ct /= 2;
    g.tiles = (nvec + g.ct - 1) / g.ct;
    g.per = 256 / g.ct;
    g.strips = (d->rows + kStripRows - 1) / kStripRows;
    const int64_t most = (g.strips + g.per - 1) / g.per;
    g.blocks_r = (int)(most < kBackwardBlocks ? most : kBackwardBlocks);
    return g;
}

#define CONV_TAPS(T, V, CALL)                                                                         \
    switch (d->taps) {                                                                                \
    case 2: CALL(T, 2, V); break; case 3: CALL(T, 3, V); break; case 4: CALL(T, 4, V); break;         \
    case 5: CALL(T, 5, V); break; case 6: CALL(T, 6, V); break; case 7: CALL(T, 7, V); break;         \
    default: CALL(T, 8, V); break;                                                                    \
    }
#define CONV_DISPATCH(WIDE32, WIDE16, vec, CALL)                                                      \
    if (d->type == REC_TYPE_F32) { if (vec > 1) { CONV_TAPS(float, WIDE32, CALL) } else { CONV_TAPS(float, 1, CALL) } }             \
    else if (d->type == REC_TYPE_F16) { if (vec > 1) { CONV_TAPS(_Float16, WIDE16, CALL) } else { CONV_TAPS(_Float16, 1, CALL) } }  \
    else { if (vec > 1) { CONV_TAPS(__bf16, WIDE16, CALL) } else { CONV_TAPS(__bf16, 1, CALL) } }

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
        const int size = rec_type_size(d->type), wide = 16 / size;
        REC_REFUSE(rec_overlap(rows_of(d, x, x_stride), rows_of(d, y, y_stride)), "the output overlaps the input");
        if (int rc = rec_check_device(d->device)) return rc;
        const Layout l = layout_of(d, wide, {x, y, initial, final_window}, {x_stride, y_stride});
        ConvArgs a = {};
        a.x = x; a.initial = initial; a.y = y; a.final_window = final_window; a.weight = weight; a.bias = bias; a.off = seq_off;
        a.x_stride = x_stride; a.y_stride = y_stride; a.rows = d->rows; a.n_seq = d->n_seq; a.channels = d->channels; a.nvec = l.nvec;
        a.silu = d->silu; a.zero_rest = d->zero_rest; a.strip_rows = kStripRows;
        a.strips = (d->rows + kStripRows - 1) / kStripRows;
        const int64_t main_blocks = (a.strips * l.nvec + 255) / 256;
        const int64_t more = final_window ? ((int64_t)d->n_seq * (d->taps - 1) * l.nvec + 255) / 256 : 0;
        if (int rc = check_blocks(main_blocks + more)) return rc;
        if (main_blocks + more == 0) return 0;
        a.main_blocks = (int)main_blocks;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
#define CALL(T, W, V) conv_forward_kernel<T, W, V><<<(unsigned)(main_blocks + more), 256, 0, (hipStream_t)stream>>>(a)
        CONV_DISPATCH(4, 8, l.vec, CALL)
#undef CALL
        HIP_TRY(hipGetLastError());
        return 0;
    });
}

extern "C" int64_t rec_history_conv_backward_workspace(const rec_conv_desc* d)
{
    if (check_desc(d)) return -1;
    // the narrow layout has at most as many blocks as the limit, whatever the alignment of the arrays turns out to be
    const int64_t strips = (d->rows + kStripRows - 1) / kStripRows;
    const int64_t blocks = strips < kBackwardBlocks ? strips : kBackwardBlocks;
    return blocks * d->channels * (d->taps + 1) * 4;
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
        const bool sums = dweight || dbias;
        REC_REFUSE(sums && workspace_bytes < rec_history_conv_backward_workspace(d), "the workspace is too small");
        REC_REFUSE(sums && rec_history_conv_backward_workspace(d) > 0 && (!workspace || !rec_aligned(workspace, 16)), "the workspace is null or not aligned to 16 bytes");
        if (int rc = rec_check_device(d->device)) return rc;
        const Layout l = layout_of(d, 4, {x, dy, dx, initial, dfinal, dinitial}, {x_stride, dy_stride, dx_stride});
        const BackwardGrid g = backward_grid(d, l.nvec);
        ConvArgs a = {};
        a.x = x; a.initial = initial; a.dy = dy; a.dfinal = dfinal; a.dx = dx; a.dinitial = dinitial; a.weight = weight; a.bias = bias;
        a.off = seq_off; a.x_stride = x_stride; a.dy_stride = dy_stride; a.dx_stride = dx_stride; a.rows = d->rows; a.n_seq = d->n_seq;
        a.channels = d->channels; a.nvec = l.nvec; a.silu = d->silu; a.zero_rest = d->zero_rest; a.strip_rows = kStripRows;
        a.strips = g.strips; a.ct = g.ct; a.tiles = g.tiles;
        a.partial = sums ? (float*)workspace : nullptr;
        const int64_t main_blocks = (int64_t)g.blocks_r * g.tiles;
        const int64_t more = dinitial ? ((int64_t)d->n_seq * (d->taps - 1) * l.nvec + 255) / 256 : 0;
        if (int rc = check_blocks(main_blocks + more)) return rc;
        a.main_blocks = (int)main_blocks;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
        if (main_blocks + more > 0) {
#define CALL(T, W, V) conv_backward_kernel<T, W, V><<<(unsigned)(main_blocks + more), 256, 0, (hipStream_t)stream>>>(a)
            CONV_DISPATCH(4, 4, l.vec, CALL)
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
        const RowsOf pool = {window, 1, INT64_MAX, (int64_t)d->n_seq * (d->taps - 1) * d->channels * size};
        REC_REFUSE(rec_overlap(xr, yr) || rec_overlap(pool, yr) || rec_overlap(pool, xr), "x, y and the window must not overlap");
        if (int rc = rec_check_device(d->device)) return rc;
        if (d->rows == 0) return 0;
        const Layout l = layout_of(d, wide, {x, y, window}, {x_stride, y_stride});
        ConvArgs a = {};
        a.x = x; a.y = y; a.weight = weight; a.bias = bias; a.x_stride = x_stride; a.y_stride = y_stride; a.rows = d->rows;
        a.n_seq = d->n_seq; a.channels = d->channels; a.nvec = l.nvec; a.silu = d->silu;
        const int threads = l.nvec >= 256 ? 256 : (l.nvec + 63) / 64 * 64;
        a.tiles = (l.nvec + threads - 1) / threads;
        const int64_t blocks = d->rows * a.tiles;
        if (int rc = check_blocks(blocks)) return rc;
        DeviceScope scope;
        HIP_TRY(scope.enter(d->device));
#define CALL(T, W, V) conv_step_kernel<T, W, V><<<(unsigned)blocks, threads, 0, (hipStream_t)stream>>>(a, slots, (T*)window)
        CONV_DISPATCH(4, 8, l.vec, CALL)
#undef CALL
        HIP_TRY(hipGetLastError());
        return 0;
    });
}
