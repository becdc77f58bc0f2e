// What the device operators (history_conv, history_scan, catalog_loss) share.
#pragma once
#include "common.h"
#include <limits.h>
#include <math.h>

// ---- host side: an entry point works on the caller's device and stream, and nothing is thrown across the C boundary
struct DeviceScope {
    int before = -1;
    bool moved = false;
    hipError_t enter(int device)
    {
        hipError_t rc = hipGetDevice(&before);
        if (rc == hipSuccess && before != device) { rc = hipSetDevice(device); moved = rc == hipSuccess; }
        return rc;
    }
    ~DeviceScope() { if (moved) (void)hipSetDevice(before); }
};

#define REC_REFUSE(cond, msg)                       \
    do {                                            \
        if (cond) { rec_set_error(msg); return -1; } \
    } while (0)

template <class F> auto rec_guarded(F&& f) -> decltype(f())
{
    try { return f(); } catch (...) { return -3; }   // only the message's own allocation can throw
}

inline int rec_check_device(int device)
{
    static const int n = [] { int c = 0; return hipGetDeviceCount(&c) == hipSuccess ? c : 0; }();
    REC_REFUSE(device < 0 || device >= n, "no such HIP device");
    return 0;
}

inline bool rec_overlap(const void* a, int64_t a_bytes, const void* b, int64_t b_bytes)
{
    const uintptr_t x = (uintptr_t)a, y = (uintptr_t)b;
    return a && b && a_bytes > 0 && b_bytes > 0 && x < y + (uintptr_t)b_bytes && y < x + (uintptr_t)a_bytes;
}

// Rows of an array, in bytes: `width` of them every `stride`.  Two such arrays share a byte if their extents do, unless they are
// different columns of one wider array.
struct RowsOf { const void* p; int64_t rows, stride, width; };
inline bool rec_overlap(const RowsOf& a, const RowsOf& b)
{
    if (a.rows < 1 || b.rows < 1 || !rec_overlap(a.p, (a.rows - 1) * a.stride + a.width, b.p, (b.rows - 1) * b.stride + b.width)) return false;
    if (a.stride != b.stride) return true;
    const int64_t off = (int64_t)((uintptr_t)b.p - (uintptr_t)a.p) % a.stride, ahead = off < 0 ? off + a.stride : off;
    return ahead < a.width || a.stride - ahead < b.width;
}

inline int rec_type_size(int type) { return type == REC_TYPE_F32 ? 4 : 2; }
inline bool rec_aligned(const void* p, size_t n) { return ((uintptr_t)p & (n - 1)) == 0; }

// sums over the rows of a partial matrix [n_rows][n_cols], in row order, in 64 bits: columns [0, n0) to out0, [n0, n0 + n1) to
// out1, the rest to out2 (each may be null)
int launch_sum_partials(const float* part, int64_t n_rows, int64_t n_cols, float* out0, int64_t n0, float* out1, int64_t n1, float* out2, hipStream_t st);
// the launch's size, in blocks of 256 threads
int64_t sum_partials_blocks(int64_t n_cols);

#ifdef __HIPCC__
// ---- device side
template <class T> __device__ __forceinline__ float to_f32(T v) { return (float)v; }
template <class T> __device__ __forceinline__ T from_f32(float v) { return (T)v; }   // rounds to nearest even, once, at the store

template <class T, int V> struct alignas(sizeof(T) * V) Pack { T v[V]; };

// The sequence a packed row lies in: the largest s with off[s] <= row; -1 in front of the first, n_seq behind the last.
// Only compares what it reads: offsets that are out of order lead to some s in [-1, n_seq], never out of the arrays.
__device__ __forceinline__ int sequence_of(const int64_t* __restrict__ off, int n_seq, int64_t row)
{
    int lo = 0, hi = n_seq + 1;   // first index whose offset is beyond the row (n_seq < 2^31 - 1; lo + hi may be more than an int)
    while (lo < hi) {
        const int mid = lo + ((hi - lo) >> 1);
        if (off[mid] <= row) lo = mid + 1; else hi = mid;
    }
    return lo - 1;
}

// Walks packed rows forwards: the current sequence, and the first row that is not in it any more.
struct SeqCursor {
    int s;
    int64_t next;
    __device__ __forceinline__ void begin(const int64_t* __restrict__ off, int n_seq, int64_t row)
    {
        s = sequence_of(off, n_seq, row);
        next = s < n_seq ? off[s + 1] : INT64_MAX;
    }
    __device__ __forceinline__ void advance(const int64_t* __restrict__ off, int n_seq, int64_t row)   // row >= next
    {
        s++;
        for (int k = 0; s < n_seq && off[s + 1] <= row; k++) {   // empty histories in between
            s++;
            if (k < 16) continue;
            int lo = s, hi = n_seq;   // many of them: the last index with off <= row
            while (lo < hi) {
                const int mid = lo + ((hi - lo + 1) >> 1);
                if (off[mid] <= row) lo = mid; else hi = mid - 1;
            }
            s = lo;
        }
        next = s < n_seq ? off[s + 1] : INT64_MAX;
    }
    __device__ __forceinline__ bool inside(int n_seq) const { return s >= 0 && s < n_seq; }
};

__device__ __forceinline__ float fast_exp2(float x) { return __builtin_amdgcn_exp2f(x); }   // v_exp_f32: 1 ulp, results below 2^-126 are 0
#define REC_LOG2E 1.44269504088896340736f
__device__ __forceinline__ float fast_exp(float x) { return fast_exp2(x * REC_LOG2E); }
__device__ __forceinline__ float sigmoid_f32(float v) { return __builtin_amdgcn_rcpf(1.0f + fast_exp(-v)); }   // v_rcp_f32: 1 ulp
__device__ __forceinline__ float silu_f32(float v) { return v * sigmoid_f32(v); }
__device__ __forceinline__ float dsilu_f32(float v)
{
    const float g = sigmoid_f32(v);
    return g * (1.0f + v * (1.0f - g));
}
// log(1 + e^v) = max(v, 0) + log(1 + e) with e = e^-|v| in (0, 1]; log(1 + e) / e by a polynomial fitted to it on [0, 1] in
// Chebyshev nodes (off by 5e-9; evaluated in f32, the product is within 2.4 ulp), so that small results keep their precision
__device__ __forceinline__ float softplus_f32(float v)
{
    const float e = fast_exp(-fabsf(v));
    float p = -0.003256378462538123f;
    p = fmaf(p, e, 0.019907161593437195f);
    p = fmaf(p, e, -0.057064201682806015f);
    p = fmaf(p, e, 0.10614264756441116f);
    p = fmaf(p, e, -0.15311862528324127f);
    p = fmaf(p, e, 0.19678117334842682f);
    p = fmaf(p, e, -0.24954558908939362f);
    p = fmaf(p, e, 0.33330005407333374f);
    p = fmaf(p, e, -0.4999990463256836f);
    p = fmaf(p, e, 1.0f);
    return fmaf(p, e, fmaxf(v, 0.0f));
}

// the largest of a wavefront's values, in every lane
__device__ __forceinline__ float wave_max(float v)
{
    v = fmaxf(v, dpp_move<0xB1>(v));
    v = fmaxf(v, dpp_move<0x4E>(v));
    v = fmaxf(v, dpp_move<0x141>(v));
    v = fmaxf(v, dpp_move<0x140>(v));
    v = fmaxf(v, __shfl_xor(v, 16, 64));
    return fmaxf(v, __shfl_xor(v, 32, 64));
}

// sums over lanes in pieces: lanes below 32 end up with a of both halves added, lanes from 32 on with b of both halves
__device__ __forceinline__ float fold32(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane32_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// the same between the 16 lanes rows of each half: rows 0 and 2 get a, rows 1 and 3 get b
__device__ __forceinline__ float fold16(float a, float b)
{
    const auto r = __builtin_amdgcn_permlane16_swap(__float_as_uint(a), __float_as_uint(b), false, false);
    return __uint_as_float(r[0]) + __uint_as_float(r[1]);
}
// sum over the lanes of a row of 16 that are equal modulo LN (2 .. 16), in every one of them
template <int LN> __device__ __forceinline__ float row_sum_strided(float v)
{
    if constexpr (LN <= 8) v += dpp_move<0x128>(v);   // row_ror:8
    if constexpr (LN <= 4) v += dpp_move<0x124>(v);
    if constexpr (LN <= 2) v += dpp_move<0x122>(v);
    return v;
}

// Rows of a step that name the same slot.  The block's threads look through the slots together: each wavefront leaves what it has
// seen in `seen` (bit 0: a row in front of `row` names `slot`, bit 1: one behind it does); behind the next barrier
// slots_seen() joins them.
__device__ __forceinline__ void look_for_slot(const int32_t* __restrict__ slots, int64_t rows, int64_t row, int slot, unsigned (&seen)[4])
{
    const int n = (int)rows, me = (int)row;   // a step has at most 65536 rows
    bool e = false, l = false;
#pragma unroll 4
    for (int i = threadIdx.x; i < n; i += blockDim.x) {
        const bool same = slots[i] == slot;
        e |= same && i < me;
        l |= same && i > me;
    }
    const unsigned bits = (__any(e) ? 1u : 0u) | (__any(l) ? 2u : 0u);
    if ((threadIdx.x & 63) == 0) seen[threadIdx.x >> 6] = bits;
}
__device__ __forceinline__ unsigned slots_seen(const unsigned (&seen)[4])
{
    unsigned bits = 0;
    for (unsigned w = 0; w < blockDim.x / 64; w++) bits |= seen[w];
    return bits;
}
// the next row behind `row` that names `slot` (`rows`: there is none), looked for by whole wavefronts
__device__ __forceinline__ int next_row_of(const int32_t* __restrict__ slots, int rows, int row, int slot)
{
    const int lane = threadIdx.x & 63;
    for (int at = row + 1; at < rows; at += 64) {
        const uint64_t hit = __ballot(at + lane < rows && slots[min(at + lane, rows - 1)] == slot);
        if (hit) return at + __ffsll((unsigned long long)hit) - 1;
    }
    return rows;
}
// Rows of one of a step's launches: each block looks through all of its launch's slots, so the work grows with the square of the
// rows.  65536 rows of 128 bf16 channels: convolution (4 taps) 2264 us in one launch, 289, 265 and 369 in launches of 4096, 2048
// and 1024 rows; scan (16 states) 3081, 660, 623 and 662.  Launches behind each other keep the rows' order, shared slots included.
constexpr int64_t kStepRows = 2048;
#endif
