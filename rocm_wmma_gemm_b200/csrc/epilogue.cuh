// Device side of the products with epilogues and of the grouped products: the activation
// functions and their derivatives, the epilogue's parameters, ragged-row bookkeeping, and the
// kernels around the tcgen05 GEMM (bias gradient sums, backward of an activation).
//
//   forward    Z = A*B + bias      C = act(Z) + residual          (Z kept on request)
//   gradient   C = (A*B) .* act'(Z)      bias_grad = sum of C over the rows, before rounding
//
// All of it is computed in f32 from the f32 accumulators and rounded once, when C (and Z) are
// stored; the bias gradient is a sum of the unrounded f32 values.
#pragma once

#include "ptx_sm100.cuh"

#include <cuda_bf16.h>
#include <cuda_fp16.h>

#include <type_traits>

namespace b200 {

// Activations.  silu and the tanh form of gelu are one function, x * sigmoid(x * (c0 + c1 x^2)):
// silu has c0 = 1, c1 = 0; 0.5 x (1 + tanh(u)) = x * sigmoid(2 u) with
// 2 u = 2 sqrt(2 / pi) (x + 0.044715 x^3).
enum : uint32_t { ACT_NONE = 0, ACT_RELU = 1, ACT_SIGMOID = 2, ACT_GELU = 3 };

enum : uint32_t { RAGGED_NONE = 0, RAGGED_ROWS = 1, RAGGED_K = 2 };

constexpr uint32_t MAX_GROUPS = 1024;

// Division by a number the host knows, for dividends below 2^31: with l = ceil(log2 d) and
// m = floor(2^(31 + l) / d) + 1, n / d = (n m) >> (31 + l) (m d exceeds 2^(31 + l) by at most d <= 2^l, so
// the excess n (m d - 2^(31 + l)) / d stays below one step).  A hardware division costs an epilogue
// warp some 150 cycles, and a tile's coordinates took four.
struct FastDiv {
    uint32_t d, m, shift;
};
__device__ __forceinline__ uint32_t fast_div(uint32_t n, const FastDiv& f) { return f.d == 1u ? n : __umulhi(n, f.m) >> f.shift; }

struct EpilogueParams {
    const void*    bias;        // forward: nullptr or one value per column of the caller's C, C's type
    const void*    residual;    // forward: nullptr or a matrix like C (may be C itself)
    void*          preact;      // forward: nullptr or where Z goes; gradient: Z (may be C itself)
    float*         part;        // gradient: nullptr or partial bias gradients [batch][part_blocks][length]
    uint64_t       bias_stride; // elements between the biases of consecutive batch items / groups
    uint32_t       act;
    float          k0, k1;      // ACT_SIGMOID: -c0 log2(e), -c1 log2(e); silu's k1 is the smallest normal number, so that k1 x^2 is not 0 times infinity
    float          slope0, slope1; // ACT_SIGMOID: c0, 3 c1
    uint32_t       gradient;
    uint32_t       part_blocks; // blocks per batch item (all groups together)
    uint32_t       part_rows;   // rows of the caller's C per block
    uint32_t       ragged;
    const int32_t* offsets;     // ragged: groups + 1 row offsets on the device
    uint32_t       groups;
    uint32_t       rows;        // ragged: rows of the ragged operands
    // the products only
    uint32_t           bias_on_rows; // the bias runs along the kernel view's rows, not its columns
    uint32_t           streamed;     // a matrix is read through the staging buffers (EpilogueMaps::in)
    uint32_t           aux;          // Z is written (EpilogueMaps::aux)
    uint32_t           unaligned;    // TMA cannot address C or the matrices like it
    uint32_t           plain;        // nothing but the conversion to C's type
    uint32_t           whole_a, whole_b; // pairs: an MN-major operand's 128 rows arrive in one box (encode_operand_pair)
    uint32_t           bufs;         // staging buffers per warp for C: 1 or 2
    uint32_t           table_at;     // ragged: byte offset of the group table in dynamic shared memory
    FastDiv            per_item, per_band, per_column; // tiles per batch item (ragged rows: of the other extent), per raster band, rows per band or column
    const CUtensorMap* maps;         // ragged K: two maps per group, their row extents ending at the group's end
};

// Two elements at a time: the packed f32 instructions halve the issue slots of everything but the
// special functions.
__device__ __forceinline__ float2 splat(float v) { return make_float2(v, v); }
__device__ __forceinline__ float  ex2(float x)
{
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float rcp(float x)
{
    float y;
    asm("rcp.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ float2 ex2(float2 x) { return make_float2(ex2(x.x), ex2(x.y)); }
__device__ __forceinline__ float2 rcp(float2 x) { return make_float2(rcp(x.x), rcp(x.y)); }

constexpr float LOG2E = 1.4426950408889634f;

// Minimum and maximum that keep a NaN.
__device__ __forceinline__ float min_nan(float a, float b)
{
    float y;
    asm("min.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}
__device__ __forceinline__ float max_nan(float a, float b)
{
    float y;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(y) : "f"(a), "f"(b));
    return y;
}

// Arguments are taken at most this large where an infinity would meet a factor that has become 0
// (NaN): x itself, or x^2, which overflows from 1.8e19 on.  Every sigmoid and tail here is 0 or 1
// in f32 from |x| = 105 on, so nothing else changes, and the infinities get the limits (a Z that has
// overflowed in f16 has a slope).  Cost, 4096 x 4096 x 1024: value 33.5 -> 34.1 us, slope 46.6 -> 47.4
// (silu and tanh gelu); nothing with the exact gelu, whose formulas are shorter in |x|.
constexpr float FAR = 1e9f;
__device__ __forceinline__ float2 not_below(float2 x) { return make_float2(max_nan(x.x, -FAR), max_nan(x.y, -FAR)); }
__device__ __forceinline__ float2 not_above(float2 x) { return make_float2(min_nan(x.x, FAR), min_nan(x.y, FAR)); }

// The same for pairs of 16-bit values (f16: the infinities become the largest values), where the slope is
// a sigmoid's; half the instructions.
template <uint32_t ACT, class T, int N>
__device__ __forceinline__ void limit_words(uint32_t (&w)[N])
{
    if constexpr (ACT == ACT_SIGMOID && sizeof(T) == 2) {
#pragma unroll
        for (int i = 0; i < N; ++i) {
            if constexpr (std::is_same_v<T, __half>)
                asm("max.NaN.f16x2 %0, %0, %1;\n\tmin.NaN.f16x2 %0, %0, %2;" : "+r"(w[i]) : "r"(0xfbfffbffu), "r"(0x7bff7bffu));
            else
                asm("max.NaN.bf16x2 %0, %0, %1;\n\tmin.NaN.bf16x2 %0, %0, %2;" : "+r"(w[i]) : "r"(0xce6ece6eu), "r"(0x4e6e4e6eu)); // FAR
        }
    }
}

// sigmoid(x (c0 + c1 x^2)) for k0 = -c0 log2(e), k1 = -c1 log2(e); x2 = x^2.  Far left 2^s overflows to
// infinity and its reciprocal is 0, which is right; so it is where x2 has overflowed.
__device__ __forceinline__ float2 sigmoid_of(float2 x, float2 x2, float k0, float k1)
{
    const float2 s = __fmul2_rn(x, __ffma2_rn(x2, splat(k1), splat(k0)));
    return rcp(__fadd2_rn(ex2(s), splat(1.f)));
}

// Normal distribution for a = |x| <= FAR: tail = 1 - Phi(a) and e = exp(-a^2 / 2), which the density shares.
// The tail is e / 2 times a polynomial in t = 1 / (1 + 0.3275911 a / sqrt 2): Abramowitz and Stegun 7.1.26,
// erf within 1.5e-7; in f32 the tail is within 0.75e-7 + 5.5e-7 e.  The error is absolute: relative to
// the tail it is 5e-5 at a = 3, 1.6e-3 at 5 and 3.6e-3 at 6.
__device__ __forceinline__ void normal_tail(float2 a, float2& tail, float2& e)
{
    const float2 t = rcp(__ffma2_rn(a, splat(0.23164190f), splat(1.f)));
    e              = ex2(__fmul2_rn(__fmul2_rn(a, a), splat(-0.5f * LOG2E)));
    float2 q       = __ffma2_rn(t, splat(0.5f * 1.061405429f), splat(0.5f * -1.453152027f));
    q              = __ffma2_rn(q, t, splat(0.5f * 1.421413741f));
    q              = __ffma2_rn(q, t, splat(0.5f * -0.284496736f));
    q              = __ffma2_rn(q, t, splat(0.5f * 0.254829592f));
    tail           = __fmul2_rn(__fmul2_rn(q, t), e);
}

// The activation and its slope.  (A NaN stays a NaN under every activation.)
template <uint32_t ACT>
__device__ __forceinline__ float2 act_value(float2 x, const EpilogueParams& ep)
{
    if constexpr (ACT == ACT_RELU) {
        return make_float2(x.x < 0.f ? 0.f : x.x, x.y < 0.f ? 0.f : x.y);
    } else if constexpr (ACT == ACT_SIGMOID) {
        const float2 c = not_below(x); // (only minus infinity would meet a 0)
        return __fmul2_rn(c, sigmoid_of(c, __fmul2_rn(c, c), ep.k0, ep.k1));
    } else if constexpr (ACT == ACT_GELU) {
        const float2 a = not_above(make_float2(fabsf(x.x), fabsf(x.y)));
        float2       tail, e;
        normal_tail(a, tail, e);
        // x Phi(x) = -a tail on the left, x - a tail on the right (fmaxf loses a NaN, a keeps it)
        return __ffma2_rn(make_float2(-a.x, -a.y), tail, make_float2(fmaxf(x.x, 0.f), fmaxf(x.y, 0.f)));
    } else {
        return x;
    }
}

// LIMITED: x has been through limit_words.
template <uint32_t ACT, bool LIMITED = false>
__device__ __forceinline__ float2 act_slope(float2 x, const EpilogueParams& ep)
{
    if constexpr (ACT == ACT_RELU) {
        return make_float2(x.x > 0.f ? 1.f : (x.x <= 0.f ? 0.f : x.x), x.y > 0.f ? 1.f : (x.y <= 0.f ? 0.f : x.y));
    } else if constexpr (ACT == ACT_SIGMOID) {
        // d/dx x s(u(x)) = s + x s (1 - s) u'(x),  u = c0 x + c1 x^3
        const float2 c  = LIMITED ? x : not_above(not_below(x));
        const float2 x2 = __fmul2_rn(c, c);
        const float2 s  = sigmoid_of(c, x2, ep.k0, ep.k1);
        const float2 w  = __fmul2_rn(__fmul2_rn(c, s), __ffma2_rn(s, splat(-1.f), splat(1.f)));
        return __ffma2_rn(w, __ffma2_rn(x2, splat(ep.slope1), splat(ep.slope0)), s);
    } else if constexpr (ACT == ACT_GELU) {
        // Phi(x) + x phi(x) = r on the left and 1 - r on the right, r = tail(a) - a phi(a)
        const float2 a = not_above(make_float2(fabsf(x.x), fabsf(x.y)));
        float2       tail, e;
        normal_tail(a, tail, e);
        const float2 r = __ffma2_rn(__fmul2_rn(a, splat(-0.39894228f)), e, tail);
        return make_float2(x.x > 0.f ? 1.f - r.x : r.x, x.y > 0.f ? 1.f - r.y : r.y);
    } else {
        return splat(1.f);
    }
}

// One element.
template <uint32_t ACT>
__device__ __forceinline__ float act_value(float x, const EpilogueParams& ep) { return act_value<ACT>(splat(x), ep).x; }
template <uint32_t ACT>
__device__ __forceinline__ float act_slope(float x, const EpilogueParams& ep) { return act_slope<ACT>(splat(x), ep).x; }

// Calls f with the activation as a compile-time constant (the loop over a tile's elements is
// inside f, so the choice is made once per chunk).
template <uint32_t V>
struct ActTag {
    static constexpr uint32_t value = V;
};
template <class F>
__device__ __forceinline__ void with_act(uint32_t act, F&& f)
{
    switch (act) {
        case ACT_RELU: f(ActTag<ACT_RELU>{}); break;
        case ACT_SIGMOID: f(ActTag<ACT_SIGMOID>{}); break;
        case ACT_GELU: f(ActTag<ACT_GELU>{}); break;
        default: f(ActTag<ACT_NONE>{}); break;
    }
}

template <class T>
__device__ __forceinline__ float to_f32(T v) { return static_cast<float>(v); }
template <class T>
__device__ __forceinline__ T from_f32(float v)
{
    if constexpr (sizeof(T) == 4) return v;
    else if constexpr (std::is_same_v<T, __half>) return __float2half_rn(v);
    else return __float2bfloat16_rn(v);
}

// ---------------------------------------------------------------------------------------------
// Ragged rows.  Group e owns rows [first_row(e), first_row(e + 1)).  Offsets are used as their
// running maximum clamped to [0, rows]: whatever the array holds, every row index stays inside
// the matrices, every row has at most one owner and the tiles of all groups together are at
// most rows / tile + groups.
// ---------------------------------------------------------------------------------------------
__device__ __forceinline__ uint32_t clamp_offset(int32_t v, uint32_t rows)
{
    return v < 0 ? 0u : min(static_cast<uint32_t>(v), rows);
}

__device__ __forceinline__ uint32_t warp_scan_max(uint32_t v, uint32_t lane)
{
#pragma unroll
    for (uint32_t d = 1; d < 32; d *= 2) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v = max(v, t);
    }
    return v;
}

__device__ __forceinline__ uint32_t warp_scan_add(uint32_t v, uint32_t lane)
{
#pragma unroll
    for (uint32_t d = 1; d < 32; d *= 2) {
        const uint32_t t = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += t;
    }
    return v;
}

// First partial-sum block of a group: blocks of `part_rows` rows start at the group's first row.
// floor(first / b) + e is non-decreasing and leaves room for ceil(length / b) blocks per group.
__device__ __forceinline__ uint32_t group_first_block(uint32_t first_row, uint32_t e, uint32_t part_rows)
{
    return first_row / part_rows + e;
}

// Walks the groups in order, 32 at a time, by one warp: f(g, lo, hi) for group g = this lane's of the 32,
// with its sanitised rows [lo, hi) (empty past the last group); stops when f returns true.  The
// offsets of GROUP_BATCH x 32 groups are loaded together, so that their latencies overlap.
constexpr uint32_t GROUP_BATCH = 4;

template <class F>
__device__ __forceinline__ void for_each_group(const int32_t* offsets, uint32_t groups, uint32_t rows, F&& f)
{
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t       top  = clamp_offset(offsets[0], rows); // running maximum up to the first of the 32
    for (uint32_t b0 = 0; b0 < groups; b0 += 32u * GROUP_BATCH) {
        uint32_t end[GROUP_BATCH];
#pragma unroll
        for (uint32_t i = 0; i < GROUP_BATCH; ++i) {
            const uint32_t g = b0 + i * 32u + lane;
            end[i]           = g < groups ? clamp_offset(offsets[g + 1u], rows) : 0u;
        }
#pragma unroll
        for (uint32_t i = 0; i < GROUP_BATCH; ++i) {
            if (b0 + i * 32u >= groups) return;
            const uint32_t hi = max(warp_scan_max(end[i], lane), top);
            uint32_t       lo = __shfl_up_sync(0xffffffffu, hi, 1);
            if (lane == 0) lo = top;
            if (f(b0 + i * 32u + lane, lo, hi)) return;
            top = __shfl_sync(0xffffffffu, hi, 31);
        }
    }
}

// The group and rows of row-tile number `want` (tiles of `tile` rows, groups in order); the whole
// warp takes part.  False when there are fewer tiles.
__device__ __forceinline__ bool locate_row_tile(const int32_t* offsets, uint32_t groups, uint32_t rows,
                                                uint32_t tile, uint32_t want, uint32_t& e, uint32_t& first,
                                                uint32_t& row0, uint32_t& row1)
{
    const uint32_t lane   = threadIdx.x & 31u;
    uint32_t       before = 0u; // tiles of the groups so far
    bool           found  = false;
    for_each_group(offsets, groups, rows, [&](uint32_t g, uint32_t lo, uint32_t hi) {
        const uint32_t tiles = (hi - lo + tile - 1u) / tile;
        const uint32_t incl  = before + warp_scan_add(tiles, lane);
        const uint32_t hit   = __ballot_sync(0xffffffffu, want < incl);
        if (hit) {
            const int src      = __ffs(hit) - 1;
            e                  = __shfl_sync(0xffffffffu, g, src);
            first              = __shfl_sync(0xffffffffu, lo, src);
            const uint32_t end = __shfl_sync(0xffffffffu, hi, src);
            const uint32_t tb  = __shfl_sync(0xffffffffu, incl - tiles, src);
            row0               = first + (want - tb) * tile;
            row1               = min(end, row0 + tile);
            found              = true;
            return true;
        }
        before = __shfl_sync(0xffffffffu, incl, 31);
        return false;
    });
    return found;
}

// Rows [lo, hi) of group e; the whole warp takes part.
__device__ __forceinline__ void group_rows(const int32_t* offsets, uint32_t e, uint32_t rows, uint32_t& lo,
                                           uint32_t& hi)
{
    const uint32_t lane = threadIdx.x & 31u;
    uint32_t       top  = 0u;
#pragma unroll 8
    for (uint32_t g = lane; g <= e; g += 32u) top = max(top, clamp_offset(offsets[g], rows));
#pragma unroll
    for (int d = 16; d > 0; d /= 2) top = max(top, __shfl_xor_sync(0xffffffffu, top, d));
    lo = top;
    hi = max(lo, clamp_offset(offsets[e + 1u], rows));
}

// ---------------------------------------------------------------------------------------------
// Bias gradient from the partial sums: out[g][n] = sum over g's blocks of part[block][n], blocks
// in a fixed order, so the result does not depend on timing.  blockIdx.y = g: a batch item
// (`items` items per output: all of them when the bias is shared) or a group of ragged rows.
// ---------------------------------------------------------------------------------------------
constexpr uint32_t SUM_LANES = 16;

static __global__ void __launch_bounds__(32 * SUM_LANES)
    bias_grad_sum_kernel(const float* part, float* out, uint32_t length, uint64_t out_stride,
                         uint64_t blocks, const int32_t* offsets, uint32_t rows, uint32_t part_rows)
{
    __shared__ float s_sum[SUM_LANES][32];
    const uint32_t tx = threadIdx.x & 31u, ty = threadIdx.x >> 5, n = blockIdx.x * 32u + tx;
    ptx::grid_dep_wait(); // the partial sums are those of the kernel before this one
    ptx::grid_dep_launch();
    uint64_t b0 = static_cast<uint64_t>(blockIdx.y) * blocks, count = blocks;
    if (offsets) {
        uint32_t lo, hi;
        group_rows(offsets, blockIdx.y, rows, lo, hi);
        b0    = group_first_block(lo, blockIdx.y, part_rows);
        count = (hi - lo + part_rows - 1u) / part_rows;
    }
    float s = 0.f;
    if (n < length)
#pragma unroll 4
        for (uint64_t b = ty; b < count; b += SUM_LANES) s += part[(b0 + b) * length + n];
    s_sum[ty][tx] = s;
    __syncthreads();
    if (ty == 0 && n < length) {
        float t = 0.f;
#pragma unroll
        for (uint32_t i = 0; i < SUM_LANES; ++i) t += s_sum[i][tx];
        out[blockIdx.y * out_stride + n] = t;
    }
}

// ---------------------------------------------------------------------------------------------
// Epilogue of a product whose K partitions lie in an f32 workspace: adds them in partition order and
// applies the epilogue to the sum.  Memory view of C: `lines` lines of `length` contiguous elements
// per batch item (a multiple of 4).  A block covers `strip` lines x 256 elements: threadIdx.x owns
// four neighbouring elements, threadIdx.y every fourth line.  Without bias gradients a strip is four
// lines, one per thread: a thread's loads wait for its stores to the line before.  Bias gradients only
// where the bias runs along the lines' elements (row-major C): a block's sums are one row of partials.
// L2-bound: (4 split + sizeof(out) x matrices) bytes per element.
// ---------------------------------------------------------------------------------------------
constexpr uint32_t SPLIT_STRIP = 16; // with bias gradients

template <class T>
__global__ void __launch_bounds__(256)
    splitk_epilogue_kernel(const float* ws, T* out, const EpilogueParams ep, uint32_t lines, uint32_t length, uint32_t split, uint32_t strip)
{
    __shared__ float4 s_sum[4][64];
    const uint32_t tx = threadIdx.x, ty = threadIdx.y, n = (blockIdx.x * 64u + tx) * 4u;
    const uint32_t l0 = blockIdx.y * strip, z = blockIdx.z;
    ptx::grid_dep_wait(); // the partials are complete once the product's grid has finished
    ptx::grid_dep_launch();
    const uint64_t item = static_cast<uint64_t>(lines) * length;
    const float*   part = ws + z * split * item;
    const T*       bias = static_cast<const T*>(ep.bias) + (ep.bias ? z * ep.bias_stride : 0u);
    const T*       read = static_cast<const T*>(ep.gradient ? ep.preact : ep.residual);
    T*             aux  = ep.aux ? static_cast<T*>(ep.preact) : nullptr;
    float          sum[4] = {};
    // four elements of C's type
    struct alignas(4 * sizeof(T)) Four {
        T v[4];
    };
    if (n < length) {
        float b[4] = {};
        if (ep.bias && !ep.bias_on_rows)
#pragma unroll
            for (int k = 0; k < 4; ++k) b[k] = to_f32(bias[n + k]);
        for (uint32_t l = l0 + ty; l < min(lines, l0 + strip); l += 4u) {
            const uint64_t at = static_cast<uint64_t>(l) * length + n, to = z * item + at;
            float4         a  = *reinterpret_cast<const float4*>(part + at);
#pragma unroll 4
            for (uint32_t s = 1; s < split; ++s) {
                const float4 t = *reinterpret_cast<const float4*>(part + s * item + at);
                a.x += t.x, a.y += t.y, a.z += t.z, a.w += t.w;
            }
            float v[4] = {a.x, a.y, a.z, a.w}, r[4] = {};
            if (ep.streamed) {
                const Four f = *reinterpret_cast<const Four*>(read + to);
#pragma unroll
                for (int k = 0; k < 4; ++k) r[k] = to_f32(f.v[k]);
            }
            Four o;
            if (ep.gradient) {
                if (ep.streamed)
                    with_act(ep.act, [&](auto tag) {
                        constexpr uint32_t ACT = decltype(tag)::value;
#pragma unroll
                        for (int k = 0; k < 4; ++k) v[k] = __fmul_rn(v[k], act_slope<ACT>(r[k], ep));
                    });
#pragma unroll
                for (int k = 0; k < 4; ++k) sum[k] += v[k];
            } else {
                if (ep.bias && ep.bias_on_rows) b[0] = b[1] = b[2] = b[3] = to_f32(bias[l]);
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += b[k];
                if (aux) {
#pragma unroll
                    for (int k = 0; k < 4; ++k) o.v[k] = from_f32<T>(v[k]);
                    *reinterpret_cast<Four*>(aux + to) = o;
                }
                with_act(ep.act, [&](auto tag) {
                    constexpr uint32_t ACT = decltype(tag)::value;
#pragma unroll
                    for (int k = 0; k < 4; ++k) v[k] = act_value<ACT>(v[k], ep);
                });
#pragma unroll
                for (int k = 0; k < 4; ++k) v[k] += r[k];
            }
#pragma unroll
            for (int k = 0; k < 4; ++k) o.v[k] = from_f32<T>(v[k]);
            *reinterpret_cast<Four*>(out + to) = o;
        }
    }
    if (!ep.part) return;
    s_sum[ty][tx] = make_float4(sum[0], sum[1], sum[2], sum[3]);
    __syncthreads();
    if (ty == 0 && n < length) {
        float4 t = s_sum[0][tx];
#pragma unroll
        for (int y = 1; y < 4; ++y) t.x += s_sum[y][tx].x, t.y += s_sum[y][tx].y, t.z += s_sum[y][tx].z, t.w += s_sum[y][tx].w;
        *reinterpret_cast<float4*>(ep.part + (static_cast<uint64_t>(z) * ep.part_blocks + blockIdx.y) * length + n) = t;
    }
}

// ---------------------------------------------------------------------------------------------
// Backward of an activation where no product precedes it: dZ = dY .* act'(Z), and the sums of dZ
// over the rows (of the rounded f32 products: no contraction into the sum, so that the sums are the
// same bits whether dZ is stored or not).  Memory view: `lines` lines of `length` contiguous elements.  Row-major C: a
// line is a row and the sums run over lines; column-major C: a line is a column and the sums run
// along it.
// ---------------------------------------------------------------------------------------------
struct ActBackwardParams {
    void*       dz;     // nullptr: only the sums are wanted
    const void* dy;
    const void* z;      // nullptr with ACT_NONE
    uint32_t    lines, length;
    uint32_t    strip;  // row-major: lines per block; column-major: elements of a line per block
    uint32_t    blocks_x;
    uint64_t    stride; // elements per batch item
    uint32_t    z0;
};

// V neighbouring elements: 16 bytes, or one.
template <class T, int V>
struct Pack {
    alignas(V > 1 ? 16 : sizeof(T)) T v[V];
    __device__ __forceinline__ void load(const T* from)
    {
        if constexpr (V > 1) {
            static_assert(V * sizeof(T) == 16, "a pack is 16 bytes");
            const uint4 w = __ldcs(reinterpret_cast<const uint4*>(from));
            *reinterpret_cast<uint4*>(v) = w;
        } else {
            v[0] = *from;
        }
    }
    __device__ __forceinline__ void store(T* to) const
    {
        if constexpr (V > 1) __stcs(reinterpret_cast<uint4*>(to), *reinterpret_cast<const uint4*>(v));
        else *to = v[0];
    }
};

// Two neighbouring values as f32 and back, by the packed conversions.
template <class T>
__device__ __forceinline__ float2 load_pair(const T* from)
{
    if constexpr (sizeof(T) == 4) return make_float2(from[0], from[1]);
    else if constexpr (std::is_same_v<T, __half>) return __half22float2(*reinterpret_cast<const __half2*>(from));
    else return __bfloat1622float2(*reinterpret_cast<const __nv_bfloat162*>(from));
}
template <class T>
__device__ __forceinline__ void store_pair(T* to, float2 v)
{
    if constexpr (sizeof(T) == 4) to[0] = v.x, to[1] = v.y;
    else if constexpr (std::is_same_v<T, __half>) *reinterpret_cast<__half2*>(to) = __float22half2_rn(v);
    else *reinterpret_cast<__nv_bfloat162*>(to) = __float22bfloat162_rn(v);
}

// g becomes dZ = g act'(x); its f32 values are added to `sum`.
template <uint32_t ACT, class T, int V>
__device__ __forceinline__ void act_backward_pack(Pack<T, V>& g, Pack<T, V>& x, float (&sum)[V], const EpilogueParams& ep)
{
    if constexpr (V > 1) {
        if constexpr (sizeof(T) == 2) limit_words<ACT, T>(reinterpret_cast<uint32_t (&)[V / 2]>(x.v));
#pragma unroll
        for (int i = 0; i < V; i += 2) {
            float2 v = load_pair(g.v + i);
            if constexpr (ACT != ACT_NONE) v = __fmul2_rn(v, act_slope<ACT, sizeof(T) == 2>(load_pair(x.v + i), ep));
            store_pair(g.v + i, v);
            const float2 t = __fadd2_rn(make_float2(sum[i], sum[i + 1]), v);
            sum[i] = t.x, sum[i + 1] = t.y;
        }
    } else {
        float v = to_f32(g.v[0]);
        if constexpr (ACT != ACT_NONE) v = __fmul_rn(v, act_slope<ACT>(to_f32(x.v[0]), ep));
        g.v[0] = from_f32<T>(v);
        sum[0] += v;
    }
}

constexpr uint32_t ACT_ROWS = 4; // packs in flight per thread and operand

// Row-major: each thread owns V consecutive columns (V = 16 bytes' worth, or 1 where the rows are
// not 16-byte aligned) and walks the strip's lines; threads of equal column and different
// threadIdx.y share a strip and add their sums through shared memory.  HBM-bound: three matrices.
template <class T, int V>
__global__ void __launch_bounds__(256) act_backward_rows_kernel(const ActBackwardParams p, const EpilogueParams ep)
{
    __shared__ float    s_sum[256 * V];
    __shared__ uint32_t s_where[4];
    const uint32_t tx = threadIdx.x, ty = threadIdx.y, tid = ty * blockDim.x + tx;
    const uint32_t n  = ((blockIdx.x % p.blocks_x) * blockDim.x + tx) * V;
    const uint32_t st = blockIdx.x / p.blocks_x;
    uint32_t       r0 = st * p.strip, r1 = min(p.lines, r0 + p.strip);
    uint64_t       block = static_cast<uint64_t>(blockIdx.z + p.z0) * ep.part_blocks + st;
    if (ep.ragged == RAGGED_ROWS) {
        if (tid < 32u) {
            uint32_t   e = 0, first = 0, a = 0, b = 0;
            const bool ok = locate_row_tile(ep.offsets, ep.groups, ep.rows, p.strip, st, e, first, a, b);
            if (tid == 0) {
                s_where[0] = ok ? 1u : 0u;
                s_where[1] = a;
                s_where[2] = b;
                s_where[3] = group_first_block(first, e, p.strip) + (a - first) / p.strip;
            }
        }
        __syncthreads();
        if (!s_where[0]) return;
        r0    = s_where[1];
        r1    = s_where[2];
        block = s_where[3];
    }
    const uint64_t base = (blockIdx.z + p.z0) * p.stride;
    const T*       dy   = static_cast<const T*>(p.dy) + base;
    const T*       z    = p.z ? static_cast<const T*>(p.z) + base : nullptr;
    T*             dz   = p.dz ? static_cast<T*>(p.dz) + base : nullptr;
    float          sum[V] = {};
    if (n < p.length) {
        with_act(ep.act, [&](auto tag) {
            constexpr uint32_t ACT = decltype(tag)::value;
            // ACT_ROWS lines' loads before their stores: dZ may be dY or Z, so the compiler cannot move a
            // later line's loads up by itself
            for (uint32_t r = r0 + ty; r < r1; r += ACT_ROWS * blockDim.y) {
                Pack<T, V> g[ACT_ROWS], x[ACT_ROWS];
#pragma unroll
                for (uint32_t k = 0; k < ACT_ROWS; ++k) {
                    const uint64_t at = static_cast<uint64_t>(r + k * blockDim.y) * p.length + n;
                    if (r + k * blockDim.y < r1) {
                        g[k].load(dy + at);
                        if (ACT != ACT_NONE) x[k].load(z + at);
                    }
                }
#pragma unroll
                for (uint32_t k = 0; k < ACT_ROWS; ++k) {
                    if (r + k * blockDim.y < r1) {
                        act_backward_pack<ACT>(g[k], x[k], sum, ep);
                        if (dz) g[k].store(dz + static_cast<uint64_t>(r + k * blockDim.y) * p.length + n);
                    }
                }
            }
        });
    }
    if (!ep.part) return;
#pragma unroll
    for (int i = 0; i < V; ++i) s_sum[tid * V + i] = sum[i];
    __syncthreads();
    if (ty == 0 && n < p.length) {
#pragma unroll
        for (int i = 0; i < V; ++i) {
            float t = 0.f;
            for (uint32_t y = 0; y < blockDim.y; ++y) t += s_sum[(y * blockDim.x + tx) * V + i];
            ep.part[block * p.length + n + i] = t;
        }
    }
}

// Column-major: one warp per line and strip.
template <class T, int V>
__global__ void __launch_bounds__(256) act_backward_cols_kernel(const ActBackwardParams p, const EpilogueParams ep)
{
    const uint32_t lane = threadIdx.x, line = (blockIdx.x / p.blocks_x) * blockDim.y + threadIdx.y;
    const uint32_t st = blockIdx.x % p.blocks_x;
    if (line >= p.lines) return;
    const uint32_t e0 = st * p.strip, e1 = min(p.length, e0 + p.strip);
    const uint64_t base = (blockIdx.z + p.z0) * p.stride + static_cast<uint64_t>(line) * p.length;
    const T*       dy   = static_cast<const T*>(p.dy) + base;
    const T*       z    = p.z ? static_cast<const T*>(p.z) + base : nullptr;
    T*             dz   = p.dz ? static_cast<T*>(p.dz) + base : nullptr;
    float          sum  = 0.f;
    float          sums[V] = {};
    with_act(ep.act, [&](auto tag) {
        constexpr uint32_t ACT = decltype(tag)::value;
        for (uint32_t i0 = e0 + lane * V; i0 < e1; i0 += ACT_ROWS * 32u * V) {
            Pack<T, V> g[ACT_ROWS], x[ACT_ROWS];
#pragma unroll
            for (uint32_t k = 0; k < ACT_ROWS; ++k) {
                if (i0 + k * 32u * V < e1) {
                    g[k].load(dy + i0 + k * 32u * V);
                    if (ACT != ACT_NONE) x[k].load(z + i0 + k * 32u * V);
                }
            }
#pragma unroll
            for (uint32_t k = 0; k < ACT_ROWS; ++k) {
                if (i0 + k * 32u * V < e1) {
                    act_backward_pack<ACT>(g[k], x[k], sums, ep);
                    if (dz) g[k].store(dz + i0 + k * 32u * V);
                }
            }
        }
    });
#pragma unroll
    for (int i = 0; i < V; ++i) sum += sums[i];
    if (!ep.part) return;
#pragma unroll
    for (int d = 16; d > 0; d /= 2) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if (lane == 0) ep.part[(static_cast<uint64_t>(blockIdx.z + p.z0) * ep.part_blocks + st) * p.lines + line] = sum;
}

} // namespace b200
