// Operators on rows of logits (include/leo_b200.h): penalties, biases and
// grammar masks; the pick of the next symbol; the cross entropy over the
// allowed symbols with its gradient.
//
// Each has to read the logits once (and write as much, except the pick); what it
// is bound by stands at its kernel.  Rows start anywhere, so they are read in groups of eight symbols
// laid so that the addresses are multiples of 16 bytes, the ends of a row one by
// one; a row of 257 classes and the like is one warp's in the loss.
#include <cooperative_groups.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <cmath>
#include <type_traits>

#include "../../include/leo_b200.h"
#include "leo_operator_device.cuh"
#include "leo_operator_host.h"

namespace {

using namespace leo_operator;
namespace cg = cooperative_groups;

constexpr uint32_t kAll = 0xffffffffu;

__device__ __forceinline__ float warp_max(float v) {
    for (int off = 16; off > 0; off >>= 1) v = fmaxf(v, __shfl_xor_sync(kAll, v, off));
    return v;
}
__device__ __forceinline__ float warp_sum(float v) {
    for (int off = 16; off > 0; off >>= 1) v += __shfl_xor_sync(kAll, v, off);
    return v;
}

// Eight neighbours of a row as they lie in memory.
template <typename T> struct Eight {
    uint4 raw[sizeof(T) / 2];
    __device__ __forceinline__ float operator[](int i) const {
        const uint32_t* w = reinterpret_cast<const uint32_t*>(raw);
        if constexpr (std::is_same_v<T, float>) {
            return __uint_as_float(w[i]);
        } else if constexpr (std::is_same_v<T, __nv_bfloat16>) {
            return __uint_as_float(i & 1 ? w[i / 2] & 0xffff0000u : w[i / 2] << 16);
        } else {
            return __half2float(__ushort_as_half((unsigned short)(w[i / 2] >> 16 * (i & 1))));
        }
    }
    __device__ __forceinline__ const uint32_t* words() const { return reinterpret_cast<const uint32_t*>(raw); }
    // Elements 2 i and 2 i + 1.
    __device__ __forceinline__ Pair32 pair(int i) const { return PairOf<T>::unpack(words() + i * (sizeof(T) / 2)); }
    __device__ __forceinline__ void set_pair(int i, Pair32 v) {
        PairOf<T>::pack(v, reinterpret_cast<uint32_t*>(raw) + i * (sizeof(T) / 2));
    }
    __device__ __forceinline__ float largest() const {
        if constexpr (std::is_same_v<T, float>) {
            float m = (*this)[0];
#pragma unroll
            for (int i = 1; i < 8; ++i) m = fmaxf(m, (*this)[i]);
            return m;
        } else {
            using Two = std::conditional_t<std::is_same_v<T, __nv_bfloat16>, __nv_bfloat162, __half2>;
            const Two* w = reinterpret_cast<const Two*>(raw);
            const Two m = __hmax2(__hmax2(w[0], w[1]), __hmax2(w[2], w[3]));
            return fmaxf(load(&m.x), load(&m.y));
        }
    }
    __device__ __forceinline__ void set(int i, float v) {  // i ascending
        uint32_t* w = reinterpret_cast<uint32_t*>(raw);
        if constexpr (std::is_same_v<T, float>) {
            w[i] = __float_as_uint(v);
        } else {
            uint32_t bits;
            if constexpr (std::is_same_v<T, __nv_bfloat16>)
                bits = __bfloat16_as_ushort(__float2bfloat16_rn(v));
            else
                bits = __half_as_ushort(__float2half_rn(v));
            w[i / 2] = i & 1 ? w[i / 2] | bits << 16 : bits;
        }
    }
};

// A row in groups of eight symbols whose addresses are multiples of 16 bytes:
// group g holds symbols first + 8 g and on; the first and the last may be short.
template <typename T>
struct Row {
    const T* p;
    int32_t first;  // at most 0
    uint32_t vocabulary, groups;
    __device__ __forceinline__ Row(const T* row, uint32_t vocabulary_) : p(row), vocabulary(vocabulary_) {
        const uint32_t off = (uint32_t)(reinterpret_cast<uintptr_t>(row) / sizeof(T)) % (16 / sizeof(T));
        first = -(int32_t)off;
        groups = (vocabulary + off + 7) / 8;
    }
    __device__ __forceinline__ bool whole(int32_t v) const { return v >= 0 && (uint32_t)v + 8 <= vocabulary; }
    __device__ __forceinline__ bool in(int32_t v) const { return (uint32_t)v < vocabulary; }
    // Symbols v .. v + 7; zero outside the row.
    __device__ __forceinline__ Eight<T> read(int32_t v) const {
        Eight<T> e;
        if (whole(v)) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) e.raw[i] = __ldcs(reinterpret_cast<const uint4*>(p + v) + i);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) e.set(i, in(v + i) ? load(p + v + i) : 0.0f);
        }
        return e;
    }
    // The same symbols of another row: whole groups at once where it is aligned alike.
    __device__ __forceinline__ bool alike(const T* other) const {
        return (reinterpret_cast<uintptr_t>(other) ^ reinterpret_cast<uintptr_t>(p)) % 16 == 0;
    }
    __device__ __forceinline__ void write(T* out, bool aligned, int32_t v, const Eight<T>& e) const {
        if (aligned && whole(v)) {
#pragma unroll
            for (int i = 0; i < (int)sizeof(T) / 2; ++i) __stcs(reinterpret_cast<uint4*>(out + v) + i, e.raw[i]);
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (in(v + i)) store(out + v + i, e[i]);
        }
    }
};

// What a row of the mask table says: all symbols, none, or its words.
struct MaskRow {
    const uint32_t* words;  // nullptr: see `open`
    bool open;
    __device__ __forceinline__ bool allows(uint32_t v) const {
        return words ? (words[v >> 5] >> (v & 31u)) & 1u : open;
    }
    // Bit i: symbol v + i is allowed, of those inside the row.
    __device__ __forceinline__ uint32_t eight(int32_t v, uint32_t vocabulary) const {
        if (!words) return open ? 0xffu : 0u;
        const int32_t low = max(v, 0) >> 5, high = min(v + 7, (int32_t)vocabulary - 1) >> 5;
        const uint64_t bits = (uint64_t)__ldg(words + high) << 32 | __ldg(words + low);
        // two words of one number are the same word
        return v < 0 ? (uint32_t)bits << -v & 0xffu : (uint32_t)((low == high ? bits & 0xffffffffu : bits) >> (v & 31)) & 0xffu;
    }
};

__device__ __forceinline__ MaskRow mask_row(const uint32_t* allowed, int64_t stride, uint32_t states,
                                            const int32_t* state, uint32_t row) {
    if (!allowed) return {nullptr, true};
    int64_t s = states == 1 ? 0 : row;
    if (state) s = state[row];
    if (s == -1) return {nullptr, true};
    if (s < 0 || s >= (int64_t)states) return {nullptr, false};
    return {allowed + s * stride, true};
}

struct RowRules {
    const int32_t* history;
    uint32_t length;
    float repetition, presence, frequency;
    const float* bias;
    MaskRow mask;
};

__device__ __forceinline__ RowRules row_rules(const LeoB200LogitRules& r, uint32_t row) {
    RowRules k;
    k.history = r.history ? r.history + (int64_t)row * r.history_stride : nullptr;
    int64_t n = r.history ? (int64_t)r.history_capacity : 0;
    if (r.history && r.lengths) n = min(n, max((int64_t)r.lengths[row], (int64_t)0));
    k.length = (uint32_t)n;
    k.repetition = r.repetition ? r.repetition[row] : r.repetition_value;
    k.presence = r.presence ? r.presence[row] : r.presence_value;
    k.frequency = r.frequency ? r.frequency[row] : r.frequency_value;
    k.bias = r.bias ? r.bias + (int64_t)row * r.bias_stride : nullptr;
    k.mask = mask_row(r.allowed, r.allowed_stride, r.states, r.state, row);
    return k;
}

// Counts of the history's symbols in [first, first + span), span a multiple of
// four, by the whole block.
__device__ __forceinline__ void count_history(const RowRules& k, int32_t first, uint32_t span, uint32_t* counts) {
    for (uint32_t i = threadIdx.x; i < span / 4; i += blockDim.x)
        reinterpret_cast<uint4*>(counts)[i] = make_uint4(0, 0, 0, 0);
    __syncthreads();
#pragma unroll 4
    for (uint32_t i = threadIdx.x; i < k.length; i += blockDim.x) {
        const int32_t symbol = __ldg(k.history + i);
        const uint32_t v = (uint32_t)(symbol - first);
        if (symbol >= 0 && v < span) atomicAdd(&counts[v], 1u);
    }
    __syncthreads();
}

__device__ __forceinline__ float quotient(float x, float y, float) { return x / y; }
// x / y rounded as a division is, from the rounded reciprocal of y (P. W.
// Markstein, IBM J. Res. Dev. 34, 1990): the remainder of the first quotient
// is exact, as x and y are floats and nothing leaves the range of double.  An
// infinite quotient has none.
__device__ __forceinline__ double quotient(double x, double y, double reciprocal) {
    const double q = x * reciprocal;
    return isinf(q) ? q : fma(fma(-q, y, x), reciprocal, q);
}

// The penalties, the bias and the mask, every operation rounded by itself in F.
template <typename F>
__device__ __forceinline__ F adjusted(F z, uint32_t count, const RowRules& k, F reciprocal, float bias, bool allowed) {
    const F penalised = (z > (F)0 ? quotient(z, (F)k.repetition, reciprocal) : z * (F)k.repetition) -
                        ((F)k.presence + (F)k.frequency * (F)count);
    z = count ? penalised : z;
    if (k.bias) z += (F)bias;
    return allowed ? z : -(F)CUDART_INF;
}

struct LogitArgs {
    const void* logits;
    int64_t logits_stride;
    uint32_t rows, vocabulary;
    LeoB200LogitRules rules;
    void* out;
    int64_t out_stride;
    // pick
    const float* temperature;
    float temperature_value;
    const double* uniforms;
    int32_t* symbols;
    float* log_probability;
};

// Biases of symbols v .. v + 7.
template <typename T>
__device__ __forceinline__ void read_bias(const RowRules& k, const Row<T>& row, int32_t v, float (&bias)[8]) {
    if (!k.bias) return;
    if (row.whole(v) && reinterpret_cast<uintptr_t>(k.bias + v) % 16 == 0) {
        const float4 x = __ldg(reinterpret_cast<const float4*>(k.bias + v)),
                     y = __ldg(reinterpret_cast<const float4*>(k.bias + v) + 1);
        bias[0] = x.x, bias[1] = x.y, bias[2] = x.z, bias[3] = x.w;
        bias[4] = y.x, bias[5] = y.y, bias[6] = y.z, bias[7] = y.w;
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) bias[i] = row.in(v + i) ? __ldg(k.bias + v + i) : 0.0f;
    }
}

// A block takes a run of a row, of up to kAdjustRun symbols: it counts the
// history's symbols in it once, in shared memory, then goes through it with the
// groups of the next turn in flight.  Any vocabulary and history fit, and the runs
// of a long row go side by side.  256 x 50,001 bfloat16 with 1,000 symbols of history
// and a bias row each: 27 us, 31 us with nothing in L2, where a copy's rate gives 16 us;
// 33 us in runs of 4,096 symbols, whose counts then take longer than their logits.
constexpr uint32_t kAdjustThreads = 256;
constexpr uint32_t kAdjustTurn = kAdjustThreads * 8;   // symbols of a turn
constexpr uint32_t kAdjustRun = 4 * kAdjustTurn;

template <typename T>
__global__ void __launch_bounds__(kAdjustThreads) adjust_kernel(const __grid_constant__ LogitArgs a, uint32_t runs,
                                                                uint32_t turns) {
    extern __shared__ __align__(16) uint32_t run_counts[];
    const uint32_t at = blockIdx.x / runs, run = blockIdx.x - at * runs;
    const Row<T> row(static_cast<const T*>(a.logits) + (int64_t)at * a.logits_stride, a.vocabulary);
    T* out = static_cast<T*>(a.out) + (int64_t)at * a.out_stride;
    const RowRules k = row_rules(a.rules, at);
    const bool aligned = row.alike(out);
    const int32_t first = row.first + (int32_t)(run * turns * kAdjustTurn);
    const auto symbol_of = [&](uint32_t turn) { return first + (int32_t)(turn * kAdjustTurn + threadIdx.x * 8); };
    Eight<T> next;
    float next_bias[8] = {};
    const auto ask = [&](uint32_t turn) {
        const int32_t v = symbol_of(turn);
        if (turn < turns && v < (int32_t)a.vocabulary) {
            next = row.read(v);
            read_bias(k, row, v, next_bias);
        }
    };
    ask(0);
    if (k.length) count_history(k, first, turns * kAdjustTurn, run_counts);
    for (uint32_t turn = 0; turn < turns; ++turn) {
        const int32_t v = symbol_of(turn);
        if (v >= (int32_t)a.vocabulary) return;
        const Eight<T> e = next;
        float bias[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) bias[i] = next_bias[i];
        ask(turn + 1);
        const uint32_t ok = k.mask.eight(v, a.vocabulary);
        uint4 c[2] = {};
        if (k.length) {
            c[0] = *reinterpret_cast<const uint4*>(run_counts + (v - first));
            c[1] = *reinterpret_cast<const uint4*>(run_counts + (v - first) + 4);
        }
        float z[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = k.bias ? e[i] + bias[i] : e[i];
        if (((c[0].x | c[0].y) | (c[0].z | c[0].w) | (c[1].x | c[1].y) | (c[1].z | c[1].w)) != 0) {
            const uint32_t count[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w};
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (count[i]) z[i] = adjusted(e[i], count[i], k, 0.0f, bias[i], true);
        }
        if (ok != 0xffu) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(ok >> i & 1u)) z[i] = -CUDART_INF_F;
        }
        Eight<T> r;
#pragma unroll
        for (int i = 0; i < 4; ++i) r.set_pair(i, pair_of(z[2 * i], z[2 * i + 1]));
        row.write(out, aligned, v, r);
    }
}

// exp(y ln 2 / 64) for y <= 0 after Tang's table-driven method (P. T. P. Tang,
// ACM TOMS 15, 1989): y = 64 q + j + d with |d| <= 1/2, so the value is
// 2^q 2^(j/64) exp(d ln 2 / 64), the last by its Taylor polynomial of degree 5
// in d (its rest is below 2^-58).  Below e^-708 it is 0, which no double sum
// beside a weight of 1 can tell.
constexpr uint32_t kPowers = 64;
__device__ const double kTwoTo[kPowers] = {
    0x1.0000000000000p+0, 0x1.02c9a3e778061p+0, 0x1.059b0d3158574p+0, 0x1.0874518759bc8p+0,
    0x1.0b5586cf9890fp+0, 0x1.0e3ec32d3d1a2p+0, 0x1.11301d0125b51p+0, 0x1.1429aaea92de0p+0,
    0x1.172b83c7d517bp+0, 0x1.1a35beb6fcb75p+0, 0x1.1d4873168b9aap+0, 0x1.2063b88628cd6p+0,
    0x1.2387a6e756238p+0, 0x1.26b4565e27cddp+0, 0x1.29e9df51fdee1p+0, 0x1.2d285a6e4030bp+0,
    0x1.306fe0a31b715p+0, 0x1.33c08b26416ffp+0, 0x1.371a7373aa9cbp+0, 0x1.3a7db34e59ff7p+0,
    0x1.3dea64c123422p+0, 0x1.4160a21f72e2ap+0, 0x1.44e086061892dp+0, 0x1.486a2b5c13cd0p+0,
    0x1.4bfdad5362a27p+0, 0x1.4f9b2769d2ca7p+0, 0x1.5342b569d4f82p+0, 0x1.56f4736b527dap+0,
    0x1.5ab07dd485429p+0, 0x1.5e76f15ad2148p+0, 0x1.6247eb03a5585p+0, 0x1.6623882552225p+0,
    0x1.6a09e667f3bcdp+0, 0x1.6dfb23c651a2fp+0, 0x1.71f75e8ec5f74p+0, 0x1.75feb564267c9p+0,
    0x1.7a11473eb0187p+0, 0x1.7e2f336cf4e62p+0, 0x1.82589994cce13p+0, 0x1.868d99b4492edp+0,
    0x1.8ace5422aa0dbp+0, 0x1.8f1ae99157736p+0, 0x1.93737b0cdc5e5p+0, 0x1.97d829fde4e50p+0,
    0x1.9c49182a3f090p+0, 0x1.a0c667b5de565p+0, 0x1.a5503b23e255dp+0, 0x1.a9e6b5579fdbfp+0,
    0x1.ae89f995ad3adp+0, 0x1.b33a2b84f15fbp+0, 0x1.b7f76f2fb5e47p+0, 0x1.bcc1e904bc1d2p+0,
    0x1.c199bdd85529cp+0, 0x1.c67f12e57d14bp+0, 0x1.cb720dcef9069p+0, 0x1.d072d4a07897cp+0,
    0x1.d5818dcfba487p+0, 0x1.da9e603db3285p+0, 0x1.dfc97337b9b5fp+0, 0x1.e502ee78b3ff6p+0,
    0x1.ea4afa2a490dap+0, 0x1.efa1bee615a27p+0, 0x1.f50765b6e4540p+0, 0x1.fa7c1819e90d8p+0};
constexpr double kSixtyFourths = 0x1.71547652b82fep+6;  // 64 / ln 2
__device__ __forceinline__ double exp_down(double y, const double* two_to) {
    const double magic = 0x1.8p52;
    // y < -65,372 (-inf too, by the bits of its high word)
    const bool none = (uint32_t)__double2hiint(y) >= 0xc0efeb80u;
    const double shifted = y + magic;
    const int32_t n = __double2loint(shifted);
    const double d = y - (shifted - magic);
    double p = fma(d, 0x1.5d87fe78a6731p-40, 0x1.3b2ab6fba4e77p-31);
    p = fma(p, d, 0x1.c6b08d704a0c0p-23);
    p = fma(p, d, 0x1.ebfbdff82c58fp-15);
    p = fma(p, d, 0x1.62e42fefa39efp-7) * d;
    const double scale = two_to[n & 63];
    const double v = fma(scale, p, scale);
    const int32_t high = __double2hiint(v) + ((n >> 6) << 20);
    return none ? 0.0 : __hiloint2double(high, __double2loint(v));
}

// 64 / ln 2 / heat.  Above 0, so that a masked place's -inf stays -inf at an infinite temperature.
__device__ __forceinline__ double cold_of(double heat) { return fmax(kSixtyFourths / heat, 0x1p-1000); }

// A sum of weights exp((z - top) / heat), by its own top; `cold` is cold_of(heat).
struct Weights {
    double top, sum;
};
__device__ __forceinline__ Weights no_weights() { return {-CUDART_INF, 0.0}; }
// A masked place's -inf gives 0 by itself; beside an infinite top only its equals count.
__device__ __forceinline__ double weight_of(double z, double top, double cold, const double* two_to) {
    return top == CUDART_INF ? (z == top ? 1.0 : 0.0) : exp_down((z - top) * cold, two_to);
}
__device__ __forceinline__ void weights_of(const double (&z)[8], double top, double cold, const double* two_to,
                                           double (&w)[8]) {
    if (top == CUDART_INF) {
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = z[i] == top ? 1.0 : 0.0;
    } else {  // eight at a time: an exponential is a chain of some fifteen operations
#pragma unroll
        for (int i = 0; i < 8; ++i) w[i] = exp_down((z[i] - top) * cold, two_to);
    }
}

// What a part of a row knows: its weights, its largest logit and the lowest
// symbol of that value, and whether a NaN is among them.
struct Part {
    Weights weights;
    uint32_t best;
    uint32_t bad;
};

// A cluster of blocks takes a row, each block a run of steps of 256 symbols,
// a step a warp.  One pass over the logits gives every step its weights (by a
// value near its own largest logit, so the row's is not needed first); the
// blocks exchange theirs through distributed shared memory, which says in which
// step the running sum passes u * total, and one warp walks that step again.
// Everything is in 64 bits: among 131,072 borders between symbols a float32 sum
// would put one in a hundred draws on the wrong side.  What bounds it is the 64-bit
// exponential, some 16 operations a symbol in a chain: 64 rows of 131,072 take 54 us,
// with the issue slots two fifths full; the operations take 9 us at the card's rate
// for them, the logits 3 us at its bandwidth.
constexpr uint32_t kStepSymbols = 256;
constexpr uint32_t kPickWindow = 96;  // steps whose counts are in shared memory at a time

template <typename T, int Warps>
__global__ void __launch_bounds__(32 * Warps) pick_kernel(const __grid_constant__ LogitArgs a, uint32_t steps) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    Weights* weights = reinterpret_cast<Weights*>(dynamic);              // [steps]
    uint32_t* counts = reinterpret_cast<uint32_t*>(weights + steps);     // of a window, if there is a history
    __shared__ double two_to[kPowers];
    __shared__ double warp_best[Warps];
    __shared__ uint32_t warp_at[Warps], warp_bad[Warps];
    __shared__ Part mine;
    __shared__ double block_best, before, target, row_best, row_total;
    __shared__ uint32_t chosen;  // step
    cg::cluster_group cluster = cg::this_cluster();
    const uint32_t blocks = cluster.num_blocks(), rank = cluster.block_rank();
    const uint32_t at = blockIdx.x / blocks, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const Row<T> row(static_cast<const T*>(a.logits) + (int64_t)at * a.logits_stride, a.vocabulary);
    const int32_t block_first = row.first + (int32_t)(rank * steps * kStepSymbols);
    const auto symbol_of = [&](uint32_t step) { return block_first + (int32_t)(step * kStepSymbols + lane * 8); };
    const auto inside = [&](uint32_t step) { return step < steps && symbol_of(step) < (int32_t)a.vocabulary; };
    Eight<T> next;
    float next_bias[8] = {};
    if (inside(warp)) next = row.read(symbol_of(warp));
    const RowRules k = row_rules(a.rules, at);
    if (inside(warp)) read_bias(k, row, symbol_of(warp), next_bias);
    const float temperature = a.temperature ? a.temperature[at] : a.temperature_value;
    const bool greedy = temperature == 0.0f;
    const double uniform = a.uniforms ? a.uniforms[at] : 0.0;
    const double heat = greedy ? 1.0 : (double)temperature, cold = cold_of(heat);
    const double reciprocal = 1.0 / (double)k.repetition;
    // A step's weights are taken by the float of its largest logit.  The two are 2^-24 of it
    // apart, which times `cold`, as weights see it, is at most a 64th of a power of two up to
    // here; beyond, where a small temperature makes more of it, the largest itself is found.
    const float near = (float)fmin(1e38, 0x1p24 / cold);
    for (uint32_t j = threadIdx.x; j < kPowers; j += 32 * Warps) two_to[j] = kTwoTo[j];

    // Bit i: symbol v + i is in the row and allowed.
    const auto allowed_at = [&](int32_t v) {
        uint32_t ok = k.mask.eight(v, a.vocabulary);
        if (!row.whole(v))
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!row.in(v + i)) ok &= ~(1u << i);
        return ok;
    };
    // The logits of a group after the rules, and roughly so, rounded to float once or twice;
    // `window`: the first symbol of the counts.
    const auto adjust = [&](const Eight<T>& e, const float (&bias)[8], int32_t v, int32_t window, double (&z)[8],
                            float (&rough)[8]) {
        const uint32_t ok = allowed_at(v);
        uint4 c[2] = {};
        if (k.length) {
            c[0] = *reinterpret_cast<const uint4*>(counts + (v - window));
            c[1] = *reinterpret_cast<const uint4*>(counts + (v - window) + 4);
        }
        const uint32_t count[8] = {c[0].x, c[0].y, c[0].z, c[0].w, c[1].x, c[1].y, c[1].z, c[1].w};
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            z[i] = k.bias ? (double)e[i] + (double)bias[i] : (double)e[i];
            rough[i] = k.bias ? e[i] + bias[i] : e[i];
        }
        if (((c[0].x | c[0].y) | (c[0].z | c[0].w) | (c[1].x | c[1].y) | (c[1].z | c[1].w)) != 0) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (count[i]) {  // a few in a step: most of a vocabulary has not been said
                    z[i] = adjusted((double)e[i], count[i], k, reciprocal, bias[i], true);
                    rough[i] = (float)z[i];
                }
        }
        if (ok != 0xffu) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!(ok >> i & 1u)) z[i] = -CUDART_INF, rough[i] = -CUDART_INF_F;
        }
    };

    double best_value = -CUDART_INF;
    float best_rough = -CUDART_INF_F;
    uint32_t best = kAll, bad = !(temperature >= 0.0f);
    for (uint32_t first = 0; first < steps; first += kPickWindow) {
        const int32_t window = block_first + (int32_t)(first * kStepSymbols);
        const uint32_t past = min(first + kPickWindow, steps);
        if (first) __syncthreads();  // the counts of the window before are read
        if (k.length)
            count_history(k, window, (past - first) * kStepSymbols, counts);
        else if (first == 0)
            __syncthreads();  // the table of powers
        for (uint32_t step = first + warp; step < past; step += Warps) {
            const Eight<T> e = next;
            float bias[8];
#pragma unroll
            for (int i = 0; i < 8; ++i) bias[i] = next_bias[i];
            const int32_t v = symbol_of(step);
            if (inside(step + Warps)) {
                next = row.read(symbol_of(step + Warps));
                read_bias(k, row, symbol_of(step + Warps), next_bias);
            }
            double z[8];
            float rough[8], most = -CUDART_INF_F;
            if (inside(step)) {
                adjust(e, bias, v, window, z, rough);
            } else {
#pragma unroll
                for (int i = 0; i < 8; ++i) z[i] = -CUDART_INF, rough[i] = -CUDART_INF_F;
            }
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                bad |= rough[i] != rough[i];
                most = fmaxf(most, rough[i]);
            }
            if (!(most < best_rough - fabsf(best_rough) * 0x1p-21f)) {  // float's order is double's but for neighbours
#pragma unroll
                for (int i = 0; i < 8; ++i)
                    if (z[i] > best_value) best_value = z[i], best = (uint32_t)(v + i);
                best_rough = fmaxf(best_rough, most);
            }
            most = warp_max(most);
            double top = (double)most;
            if (!(fabsf(most) < near)) {  // and what float calls infinite may not be
                top = z[0];
#pragma unroll
                for (int i = 1; i < 8; ++i) top = fmax(top, z[i]);
                for (int off = 16; off > 0; off >>= 1) top = fmax(top, __shfl_xor_sync(kAll, top, off));
            }
            double sum = 0.0;
            if (top != -CUDART_INF) {
                double w[8];
                weights_of(z, top, cold, two_to, w);
                sum = ((w[0] + w[1]) + (w[2] + w[3])) + ((w[4] + w[5]) + (w[6] + w[7]));
                for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kAll, sum, off);
            }
            if (lane == 0) weights[step] = {top, sum};
        }
    }
    // The block's part: its largest logit, and its weights by that.
    const auto join_best = [&](uint32_t width) {
        for (uint32_t off = width / 2; off > 0; off >>= 1) {
            const double v = __shfl_xor_sync(kAll, best_value, off);
            const uint32_t b = __shfl_xor_sync(kAll, best, off);
            if (v > best_value || (v == best_value && b < best)) best_value = v, best = b;
            bad |= __shfl_xor_sync(kAll, bad, off);
        }
    };
    // A sum of weights by another value.
    const auto by = [&](const Weights& w, double top) {
        return w.top == -CUDART_INF ? 0.0 : w.sum * weight_of(w.top, top, cold, two_to);
    };
    join_best(32);
    if (lane == 0) warp_best[warp] = best_value, warp_at[warp] = best, warp_bad[warp] = bad;
    __syncthreads();
    if (warp == 0) {
        const uint32_t w = lane % Warps;
        best_value = warp_best[w], best = warp_at[w], bad = warp_bad[w];
        join_best(Warps);
        double sum = 0.0;
        for (uint32_t j = lane; j < steps; j += 32) sum += by(weights[j], best_value);
        for (int off = 16; off > 0; off >>= 1) sum += __shfl_xor_sync(kAll, sum, off);
        if (lane == 0) mine = {{best_value, sum}, best, bad}, block_best = best_value;
        __syncwarp();
    }
    if (blocks > 1) cluster.sync();

    // The row's, the same in every block; its first warp goes on.
    if (warp == 0) {
        const Part part = lane < blocks ? (blocks > 1 ? *cluster.map_shared_rank(&mine, lane) : mine)
                                        : Part{no_weights(), kAll, 0};
        best_value = lane < blocks ? part.weights.top : -CUDART_INF;
        best = part.best, bad = part.bad;
        join_best(32);
        uint32_t pick = kAll;  // nothing to walk
        if (!bad && best != kAll) {
            const double share = blocks == 1 && lane == 0 ? part.weights.sum : by(part.weights, best_value);
            double total = 0.0;
            for (uint32_t j = 0; j < blocks; ++j) total += __shfl_sync(kAll, share, j);
            if (greedy) {
                if (rank == 0 && lane == 0) {
                    a.symbols[at] = (int32_t)best;
                    if (a.log_probability) a.log_probability[at] = (float)-log(total);
                }
            } else {
                // The block, then its step, in which the running sum passes u * total.
                const double goal = uniform * total;
                double sum = 0.0, sum_before = 0.0;
                uint32_t owner = kAll, last = 0;
                for (uint32_t j = 0; j < blocks; ++j) {
                    const double s = __shfl_sync(kAll, share, j);
                    if (owner == kAll && s > 0.0) {
                        sum_before = sum;
                        last = j;
                        if (sum + s > goal) owner = j;
                    }
                    sum += s;
                }
                if (owner == kAll) owner = last;  // u is nearly 1, and the sums were rounded
                if (rank == owner) {
                    double running = sum_before, step_before = sum_before;
                    uint32_t found = kAll, last_step = (mine.best - (uint32_t)block_first) / kStepSymbols;
                    for (uint32_t base = 0; base < steps && found == kAll; base += 32) {
                        const uint32_t j = base + lane;
                        const double s = j < steps ? by(weights[j], best_value) : 0.0;
                        double through = s;
                        for (int off = 1; off < 32; off <<= 1) {
                            const double o = __shfl_up_sync(kAll, through, off);
                            if (lane >= (uint32_t)off) through += o;
                        }
                        const uint32_t some = __ballot_sync(kAll, s > 0.0);
                        const uint32_t hits = __ballot_sync(kAll, s > 0.0 && running + through > goal);
                        if (some) {
                            const int from = hits ? __ffs(hits) - 1 : 31 - __clz(some);
                            last_step = base + from;
                            if (hits) found = last_step;
                            step_before = running + __shfl_sync(kAll, through - s, from);
                        }
                        running += __shfl_sync(kAll, through, 31);
                    }
                    pick = found != kAll ? found : last_step;
                    if (lane == 0) before = step_before, target = goal, row_best = best_value, row_total = total;
                }
            }
        } else if (rank == 0 && lane == 0) {
            a.symbols[at] = -1;
            if (a.log_probability) a.log_probability[at] = bad ? CUDART_NAN_F : -CUDART_INF_F;
        }
        if (lane == 0) chosen = pick;
    }
    // No block leaves before the others have read its part.
    if (blocks > 1)
        cluster.sync();
    else
        __syncthreads();
    if (chosen == kAll) return;

    // The step's counts are there, unless it lies in an earlier window.
    const uint32_t first = chosen / kPickWindow * kPickWindow;
    const int32_t window = block_first + (int32_t)(first * kStepSymbols);
    if (k.length && steps - first > kPickWindow) count_history(k, window, kPickWindow * kStepSymbols, counts);
    if (warp != 0) return;
    const double top = row_best, goal = target;
    const int32_t v = symbol_of(chosen);
    double z[8], w[8], sum = 0.0;
    float rough[8], bias[8] = {};
    if (v < (int32_t)a.vocabulary) {
        read_bias(k, row, v, bias);
        adjust(row.read(v), bias, v, window, z, rough);
    } else {
#pragma unroll
        for (int i = 0; i < 8; ++i) z[i] = -CUDART_INF;
    }
    weights_of(z, top, cold, two_to, w);
#pragma unroll
    for (int i = 0; i < 8; ++i) sum += w[i];
    double through = sum;  // of the lanes up to this one
    for (int off = 1; off < 32; off <<= 1) {
        const double o = __shfl_up_sync(kAll, through, off);
        if (lane >= (uint32_t)off) through += o;
    }
    double running = before + (through - sum);
    uint32_t hit = kAll, last = kAll;
    double hit_z = 0.0, last_z = 0.0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        running += w[i];
        if (w[i] > 0.0) {
            last = (uint32_t)(v + i), last_z = z[i];
            if (hit == kAll && running > goal) hit = last, hit_z = z[i];
        }
    }
    const uint32_t hits = __ballot_sync(kAll, hit != kAll);
    uint32_t some = __ballot_sync(kAll, last != kAll);
    if (some == 0) {  // the step had a weight by the float of its largest logit only: that symbol
#pragma unroll
        for (int i = 0; i < 8; ++i)
            if (last == kAll || z[i] > last_z) last = (uint32_t)(v + i), last_z = z[i];
        double most = last_z;
        for (int off = 16; off > 0; off >>= 1) most = fmax(most, __shfl_xor_sync(kAll, most, off));
        some = __ballot_sync(kAll, last_z == most);
        some &= -some;  // the lowest of equal ones
    }
    // The first lane with a hit, or, the sums having been rounded, the last with any weight.
    if (hits ? lane == (uint32_t)__ffs(hits) - 1u : lane == 31u - __clz(some)) {
        const double logit = hits ? hit_z : last_z;
        a.symbols[at] = (int32_t)(hits ? hit : last);
        if (a.log_probability)
            a.log_probability[at] = (float)((logit == top ? 0.0 : (logit - top) / heat) - log(row_total));
    }
}

// Rows of up to 128 N symbols, a block each and a symbol in N of a thread's
// registers from the logits to the pick: with a row's few symbols what counts is
// the length of the chain, and how much code a block runs through once.
template <typename T, int N>
__global__ void __launch_bounds__(128) narrow_pick_kernel(const __grid_constant__ LogitArgs a) {
    __shared__ __align__(16) uint32_t counts[128 * N];
    __shared__ double two_to[kPowers], sums[4 * N], warp_best[4];
    __shared__ uint32_t warp_at[4], warp_bad[4], hit, last;
    const uint32_t at = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const T* row = static_cast<const T*>(a.logits) + (int64_t)at * a.logits_stride;
    const RowRules k = row_rules(a.rules, at);
    const float temperature = a.temperature ? a.temperature[at] : a.temperature_value;
    const double uniform = a.uniforms ? a.uniforms[at] : 0.0;
    float logit[N], bias[N];
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t v = 128 * j + threadIdx.x;
        logit[j] = v < a.vocabulary ? load(row + v) : 0.0f;
        bias[j] = k.bias && v < a.vocabulary ? __ldg(k.bias + v) : 0.0f;
    }
    if (threadIdx.x < kPowers) two_to[threadIdx.x] = kTwoTo[threadIdx.x];
    if (threadIdx.x == 0) hit = kAll, last = 0;
    if (k.length)
        count_history(k, 0, 128 * N, counts);
    else
        __syncthreads();
    const bool greedy = temperature == 0.0f;
    const double heat = greedy ? 1.0 : (double)temperature, cold = cold_of(heat);
    const double reciprocal = 1.0 / (double)k.repetition;
    double z[N], best_value = -CUDART_INF;
    uint32_t best = kAll, bad = !(temperature >= 0.0f);
#pragma unroll
    for (int j = 0; j < N; ++j) {
        const uint32_t v = 128 * j + threadIdx.x;
        z[j] = adjusted((double)logit[j], k.length ? counts[v] : 0u, k, reciprocal, bias[j],
                        v < a.vocabulary && k.mask.allows(v));
        bad |= z[j] != z[j];
        if (z[j] > best_value) best_value = z[j], best = v;
    }
    const auto join_best = [&](uint32_t width) {
#pragma unroll 1
        for (uint32_t off = width / 2; off > 0; off >>= 1) {
            const double v = __shfl_xor_sync(kAll, best_value, off);
            const uint32_t b = __shfl_xor_sync(kAll, best, off);
            if (v > best_value || (v == best_value && b < best)) best_value = v, best = b;
            bad |= __shfl_xor_sync(kAll, bad, off);
        }
    };
    join_best(32);
    if (lane == 0) warp_best[warp] = best_value, warp_at[warp] = best, warp_bad[warp] = bad;
    __syncthreads();
    best_value = warp_best[lane & 3u], best = warp_at[lane & 3u], bad = warp_bad[lane & 3u];
    join_best(4);
    if (bad || best == kAll) {
        if (threadIdx.x == 0) {
            a.symbols[at] = -1;
            if (a.log_probability) a.log_probability[at] = bad ? CUDART_NAN_F : -CUDART_INF_F;
        }
        return;
    }
    // Running sums in the order of the symbols: of a warp's 32 here, of the warps' sums below.
    double w[N], through[N];
#pragma unroll
    for (int j = 0; j < N; ++j) through[j] = w[j] = weight_of(z[j], best_value, cold, two_to);
#pragma unroll 1
    for (int off = 1; off < 32; off <<= 1) {
#pragma unroll
        for (int j = 0; j < N; ++j) {
            const double o = __shfl_up_sync(kAll, through[j], off);
            if (lane >= (uint32_t)off) through[j] += o;
        }
    }
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (lane == 31) sums[4 * j + warp] = through[j];
    __syncthreads();
    double total = 0.0, before[N];
#pragma unroll
    for (int j = 0; j < 4 * N; ++j) {
        if ((j & 3) == (int)warp) before[j / 4] = total;
        total += sums[j];
    }
    if (greedy) {
        if (threadIdx.x == 0) {
            a.symbols[at] = (int32_t)best;
            if (a.log_probability) a.log_probability[at] = (float)-log(total);
        }
        return;
    }
    const double goal = uniform * total;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (w[j] > 0.0) {
            const uint32_t v = 128 * j + threadIdx.x;
            if (before[j] + through[j] > goal)
                atomicMin(&hit, v);
            else
                atomicMax(&last, v);
        }
    __syncthreads();
    // A uniform of nearly 1 may pass no sum, which were rounded.
    const uint32_t symbol = hit != kAll ? hit : last;
    if (threadIdx.x == (symbol & 127u)) {
        double chosen = 0.0;
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (symbol / 128 == j) chosen = z[j];
        a.symbols[at] = (int32_t)symbol;
        if (a.log_probability)
            a.log_probability[at] = (float)((chosen == best_value ? 0.0 : (chosen - best_value) / heat) - log(total));
    }
}

struct LossArgs {
    const void* logits;
    int64_t logits_stride;
    uint32_t rows, vocabulary;
    const int32_t* targets;
    const uint32_t* allowed;
    int64_t allowed_stride;
    uint32_t states;
    const int32_t* state;
    const float* weights;
    float* losses;
    void* gradient;
    int64_t gradient_stride;
};

__device__ __forceinline__ float exp2_of(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Weights by a row's largest logit as 2^(z c - top c), one multiply-add and one
// exponential each.  top c is rounded once for the whole row, which scales all
// weights alike: out of their ratios it falls, and the loss takes it out.  A
// masked place's -inf gives 0.  Beside logits so large that neighbours are
// 2^100 apart only equals count, which a c of 2^-20 gives without overflow.
struct RowScale {
    float top, c, shift, off;  // weights are 2^off times too large
    __device__ __forceinline__ explicit RowScale(float top_) : top(top_) {
        c = fabsf(top) <= 0x1p30f ? 1.44269504f : 1.0f;
        shift = top == -CUDART_INF_F ? 0.0f : top * c;
        off = top == -CUDART_INF_F ? 0.0f : fmaf(top, c, -shift);
    }
    __device__ __forceinline__ float weight(float z) const { return exp2_of(fmaf(z, c, -shift)); }
    __device__ __forceinline__ Pair32 weight(Pair32 z) const {
        const float2 x = parts(fma2(z, pair_of(c, c), pair_of(-shift, -shift)));
        return pair_of(exp2_of(x.x), exp2_of(x.y));
    }
    // What makes weights by `part`, of some of the row's symbols, weights by this one.  Where
    // the two differ in c they are so far apart that nothing of the part is left.
    __device__ __forceinline__ float of(const RowScale& part) const {
        return part.top == -CUDART_INF_F || part.c != c ? 0.0f : part.top == top ? 1.0f : exp2_of(part.shift - shift);
    }
    // Loss of a row with the sum of its weights and the (masked) logit of its target.
    __device__ __forceinline__ float loss(float sum, float z) const {
        if (sum != sum) return sum;
        if (sum == 0.0f || z == -CUDART_INF_F) return CUDART_INF_F;
        // The whole part of `off` comes out of the sum exactly.
        const float whole = rintf(off);
        return fmaf(off - whole, -0.693147181f, logf(sum * __int_as_float((127 - (int)whole) << 23))) + (top - z);
    }
};

// Rows of up to 32 N symbols, a warp each: symbol 32 j + lane is in register j,
// so the mask's word j is the warp's, and the logits are read once.  Full: all
// registers but the last are, which spares their tests.  81,984 rows of 257
// float32 take 37 us, 39 us with the tests (26 us at a copy's rate); the issue slots
// are three quarters full.
template <typename T, int N, bool Full>
__global__ void __launch_bounds__(256) narrow_loss_kernel(const __grid_constant__ LossArgs a) {
    const uint32_t lane = threadIdx.x & 31u;
    const uint64_t at = (uint64_t)blockIdx.x * 8 + (threadIdx.x >> 5);
    if (at >= a.rows) return;
    const uint32_t row = (uint32_t)at;
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride + lane;
    T* out = static_cast<T*>(a.gradient) + (int64_t)row * a.gradient_stride + lane;
    const uint32_t symbols = (a.vocabulary + 31 - lane) / 32;  // of the lane
    const auto mine = [&](int j) { return Full && j < N - 1 ? true : j < (int)symbols; };
    float z[N];
#pragma unroll
    for (int j = 0; j < N; ++j) z[j] = mine(j) ? load(in + 32 * j) : -CUDART_INF_F;
    const int32_t target = a.targets[row];
    const MaskRow mask = mask_row(a.allowed, a.allowed_stride, a.states, a.state, row);
    const bool outside = target >= 0 && (uint32_t)target >= a.vocabulary;
    if (target < 0 || outside) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (mine(j)) store(out + 32 * j, 0.0f);
        if (lane == 0) a.losses[row] = outside ? CUDART_NAN_F : 0.0f;
        return;
    }
    const bool counts = mask.allows((uint32_t)target);
    const float hit = counts ? load(in - lane + target) : -CUDART_INF_F;
    const uint32_t bit = 1u << lane;
    if (mask.words) {
#pragma unroll
        for (int j = 0; j < N; ++j)
            if (mine(j) && !(__ldg(mask.words + j) & bit)) z[j] = -CUDART_INF_F;
    } else if (!mask.open) {
#pragma unroll
        for (int j = 0; j < N; ++j) z[j] = -CUDART_INF_F;
    }
    float top = z[0];
#pragma unroll
    for (int j = 1; j < N; ++j) top = fmaxf(top, z[j]);
    const RowScale by(warp_max(top));
    float w[N], sum = 0.0f;
#pragma unroll
    for (int j = 0; j < N; ++j) {
        w[j] = by.weight(z[j]);
        sum += w[j];
    }
    sum = warp_sum(sum);
    const float scale = a.weights ? a.weights[row] : 1.0f, gain = sum == 0.0f ? 0.0f : scale / sum;
#pragma unroll
    for (int j = 0; j < N; ++j)
        if (mine(j)) store(out + 32 * j, w[j] * gain);
    // The target's term, in place of what this lane has written there.
    if (lane == ((uint32_t)target & 31u)) {
        if (counts && sum != 0.0f) store(out + (target & ~31), fmaf(by.weight(hit), gain, -scale));
        a.losses[row] = by.loss(sum, hit);
    }
}

// Wider rows, a block each, in three sweeps: the largest logit, the sum of the
// weights, the gradient.  The first two are a warp's own, by its own largest
// logit, so that the warps meet once.  A row that fits is copied into shared memory first,
// each thread the groups that it will sweep, so that it comes from memory once
// and three blocks an SM overlap their copies with the others' sweeps.  2,048 x 32,001
// bfloat16: 63 us (40 us at a copy's rate; two exponentials a symbol fill three quarters
// of the issue slots with what goes with them), 87 us with the row in registers and two
// blocks.  A larger row is read in every sweep, in part out of L2: 400 x 131,072 float32
// come from memory 2.2 times, and 1,024 of them take 377 us (165 us at a copy's rate).
// The float32 form of 512 threads spills 28 bytes a thread at its 40 registers.
template <typename T, int Threads, bool Held>
__global__ void __launch_bounds__(Threads, Held ? 3 : 2) wide_loss_kernel(const __grid_constant__ LossArgs a) {
    extern __shared__ __align__(16) unsigned char dynamic[];
    __shared__ float shared[2][32];
    const uint32_t at = blockIdx.x;
    const Row<T> row(static_cast<const T*>(a.logits) + (int64_t)at * a.logits_stride, a.vocabulary);
    T* out = static_cast<T*>(a.gradient) + (int64_t)at * a.gradient_stride;
    const bool aligned = row.alike(out);
    const auto symbol_of = [&](uint32_t g) { return row.first + (int32_t)g * 8; };
    Eight<T>* held = reinterpret_cast<Eight<T>*>(dynamic);
    if constexpr (Held) {
        for (uint32_t g = threadIdx.x; g < row.groups; g += Threads) {
            const int32_t v = symbol_of(g);
            if (row.whole(v)) {
                const uint32_t to = (uint32_t)__cvta_generic_to_shared(held + g);
#pragma unroll
                for (int i = 0; i < (int)sizeof(T) / 2; ++i)
                    asm volatile("cp.async.cg.shared.global [%0], [%1], 16;" ::"r"(to + 16 * i),
                                 "l"(reinterpret_cast<const uint4*>(row.p + v) + i)
                                 : "memory");
            } else {
                held[g] = row.read(v);
            }
        }
        asm volatile("cp.async.commit_group;" ::: "memory");
    }
    const int32_t target = a.targets[at];
    const MaskRow mask = mask_row(a.allowed, a.allowed_stride, a.states, a.state, at);
    const float scale = a.weights ? a.weights[at] : 1.0f;
    const bool outside = target >= 0 && (uint32_t)target >= a.vocabulary;
    if constexpr (Held) asm volatile("cp.async.wait_group 0;" ::: "memory");
    if (target < 0 || outside) {
        Eight<T> zero;
#pragma unroll
        for (int i = 0; i < 8; ++i) zero.set(i, 0.0f);
        for (uint32_t g = threadIdx.x; g < row.groups; g += Threads) row.write(out, aligned, symbol_of(g), zero);
        if (threadIdx.x == 0) a.losses[at] = outside ? CUDART_NAN_F : 0.0f;
        return;
    }
    // Bit i: symbol v + i counts.
    const auto counts_at = [&](int32_t v) {
        uint32_t ok = mask.eight(v, a.vocabulary);
        if (!row.whole(v))
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (!row.in(v + i)) ok &= ~(1u << i);
        return ok;
    };
    const auto each = [&](auto&& body) {
#pragma unroll 2
        for (uint32_t g = threadIdx.x; g < row.groups; g += Threads) {
            if constexpr (Held)
                body(held[g], symbol_of(g));
            else
                body(row.read(symbol_of(g)), symbol_of(g));
        }
    };
    float top = -CUDART_INF_F;
    each([&](const Eight<T>& e, int32_t v) {
        const uint32_t ok = counts_at(v);
        if (ok == 0xffu) {
            top = fmaxf(top, e.largest());
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (ok >> i & 1u) top = fmaxf(top, e[i]);
        }
    });
    const RowScale here(warp_max(top));  // this warp's
    Pair32 sums = 0;
    each([&](const Eight<T>& e, int32_t v) {
        const uint32_t ok = counts_at(v);
        if (ok == 0xffu) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sums = add2(sums, here.weight(e.pair(i)));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                if (ok >> i & 1u) sums = add2(sums, pair_of(here.weight(e[i]), 0.0f));
        }
    });
    const float2 halves = parts(sums);
    const float mine = warp_sum(halves.x + halves.y);
    if ((threadIdx.x & 31u) == 0) shared[0][threadIdx.x >> 5] = here.top, shared[1][threadIdx.x >> 5] = mine;
    __syncthreads();
    const bool warp_of = threadIdx.x % 32 < Threads / 32;
    const RowScale part(warp_of ? shared[0][threadIdx.x % 32] : -CUDART_INF_F), by(warp_max(part.top));
    const float sum = warp_sum(warp_of ? shared[1][threadIdx.x % 32] * by.of(part) : 0.0f);
    const float gain = sum == 0.0f ? 0.0f : scale / sum;
    each([&](const Eight<T>& e, int32_t v) {
        const uint32_t ok = counts_at(v);
        Eight<T> r;
        if (ok == 0xffu && (uint32_t)(target - v) >= 8u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) r.set_pair(i, mul2(by.weight(e.pair(i)), pair_of(gain, gain)));
        } else {
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const float g = fmaf(by.weight(e[i]), gain, v + i == target && sum != 0.0f ? -scale : 0.0f);
                r.set(i, ok >> i & 1u ? g : 0.0f);
            }
        }
        row.write(out, aligned, v, r);
    });
    if (threadIdx.x == 0)
        a.losses[at] = by.loss(sum, mask.allows((uint32_t)target) ? load(row.p + target) : -CUDART_INF_F);
}

template <typename Body>
void dispatch(int dtype, Body&& body) {
    switch (dtype) {
        case LEO_B200_F32: body((float*)nullptr); return;
        case LEO_B200_BF16: body((__nv_bfloat16*)nullptr); return;
        case LEO_B200_F16: body((__half*)nullptr); return;
        default: throw Failure("logits must be float32, bfloat16 or float16");
    }
}

// A block a row, or a cluster of up to eight while that leaves SMs without work.
template <typename T, int Warps>
void launch_pick(const LogitArgs& a, cudaStream_t stream) {
    const uint32_t all = (a.vocabulary + 7 + kStepSymbols - 1) / kStepSymbols;
    uint32_t blocks = 1;
    // two blocks on each of 148 SMs and no second wave: 64 rows of 131,072 take 59 us in 512 blocks, 54 us in 256
    while (blocks < 8 && blocks * 2 * Warps <= all && (uint64_t)a.rows * blocks * 2 <= 296) blocks *= 2;
    if (all > 2048) blocks = 8;
    const uint32_t steps = (all + blocks - 1) / blocks;
    require(steps <= 4096, "the vocabulary is too large for one pick");
    require((uint64_t)a.rows * blocks < (1ull << 31), "too many rows for one call");
    const auto kernel = pick_kernel<T, Warps>;
    const size_t shared = steps * sizeof(Weights) +
                          (a.rules.history ? std::min(steps, kPickWindow) * kStepSymbols * sizeof(uint32_t) : 0);
    static std::atomic<uint64_t> allowed{0};
    allow_shared(kernel, 4096 * sizeof(Weights) + kPickWindow * kStepSymbols * sizeof(uint32_t), allowed);
    cudaLaunchConfig_t config{};
    config.gridDim = dim3(a.rows * blocks);
    config.blockDim = dim3(32 * Warps);
    config.dynamicSmemBytes = shared;
    config.stream = stream;
    cudaLaunchAttribute cluster{};
    cluster.id = cudaLaunchAttributeClusterDimension;
    cluster.val.clusterDim.x = blocks;
    cluster.val.clusterDim.y = cluster.val.clusterDim.z = 1;
    config.attrs = &cluster;
    config.numAttrs = 1;
    check(cudaLaunchKernelEx(&config, kernel, a, steps), "pick_kernel");
}

// A warp a row while it holds the row in 32 registers a lane (rows of bytes and the
// end, the framework's own, in full ones), a block above.
template <typename T>
void launch_loss(const LossArgs& a, cudaStream_t stream) {
    const uint32_t v = a.vocabulary, warps = (a.rows + 7) / 8;
    if (v <= 256) narrow_loss_kernel<T, 8, false><<<warps, 256, 0, stream>>>(a);
    else if (v <= 288) narrow_loss_kernel<T, 9, true><<<warps, 256, 0, stream>>>(a);
    else if (v <= 512) narrow_loss_kernel<T, 16, false><<<warps, 256, 0, stream>>>(a);
    else if (v <= 1024) narrow_loss_kernel<T, 32, false><<<warps, 256, 0, stream>>>(a);
    else if (const size_t held = ((size_t)v + 14) / 8 * sizeof(Eight<T>); held <= 110 * 1024) {
        // three blocks an SM up to 75 KB a row, two up to 110 KB
        const bool small = v <= 8192;
        const auto kernel = small ? wide_loss_kernel<T, 256, true> : wide_loss_kernel<T, 512, true>;
        static std::atomic<uint64_t> allowed[2];
        allow_shared(kernel, 110 * 1024, allowed[small]);
        kernel<<<a.rows, small ? 256 : 512, held, stream>>>(a);
    } else {
        wide_loss_kernel<T, 512, false><<<a.rows, 512, 0, stream>>>(a);
    }
}

void check_mask(const uint32_t* allowed, int64_t stride, uint32_t states, const int32_t* state, uint32_t rows,
                uint32_t vocabulary) {
    if (!allowed) return;
    require(states > 0, "a mask needs at least one state");
    require(states == 1 || stride >= (int64_t)((vocabulary + 31) / 32), "mask rows overlap");
    require(state != nullptr || states == 1 || states == rows, "mask rows without states must be one, or one a row");
}

void check_rules(const LeoB200LogitRules* r, uint32_t rows, uint32_t vocabulary) {
    require(r != nullptr, "logit rules are null");
    check_mask(r->allowed, r->allowed_stride, r->states, r->state, rows, vocabulary);
    require(r->repetition != nullptr || (r->repetition_value > 0.0f && std::isfinite(r->repetition_value)),
            "the repetition penalty must be positive and finite");
    require(r->presence != nullptr || std::isfinite(r->presence_value), "the presence penalty must be finite");
    require(r->frequency != nullptr || std::isfinite(r->frequency_value), "the frequency penalty must be finite");
    require(r->history_capacity < (1u << 31), "the history is too long");
}

void check_rows(const void* logits, int64_t stride, uint32_t rows, uint32_t vocabulary) {
    require(vocabulary > 0, "the vocabulary must not be empty");
    require(vocabulary <= (1u << 30), "the vocabulary is too large");
    require(rows < (1u << 31), "too many rows for one call");
    require(rows == 0 || logits != nullptr, "logits are null");
    require(rows <= 1 || stride >= 0, "the row stride must not be negative");
}

}  // namespace

extern "C" {

int leo_b200_adjust_logits(int device, int dtype, const void* logits, int64_t logits_stride, uint32_t rows,
                           uint32_t vocabulary, const LeoB200LogitRules* rules, void* out, int64_t out_stride,
                           void* stream) {
    return guarded([&] {
        check_rows(logits, logits_stride, rows, vocabulary);
        check_rules(rules, rows, vocabulary);
        require(rows == 0 || out != nullptr, "the output is null");
        require(rows <= 1 || out_stride >= (int64_t)vocabulary, "output rows overlap");
        dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (rows == 0) return;
            LogitArgs a{};
            a.logits = logits;
            a.logits_stride = logits_stride;
            a.rows = rows;
            a.vocabulary = vocabulary;
            a.rules = *rules;
            a.out = out;
            a.out_stride = out_stride;
            DeviceScope scope(device);
            // A turn more than the symbols take, if a row can start off a 16-byte address.
            const uint32_t all = (vocabulary + 7 + kAdjustTurn - 1) / kAdjustTurn;
            const uint32_t turns = std::min(all, kAdjustRun / kAdjustTurn), runs = (all + turns - 1) / turns;
            require((uint64_t)rows * runs < (1ull << 31), "too many rows for one call");
            const size_t shared = rules->history ? turns * kAdjustTurn * sizeof(uint32_t) : 0;
            adjust_kernel<T><<<rows * runs, kAdjustThreads, shared, (cudaStream_t)stream>>>(a, runs, turns);
            check(cudaGetLastError(), "adjust_kernel");
        });
    });
}

int leo_b200_pick_symbols(int device, int dtype, const void* logits, int64_t logits_stride, uint32_t rows,
                          uint32_t vocabulary, const LeoB200LogitRules* rules, const float* temperature,
                          float temperature_value, const double* uniforms, int32_t* symbols, float* log_probability,
                          void* stream) {
    return guarded([&] {
        check_rows(logits, logits_stride, rows, vocabulary);
        check_rules(rules, rows, vocabulary);
        require(rows == 0 || symbols != nullptr, "the symbols are null");
        require(temperature != nullptr || temperature_value >= 0.0f, "the temperature must not be negative");
        require(uniforms != nullptr || rows == 0 || (temperature == nullptr && temperature_value == 0.0f),
                "drawing a symbol needs uniforms");
        dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (rows == 0) return;
            LogitArgs a{};
            a.logits = logits;
            a.logits_stride = logits_stride;
            a.rows = rows;
            a.vocabulary = vocabulary;
            a.rules = *rules;
            a.temperature = temperature;
            a.temperature_value = temperature_value;
            a.uniforms = uniforms;
            a.symbols = symbols;
            a.log_probability = log_probability;
            DeviceScope scope(device);
            if (vocabulary <= 384)
                narrow_pick_kernel<T, 3><<<rows, 128, 0, (cudaStream_t)stream>>>(a);
            else if (vocabulary <= 1024)
                narrow_pick_kernel<T, 8><<<rows, 128, 0, (cudaStream_t)stream>>>(a);
            else
                launch_pick<T, 8>(a, (cudaStream_t)stream);
            check(cudaGetLastError(), "pick_kernel");
        });
    });
}

int leo_b200_masked_cross_entropy(int device, int dtype, const void* logits, int64_t logits_stride, uint32_t rows,
                                  uint32_t vocabulary, const int32_t* targets, const uint32_t* allowed,
                                  int64_t allowed_stride, uint32_t states, const int32_t* state,
                                  const float* weights, float* losses, void* gradient, int64_t gradient_stride,
                                  void* stream) {
    return guarded([&] {
        check_rows(logits, logits_stride, rows, vocabulary);
        check_mask(allowed, allowed_stride, states, state, rows, vocabulary);
        require(rows == 0 || (targets && losses && gradient), "loss arrays are null");
        require(rows <= 1 || gradient_stride >= (int64_t)vocabulary, "gradient rows overlap");
        dispatch(dtype, [&](auto* t) {
            using T = std::remove_pointer_t<decltype(t)>;
            if (rows == 0) return;
            LossArgs a{logits, logits_stride, rows,    vocabulary, targets, allowed, allowed_stride,
                       states, state,         weights, losses,     gradient, gradient_stride};
            DeviceScope scope(device);
            launch_loss<T>(a, (cudaStream_t)stream);
            check(cudaGetLastError(), "cross_entropy_kernel");
        });
    });
}

}  // extern "C"
