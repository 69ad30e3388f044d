// Operators on rows of logits (include/leo_b200.h): penalties, biases and
// grammar masks; the pick of the next symbol; the cross entropy over the
// allowed symbols with its gradient.  One thread block takes one row.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <cmath>
#include <type_traits>

#include "../../include/leo_b200.h"
#include "leo_operator_host.h"

namespace {

using namespace leo_operator;

constexpr uint32_t kThreads = 256;
constexpr uint32_t kWarps = kThreads / 32;
constexpr uint32_t kChunk = 4096;  // symbols whose counts are held in shared memory at a time

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }

// What a row of the mask table says: all symbols, none, or its words.
struct MaskRow {
    const uint32_t* words;  // nullptr: see `open`
    bool open;
    __device__ __forceinline__ bool allows(uint32_t v) const {
        return words ? (words[v >> 5] >> (v & 31u)) & 1u : open;
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

// Counts of the history's symbols in [first, first + span).
__device__ void count_history(const RowRules& k, uint32_t first, uint32_t span, uint32_t* counts) {
    for (uint32_t i = threadIdx.x; i < span; i += kThreads) counts[i] = 0;
    __syncthreads();
    for (uint32_t i = threadIdx.x; i < k.length; i += kThreads) {
        const uint32_t v = (uint32_t)k.history[i] - first;
        if (v < span) atomicAdd(&counts[v], 1u);
    }
    __syncthreads();
}

// The penalties, the bias and the mask, every operation rounded by itself in F.
template <typename F>
__device__ __forceinline__ F adjusted(F z, uint32_t v, uint32_t count, const RowRules& k) {
    if (count) {
        z = z > (F)0 ? z / (F)k.repetition : z * (F)k.repetition;
        z -= (F)k.presence + (F)k.frequency * (F)count;
    }
    if (k.bias) z += (F)k.bias[v];
    return k.mask.allows(v) ? z : -(F)CUDART_INF;
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

template <typename T>
__global__ void __launch_bounds__(kThreads) adjust_kernel(LogitArgs a) {
    __shared__ uint32_t counts[kChunk];
    const uint32_t row = blockIdx.x;
    const RowRules k = row_rules(a.rules, row);
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride;
    T* out = static_cast<T*>(a.out) + (int64_t)row * a.out_stride;
    for (uint32_t first = 0; first < a.vocabulary; first += kChunk) {
        const uint32_t span = min(kChunk, a.vocabulary - first);
        count_history(k, first, span, counts);
        for (uint32_t i = threadIdx.x; i < span; i += kThreads)
            store(out + first + i, adjusted(load(in + first + i), first + i, counts[i], k));
        __syncthreads();
    }
}

// The larger of two (value, symbol) pairs, the lower symbol of equal values.
__device__ __forceinline__ void keep_best(double& v, uint32_t& at, double other, uint32_t other_at) {
    if (other > v || (other == v && other_at < at)) {
        v = other;
        at = other_at;
    }
}

template <typename T>
__global__ void __launch_bounds__(kThreads) pick_kernel(LogitArgs a) {
    __shared__ uint32_t counts[kChunk];
    __shared__ double warp_value[kWarps];
    __shared__ uint32_t warp_at[kWarps];
    __shared__ double running;
    __shared__ uint32_t found, last;
    __shared__ int bad;
    const uint32_t row = blockIdx.x, lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const RowRules k = row_rules(a.rules, row);
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride;
    const float temperature = a.temperature ? a.temperature[row] : a.temperature_value;
    if (threadIdx.x == 0) bad = !(temperature >= 0.0f);
    // pass 1: the largest adjusted logit
    double best = -CUDART_INF;
    uint32_t best_at = 0xffffffffu;
    for (uint32_t first = 0; first < a.vocabulary; first += kChunk) {
        const uint32_t span = min(kChunk, a.vocabulary - first);
        count_history(k, first, span, counts);
        for (uint32_t i = threadIdx.x; i < span; i += kThreads) {
            const double z = adjusted((double)load(in + first + i), first + i, counts[i], k);
            if (z != z) bad = 1;
            if (z > best) best = z, best_at = first + i;
        }
        __syncthreads();
    }
    for (int off = 16; off > 0; off >>= 1) {
        const double v = __shfl_xor_sync(0xffffffffu, best, off);
        const uint32_t at = __shfl_xor_sync(0xffffffffu, best_at, off);
        keep_best(best, best_at, v, at);
    }
    if (lane == 0) warp_value[warp] = best, warp_at[warp] = best_at;
    __syncthreads();
    for (uint32_t w = 0; w < kWarps; ++w) keep_best(best, best_at, warp_value[w], warp_at[w]);
    if (bad || best_at == 0xffffffffu) {
        if (threadIdx.x == 0) {
            a.symbols[row] = -1;
            if (a.log_probability) a.log_probability[row] = bad ? CUDART_NAN_F : -CUDART_INF_F;
        }
        return;
    }
    const bool greedy = temperature == 0.0f;
    const double heat = greedy ? 1.0 : (double)temperature;
    const auto weight = [&](double z) {
        return z == best ? 1.0 : z == -CUDART_INF ? 0.0 : exp((z - best) / heat);
    };
    // pass 2: the sum of the weights; pass 3: where the sums in symbol order pass u * total
    double total = 0.0, target = 0.0;
    for (int pass = 2; pass <= (greedy ? 2 : 3); ++pass) {
        __syncthreads();
        if (threadIdx.x == 0) running = 0.0, found = 0xffffffffu, last = 0;
        __syncthreads();
        for (uint32_t first = 0; first < a.vocabulary; first += kChunk) {
            const uint32_t span = min(kChunk, a.vocabulary - first);
            count_history(k, first, span, counts);
            for (uint32_t at = 0; at < span; at += kThreads) {
                const uint32_t i = at + threadIdx.x;
                const double w =
                    i < span ? weight(adjusted((double)load(in + first + i), first + i, counts[i], k)) : 0.0;
                double sum = w;
                for (int off = 1; off < 32; off <<= 1) {
                    const double v = __shfl_up_sync(0xffffffffu, sum, off);
                    if (lane >= (uint32_t)off) sum += v;
                }
                if (lane == 31) warp_value[warp] = sum;
                __syncthreads();
                double before = running;
                for (uint32_t j = 0; j < warp; ++j) before += warp_value[j];
                if (pass == 3 && w > 0.0) {
                    atomicMax(&last, first + i);
                    if (before + sum > target) atomicMin(&found, first + i);
                }
                __syncthreads();
                if (threadIdx.x == kThreads - 1) running = before + sum;
                __syncthreads();
            }
            __syncthreads();
        }
        if (pass == 2) {
            total = running;
            target = greedy ? 0.0 : a.uniforms[row] * total;
        }
    }
    const uint32_t symbol = greedy ? best_at : found != 0xffffffffu ? found : last;
    if (threadIdx.x == 0) a.symbols[row] = (int32_t)symbol;
    if (!a.log_probability) return;
    __syncthreads();
    const uint32_t first = symbol / kChunk * kChunk;
    count_history(k, first, min(kChunk, a.vocabulary - first), counts);
    if (threadIdx.x == 0) {
        const double z = adjusted((double)load(in + symbol), symbol, counts[symbol - first], k);
        a.log_probability[row] = (float)((z == best ? 0.0 : (z - best) / heat) - log(total));
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

__device__ float block_reduce(float v, bool maximum, float* shared) {
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    for (int off = 16; off > 0; off >>= 1) {
        const float o = __shfl_xor_sync(0xffffffffu, v, off);
        v = maximum ? fmaxf(v, o) : v + o;
    }
    __syncthreads();
    if (lane == 0) shared[warp] = v;
    __syncthreads();
    v = shared[0];
    for (uint32_t w = 1; w < kWarps; ++w) v = maximum ? fmaxf(v, shared[w]) : v + shared[w];
    return v;
}

template <typename T>
__global__ void __launch_bounds__(kThreads) cross_entropy_kernel(LossArgs a) {
    __shared__ float shared[kWarps];
    const uint32_t row = blockIdx.x;
    const T* in = static_cast<const T*>(a.logits) + (int64_t)row * a.logits_stride;
    T* out = static_cast<T*>(a.gradient) + (int64_t)row * a.gradient_stride;
    const int32_t target = a.targets[row];
    const MaskRow mask = mask_row(a.allowed, a.allowed_stride, a.states, a.state, row);
    const bool outside = target >= 0 && (uint32_t)target >= a.vocabulary;
    if (target < 0 || outside) {
        for (uint32_t v = threadIdx.x; v < a.vocabulary; v += kThreads) store(out + v, 0.0f);
        if (threadIdx.x == 0) a.losses[row] = outside ? CUDART_NAN_F : 0.0f;
        return;
    }
    float top = -CUDART_INF_F;
    for (uint32_t v = threadIdx.x; v < a.vocabulary; v += kThreads)
        if (mask.allows(v)) top = fmaxf(top, load(in + v));
    top = block_reduce(top, true, shared);
    float sum = 0.0f;
    // Nothing left, or only NaN: top stays -inf.  exp(NaN - top) keeps a NaN in the sum.
    for (uint32_t v = threadIdx.x; v < a.vocabulary; v += kThreads)
        if (mask.allows(v)) {
            const float z = load(in + v);
            sum += z == -CUDART_INF_F ? 0.0f : expf(z - top);
        }
    sum = block_reduce(sum, false, shared);
    const float weight = a.weights ? a.weights[row] : 1.0f;
    for (uint32_t v = threadIdx.x; v < a.vocabulary; v += kThreads) {
        float g = 0.0f;
        if (sum != 0.0f && mask.allows(v)) {
            const float z = load(in + v);
            g = (z == -CUDART_INF_F ? 0.0f : expf(z - top)) / sum;
            g = weight * (g - (v == (uint32_t)target ? 1.0f : 0.0f));
        }
        store(out + v, g);
    }
    if (threadIdx.x == 0) {
        const float z = mask.allows((uint32_t)target) ? load(in + target) : -CUDART_INF_F;
        a.losses[row] = sum == 0.0f || z == -CUDART_INF_F ? (sum != sum ? sum : CUDART_INF_F) : logf(sum) + (top - z);
    }
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
    require(vocabulary > 0 && vocabulary < (1u << 31), "the vocabulary must not be empty");
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
            adjust_kernel<T><<<rows, kThreads, 0, (cudaStream_t)stream>>>(a);
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
            pick_kernel<T><<<rows, kThreads, 0, (cudaStream_t)stream>>>(a);
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
            cross_entropy_kernel<T><<<rows, kThreads, 0, (cudaStream_t)stream>>>(a);
            check(cudaGetLastError(), "cross_entropy_kernel");
        });
    });
}

}  // extern "C"
