// The gated linear recurrence over packed stories, its backward pass and its
// one-token step (include/leo_b200.h).
//
//   h[t] = a[t] h[t-1] + x[t]
//   slope[t] = g[t] + a[t+1] slope[t+1];  dx = slope, da[t] = slope[t] h[t-1]
//
// One thread carries one channel of one story.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <stdint.h>

#include <algorithm>
#include <type_traits>

#include "../../include/leo_b200.h"
#include "leo_operator_host.h"

namespace {

using namespace leo_operator;

__device__ __forceinline__ float load(const float* p) { return *p; }
__device__ __forceinline__ float load(const __nv_bfloat16* p) { return __bfloat162float(*p); }
__device__ __forceinline__ float load(const __half* p) { return __half2float(*p); }
__device__ __forceinline__ void store(float* p, float v) { *p = v; }
__device__ __forceinline__ void store(__nv_bfloat16* p, float v) { *p = __float2bfloat16_rn(v); }
__device__ __forceinline__ void store(__half* p, float v) { *p = __float2half_rn(v); }

constexpr uint32_t kThreads = 128;

struct ScanArgs {
    LeoB200StoryTables tables;
    uint32_t channels;
    const void* drive;
    int64_t drive_stride;
    const void* decay;
    int64_t decay_stride;  // 0: one row for all tokens
    const float* initial;
    void* states;
    float* final_states;
    float* carries;
    // backward
    const void* grad_states;
    int64_t grad_states_stride;
    const float* grad_final;
    void* grad_drive;
    void* grad_decay;
    float* grad_initial;
    int decay_shared;
};

// The tokens of the story at place `at` of the order.
__device__ __forceinline__ void story_span(const LeoB200StoryTables& t, uint32_t at, uint32_t& begin, uint32_t& end) {
    // The word that holds the story's start: the last one with rank <= at.
    const uint32_t words = (t.tokens + 31) / 32;
    uint32_t lo = 0, hi = words;
    while (hi - lo > 1) {
        const uint32_t mid = (lo + hi) >> 1;
        if (t.words[mid].rank <= at)
            lo = mid;
        else
            hi = mid;
    }
    uint32_t bits = t.words[lo].starts;
    for (uint32_t skip = at - t.words[lo].rank; skip > 0; --skip) bits &= bits - 1;
    begin = lo * 32 + __ffs(bits) - 1;
    bits &= bits - 1;
    end = bits ? lo * 32 + __ffs(bits) - 1 : t.words[lo].end;
}

template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) scan_forward_kernel(ScanArgs a) {
    const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t at = blockIdx.y;
    if (c >= a.channels) return;
    const uint32_t story = a.tables.order[at];
    float h = a.initial ? a.initial[(size_t)story * a.channels + c] : 0.0f;
    if (at < a.tables.full) {
        uint32_t begin, end;
        story_span(a.tables, at, begin, end);
        const T* x = static_cast<const T*>(a.drive) + (int64_t)begin * a.drive_stride + c;
        const G* gate = static_cast<const G*>(a.decay) + (int64_t)begin * a.decay_stride + c;
        for (uint32_t t = begin; t < end; ++t, x += a.drive_stride, gate += a.decay_stride) {
            if (a.carries) a.carries[(size_t)t * a.channels + c] = h;
            h = fmaf(load(gate), h, load(x));
            store(static_cast<T*>(a.states) + (size_t)t * a.channels + c, h);
        }
    }
    a.final_states[(size_t)story * a.channels + c] = h;
}

template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) scan_backward_kernel(ScanArgs a) {
    const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
    const uint32_t at = blockIdx.y;
    if (c >= a.channels) return;
    const uint32_t story = a.tables.order[at];
    const size_t end_at = (size_t)story * a.channels + c;
    float m = a.grad_final ? a.grad_final[end_at] : 0.0f;  // decay[t + 1] * slope[t + 1]
    if (at < a.tables.full) {
        uint32_t begin, end;
        story_span(a.tables, at, begin, end);
        for (uint32_t t = end; t-- > begin;) {
            const float gate = load(static_cast<const G*>(a.decay) + (int64_t)t * a.decay_stride + c);
            const float g = load(static_cast<const T*>(a.grad_states) + (int64_t)t * a.grad_states_stride + c);
            const float slope = g + m;
            const size_t i = (size_t)t * a.channels + c;
            store(static_cast<T*>(a.grad_drive) + i, slope);
            if (!a.decay_shared) store(static_cast<G*>(a.grad_decay) + i, slope * a.carries[i]);
            m = gate * slope;
        }
    }
    if (a.grad_initial) a.grad_initial[end_at] = m;
}

// The gradient of one row of gates: the terms of every token in token order.
template <typename T, typename G>
__global__ void __launch_bounds__(kThreads) shared_decay_kernel(ScanArgs a) {
    const uint32_t c = blockIdx.x * kThreads + threadIdx.x;
    if (c >= a.channels) return;
    const float gate = load(static_cast<const G*>(a.decay) + c);
    double sum = 0.0;
    for (uint32_t at = a.tables.full; at-- > 0;) {
        uint32_t begin, end;
        story_span(a.tables, at, begin, end);
        float m = a.grad_final ? a.grad_final[(size_t)a.tables.order[at] * a.channels + c] : 0.0f;
        for (uint32_t t = end; t-- > begin;) {
            const float slope = load(static_cast<const T*>(a.grad_states) + (int64_t)t * a.grad_states_stride + c) + m;
            sum += (double)(slope * a.carries[(size_t)t * a.channels + c]);
            m = gate * slope;
        }
    }
    store(static_cast<G*>(a.grad_decay) + c, (float)sum);
}

template <typename T, typename G>
__global__ void __launch_bounds__(kThreads)
    step_kernel(uint32_t channels, const T* drive, int64_t drive_stride, const G* decay, int64_t decay_stride,
                float* state, int64_t state_stride, T* output) {
    const uint32_t c = blockIdx.y * kThreads + threadIdx.x;
    const uint32_t lane = blockIdx.x;
    if (c >= channels) return;
    float* h = state + (int64_t)lane * state_stride + c;
    const float v = fmaf(load(decay + (int64_t)lane * decay_stride + c), *h, load(drive + (int64_t)lane * drive_stride + c));
    *h = v;
    store(output + (size_t)lane * channels + c, v);
}

// Calls body(T*, G*) with null pointers of the drive's and the gates' types.
template <typename Body>
void dispatch(int dtype, int decay_dtype, Body&& body) {
    const bool same = dtype == decay_dtype;
    require(same || decay_dtype == LEO_B200_F32, "decay must be of the drive's type or float32");
    switch (dtype) {
        case LEO_B200_F32: body((float*)nullptr, (float*)nullptr); return;
        case LEO_B200_BF16:
            if (same) body((__nv_bfloat16*)nullptr, (__nv_bfloat16*)nullptr);
            else body((__nv_bfloat16*)nullptr, (float*)nullptr);
            return;
        case LEO_B200_F16:
            if (same) body((__half*)nullptr, (__half*)nullptr);
            else body((__half*)nullptr, (float*)nullptr);
            return;
        default: throw Failure("drive must be float32, bfloat16 or float16");
    }
}

void check_tables(const LeoB200StoryTables* t, uint32_t channels) {
    require(t != nullptr, "story tables are null");
    require(t->stories > 0, "a batch needs at least one story");
    require(t->stories <= 65535, "too many stories for one scan");
    require(t->tokens < (1u << 31), "too many tokens for one scan");
    require(t->full <= t->stories && (t->full > 0) == (t->tokens > 0), "story tables are inconsistent");
    require(t->order != nullptr && (t->tokens == 0 || t->words != nullptr), "story tables are null");
    require(channels > 0 && channels < (1u << 31), "channels must be positive");
}

dim3 grid_of(const LeoB200StoryTables& t, uint32_t channels) {
    return dim3((channels + kThreads - 1) / kThreads, t.stories);
}

}  // namespace

extern "C" {

int leo_b200_story_table(const uint64_t* offsets, uint32_t stories, LeoB200StoryWord* words, uint32_t* order,
                         uint32_t* full) {
    return guarded([&] {
        require(offsets != nullptr && order != nullptr && full != nullptr, "story table arrays are null");
        require(stories > 0, "a batch needs at least one story");
        require(offsets[0] == 0, "story offsets must start at 0");
        for (uint32_t s = 0; s < stories; ++s)
            require(offsets[s + 1] >= offsets[s], "story offsets must be non-decreasing");
        require(offsets[stories] < (1ull << 31), "too many tokens for one batch");
        const uint32_t tokens = (uint32_t)offsets[stories];
        require(tokens == 0 || words != nullptr, "story table arrays are null");
        uint32_t n = 0;
        for (uint32_t s = 0; s < stories; ++s)
            if (offsets[s + 1] > offsets[s]) order[n++] = s;
        *full = n;
        for (uint32_t s = 0, e = n; s < stories; ++s)
            if (offsets[s + 1] == offsets[s]) order[e++] = s;
        uint32_t next = 0;  // the next story of the order that has not started
        for (uint64_t first = 0, w = 0; first < tokens; first += LEO_B200_STORY_WORD_TOKENS, ++w) {
            LeoB200StoryWord& word = words[w];
            const uint64_t past = std::min<uint64_t>(first + LEO_B200_STORY_WORD_TOKENS, tokens);
            word.starts = 0;
            word.rank = next;
            while (next < n && offsets[order[next]] < past) {
                word.starts |= 1u << (offsets[order[next]] - first);
                ++next;
            }
            const uint32_t holder = (word.starts & 1u) ? word.rank : word.rank - 1;
            word.begin = (uint32_t)offsets[order[holder]];
            word.end = (uint32_t)offsets[order[next - 1] + 1];
        }
    });
}

size_t leo_b200_gated_scan_workspace(uint32_t, uint32_t) { return 0; }

size_t leo_b200_gated_scan_carry_count(uint32_t tokens, uint32_t channels) { return (size_t)tokens * channels; }

int leo_b200_gated_scan(int device, const LeoB200StoryTables* tables, uint32_t channels, int dtype,
                        const void* drive, int64_t drive_stride, int decay_dtype, const void* decay,
                        int64_t decay_stride, int decay_shared, const float* initial, void* states,
                        float* final_states, float* carries, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_tables(tables, channels);
        require(tables->tokens == 0 || (drive && decay && states), "scan arrays are null");
        require(final_states != nullptr, "final states are null");
        (void)workspace;
        (void)workspace_bytes;
        ScanArgs a{};
        a.tables = *tables;
        a.channels = channels;
        a.drive = drive;
        a.drive_stride = drive_stride;
        a.decay = decay;
        a.decay_stride = decay_shared ? 0 : decay_stride;
        a.initial = initial;
        a.states = states;
        a.final_states = final_states;
        a.carries = carries;
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            DeviceScope scope(device);
            scan_forward_kernel<T, G><<<grid_of(*tables, channels), kThreads, 0, (cudaStream_t)stream>>>(a);
            check(cudaGetLastError(), "scan_forward_kernel");
        });
    });
}

int leo_b200_gated_scan_backward(int device, const LeoB200StoryTables* tables, uint32_t channels, int dtype,
                                 const void* grad_states, int64_t grad_states_stride, const void* drive,
                                 int64_t drive_stride, int decay_dtype, const void* decay, int64_t decay_stride,
                                 int decay_shared, const float* initial, const float* grad_final,
                                 const float* carries, void* grad_drive, void* grad_decay, float* grad_initial,
                                 void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_tables(tables, channels);
        require(tables->tokens == 0 || (grad_states && drive && decay && carries && grad_drive),
                "scan arrays are null");
        require(grad_decay != nullptr || (tables->tokens == 0 && !decay_shared), "scan arrays are null");
        (void)workspace;
        (void)workspace_bytes;
        ScanArgs a{};
        a.tables = *tables;
        a.channels = channels;
        a.drive = drive;
        a.drive_stride = drive_stride;
        a.decay = decay;
        a.decay_stride = decay_shared ? 0 : decay_stride;
        a.decay_shared = decay_shared;
        a.initial = initial;
        a.grad_states = grad_states;
        a.grad_states_stride = grad_states_stride;
        a.grad_final = grad_final;
        a.carries = const_cast<float*>(carries);
        a.grad_drive = grad_drive;
        a.grad_decay = grad_decay;
        a.grad_initial = grad_initial;
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            DeviceScope scope(device);
            const dim3 grid = grid_of(*tables, channels);
            scan_backward_kernel<T, G><<<grid, kThreads, 0, (cudaStream_t)stream>>>(a);
            check(cudaGetLastError(), "scan_backward_kernel");
            if (decay_shared) {
                shared_decay_kernel<T, G><<<grid.x, kThreads, 0, (cudaStream_t)stream>>>(a);
                check(cudaGetLastError(), "shared_decay_kernel");
            }
        });
    });
}

int leo_b200_gated_scan_status(int device, uint32_t* gave_up) {
    return guarded([&] {
        require(gave_up != nullptr, "status is null");
        (void)device;
        *gave_up = 0;
    });
}

int leo_b200_gated_step(int device, uint32_t lanes, uint32_t channels, int dtype, const void* drive,
                        int64_t drive_stride, int decay_dtype, const void* decay, int64_t decay_stride,
                        int decay_shared, float* state, int64_t state_stride, void* output, void* stream) {
    return guarded([&] {
        require(lanes < (1u << 31), "too many lanes for one step");
        require(channels > 0, "channels must be positive");
        require(channels <= 65535u * kThreads, "too many channels for one step");
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            if (lanes == 0) return;
            require(drive && decay && state && output, "step arrays are null");
            DeviceScope scope(device);
            step_kernel<T, G><<<dim3(lanes, (channels + kThreads - 1) / kThreads), kThreads, 0, (cudaStream_t)stream>>>(
                channels, static_cast<const T*>(drive), drive_stride, static_cast<const G*>(decay),
                decay_shared ? 0 : decay_stride, state, state_stride, static_cast<T*>(output));
            check(cudaGetLastError(), "step_kernel");
        });
    });
}

}  // extern "C"
