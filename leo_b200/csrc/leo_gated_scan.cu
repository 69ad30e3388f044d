// The gated linear recurrence over packed stories, its backward pass and its
// one-token step (include/leo_b200.h).
//
//   h[t] = a[t] h[t-1] + x[t]
//   slope[t] = g[t] + a[t+1] slope[t+1];  dx = slope, da[t] = slope[t] h[t-1]
//
// Tiles.  The packed batch is cut into tiles of 128 tokens whatever its
// stories are, so a ragged batch balances by itself; a block of 8 warps takes a
// tile of 32 V channels, each thread 16 tokens in a row of V channels, which it
// reads once into registers.  A span of tokens maps the state before it to the
// state after it as h -> A h + H (A the product of the gates, H the state from
// zero), or as h -> H if a story starts inside, and such maps compose: the
// threads' maps give the tile's, the tiles' maps give the state before a tile,
// and each thread then runs its 16 tokens again from registers and writes them.
// The backward pass is the same from the right, with m -> A m + M for
// m[t] = a[t] slope[t]; h is formed anew from the tile's carry.
//
// The state before a tile comes from the tiles before it in the same launch:
// tiles are dealt by a ticket in token order, so a block only ever waits for
// blocks that have started.  Each publishes its map; every kGroup-th tile
// publishes the state after it instead, so that a tile reads at most kGroup
// slots.  Which slots are read, and in which order they are composed, depends
// on the layout alone: results are the same in every run.
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
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

constexpr uint32_t kThreads = 128;  // of the step and the reduction

constexpr int kSegment = 16;                      // tokens of a thread
constexpr int kTileWarps = 8;
constexpr uint32_t kTile = kSegment * kTileWarps;  // tokens of a block
constexpr uint32_t kTileThreads = 32 * kTileWarps;
constexpr uint32_t kGroup = 16;                    // tiles between published states
constexpr uint32_t kSpinLimit = 1u << 21;          // polls of a wait, 32 ns and a memory round trip apart
static_assert(kTile % LEO_B200_STORY_WORD_TOKENS == 0 && LEO_B200_STORY_WORD_TOKENS % kSegment == 0, "story words");

__device__ uint32_t g_gave_up;

// V elements of a row as they lie in memory, read or written once.
template <typename T, int V> struct Packed;
template <> struct Packed<float, 1> {
    using Raw = float;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = r; }
    static __device__ __forceinline__ Raw pack(const float (&v)[1]) { return v[0]; }
};
template <> struct Packed<float, 2> {
    using Raw = float2;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2]) { v[0] = r.x, v[1] = r.y; }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) { return make_float2(v[0], v[1]); }
};
template <> struct Packed<__nv_bfloat16, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = __uint_as_float((uint32_t)r << 16); }
    static __device__ __forceinline__ Raw pack(const float (&v)[1]) {
        return __bfloat16_as_ushort(__float2bfloat16_rn(v[0]));
    }
};
template <> struct Packed<__nv_bfloat16, 2> {
    using Raw = unsigned int;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2]) {
        v[0] = __uint_as_float(r << 16), v[1] = __uint_as_float(r & 0xffff0000u);
    }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) {
        return (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[0])) |
               (uint32_t)__bfloat16_as_ushort(__float2bfloat16_rn(v[1])) << 16;
    }
};
template <> struct Packed<__half, 1> {
    using Raw = unsigned short;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[1]) { v[0] = __half2float(__ushort_as_half(r)); }
    static __device__ __forceinline__ Raw pack(const float (&v)[1]) { return __half_as_ushort(__float2half_rn(v[0])); }
};
template <> struct Packed<__half, 2> {
    using Raw = unsigned int;
    static __device__ __forceinline__ void unpack(Raw r, float (&v)[2]) {
        v[0] = __half2float(__ushort_as_half((unsigned short)r));
        v[1] = __half2float(__ushort_as_half((unsigned short)(r >> 16)));
    }
    static __device__ __forceinline__ Raw pack(const float (&v)[2]) {
        return (uint32_t)__half_as_ushort(__float2half_rn(v[0])) |
               (uint32_t)__half_as_ushort(__float2half_rn(v[1])) << 16;
    }
};

template <typename T, int V>
__device__ __forceinline__ typename Packed<T, V>::Raw read_once(const T* p) {
    return __ldcs(reinterpret_cast<const typename Packed<T, V>::Raw*>(p));
}
template <typename T, int V>
__device__ __forceinline__ void write_once(T* p, const float (&v)[V]) {
    __stcs(reinterpret_cast<typename Packed<T, V>::Raw*>(p), Packed<T, V>::pack(v));
}

// The scratch of one call: the ticket, a flag for every 32 channels of a tile,
// a slot for every channel of a tile, and the partial sums of a shared gate's
// gradient.  Ticket and flags are zeroed before the launch.
struct Scratch {
    uint32_t* ticket;
    uint32_t* flags;   // [tiles][flag_row]
    double2* slots;    // [tiles][channels]: (A, H), or (-, state)
    float* partials;   // [tiles][channels]
    uint32_t flag_row;
};

struct ScanArgs {
    LeoB200StoryTables tables;
    uint32_t channels, tiles, groups;  // groups: of 32 V channels
    const void* drive;
    int64_t drive_stride;
    const void* decay;
    int64_t decay_stride;
    const float* initial;
    void* states;
    float* final_states;
    float* carries;  // [tiles][channels]: the state before each tile
    // backward
    const void* grad_states;
    int64_t grad_states_stride;
    const float* grad_final;
    void* grad_drive;
    void* grad_decay;
    float* grad_initial;
    Scratch scratch;
};

// A thread's 16 tokens among the stories.
struct Segment {
    uint32_t first;    // token
    int count;         // tokens before the batch's end
    uint32_t starts;   // bit i: token first + i is the first of its story
    uint32_t ends;     // bit i: ... the last
    uint32_t rank;     // stories that start before `first`
};

__device__ __forceinline__ Segment segment_at(const LeoB200StoryTables& t, uint32_t first) {
    Segment s{first, 0, 0, 0, 0};
    if (first >= t.tokens) return s;
    s.count = (int)min(t.tokens - first, (uint32_t)kSegment);
    const uint4 w = __ldg(reinterpret_cast<const uint4*>(t.words) + (first >> 5));  // starts, rank, begin, end
    const uint32_t base = first & ~31u, shift = first & 31u;
    const uint32_t ends = (w.x >> 1) | (w.w <= base + 32u ? 1u << (w.w - 1u - base) : 0u);
    s.starts = (w.x >> shift) & ((1u << kSegment) - 1u);
    s.ends = (ends >> shift) & ((1u << kSegment) - 1u);
    s.rank = w.y + __popc(w.x & ((1u << shift) - 1u));
    return s;
}
// The story that starts at, or ends with, token i of the segment.
__device__ __forceinline__ uint32_t story_starting(const LeoB200StoryTables& t, const Segment& s, int i) {
    return __ldg(t.order + s.rank + __popc(s.starts & ((1u << i) - 1u)));
}
__device__ __forceinline__ uint32_t story_ending(const LeoB200StoryTables& t, const Segment& s, int i) {
    return __ldg(t.order + s.rank + __popc(s.starts & ((2u << i) - 1u)) - 1u);
}

template <int V>
__device__ __forceinline__ void row_or_zero(const float* rows, uint32_t row, uint32_t channels, uint32_t c,
                                            bool active, float (&v)[V]) {
#pragma unroll
    for (int k = 0; k < V; ++k) v[k] = rows && active ? __ldg(rows + (size_t)row * channels + c + k) : 0.0f;
}

// A product of gates as hi + lo: the rounding of every factor is kept
// (p = hi a, e = hi a - p exactly), so that the map of a long span of slow
// gates is exact to float32 where a plain product would drift by a rounding a
// token, the same one in every span if the gates are constant.
struct Product {
    float hi = 1.0f, lo = 0.0f;
    __device__ __forceinline__ void times(float a) {
        const float p = hi * a;
        lo = fmaf(lo, a, fmaf(hi, a, -p));
        hi = p;
    }
    __device__ __forceinline__ double value() const {
        // an infinite product has no error term
        return isfinite(hi) ? (double)hi + (double)lo : (double)hi;
    }
};

// Waits until `flag` is set; false if it gave up.
__device__ __forceinline__ bool wait_for(const uint32_t* flag) {
    for (uint32_t n = 0; n < kSpinLimit; ++n) {
        uint32_t v;
        asm volatile("ld.acquire.gpu.global.u32 %0, [%1];" : "=r"(v) : "l"(flag) : "memory");
        if (v) return true;
        __nanosleep(32);
    }
    atomicExch(&g_gave_up, 1u);
    return false;
}

__device__ __forceinline__ double2 read_slot(const double2* p) {
    return __ldcg(p);
}

// One warp, a channel a lane.  The state before tile `tile` in the direction
// of the scan (+1: from the left), from the tile that holds the near end of the
// story that crosses into it (`holder`) or a nearer one that published a state.
template <int Direction>
__device__ __forceinline__ double carry_into(const Scratch& s, uint32_t tile, uint32_t holder, uint32_t flag_at,
                                             uint32_t channels, uint32_t c, bool active) {
    const uint32_t lane = threadIdx.x & 31u;
    // Tiles that publish a state: the last of a group of kGroup seen in the direction of the scan.
    uint32_t from = holder;
    if (Direction > 0) {
        const uint32_t p = tile / kGroup * kGroup;  // its left neighbour ends a group
        if (p > holder + 1) from = p - 1;
    } else {
        const uint32_t p = (tile / kGroup + 1) * kGroup;
        if (p < holder) from = p;
    }
    const uint32_t maps = Direction > 0 ? tile - 1 - from : from - tile - 1;  // below kGroup
    bool ok = true;
    if (lane < maps) {
        const uint32_t at = Direction > 0 ? from + 1 + lane : from - 1 - lane;
        ok = wait_for(s.flags + (size_t)at * s.flag_row + flag_at);
    }
    ok = __all_sync(0xffffffffu, ok);
    __syncwarp();
    double A = 1.0, H = 0.0;
    if (active)
        for (uint32_t j = 0; j < maps; ++j) {
            const uint32_t at = Direction > 0 ? from + 1 + j : from - 1 - j;
            const double2 m = read_slot(s.slots + (size_t)at * channels + c);
            H = fma(m.x, H, m.y);
            A *= m.x;
        }
    if (lane == 0) ok = ok && wait_for(s.flags + (size_t)from * s.flag_row + flag_at);
    ok = __all_sync(0xffffffffu, ok);
    __syncwarp();
    if (!ok) return CUDART_NAN;
    if (!active) return 0.0;
    const double before = read_slot(s.slots + (size_t)from * channels + c).y;
    return maps ? fma(A, before, H) : before;
}

__device__ __forceinline__ void publish(const Scratch& s, uint32_t tile, uint32_t flag_at, uint32_t channels,
                                        uint32_t c, bool active, double A, double H) {
    if (active) __stcg(s.slots + (size_t)tile * channels + c, make_double2(A, H));
    __syncwarp();
    if ((threadIdx.x & 31u) == 0) {
        __threadfence();
        asm volatile("st.release.gpu.global.u32 [%0], %1;" ::"l"(s.flags + (size_t)tile * s.flag_row + flag_at), "r"(1u)
                     : "memory");
    }
}

// The maps of a tile's segments, and the states before them.
template <int V>
struct TileMaps {
    double A[kTileWarps][32 * V];
    float H[kTileWarps][32 * V];
    float before[kTileWarps][32 * V];
    uint32_t reset[kTileWarps];
    uint32_t ticket;
};

// The block's tile and channel group.
template <int V>
__device__ __forceinline__ uint32_t take_ticket(const ScanArgs& a, TileMaps<V>& maps) {
    if (a.tiles == 1) return blockIdx.x;
    if (threadIdx.x == 0) maps.ticket = atomicAdd(a.scratch.ticket, 1u);
    __syncthreads();
    return maps.ticket;
}

// Composes the tile's segments after a barrier: the first V warps, a channel a
// lane, publish the tile's map or state and write the state before each segment.
// Returns the state before the tile in those warps.
template <int V, int Direction>
__device__ __forceinline__ double compose_tile(const ScanArgs& a, TileMaps<V>& maps, uint32_t tile, uint32_t group) {
    const uint32_t warp = threadIdx.x >> 5;
    double carry = 0.0;
    if (warp < V) {
        const uint32_t k = threadIdx.x;  // channel of the group
        const uint32_t c = group * 32 * V + k, flag_at = group * V + warp;
        const bool active = c < a.channels;
        double A = 1.0, H = 0.0;
        bool reset = false;
#pragma unroll
        for (int j = 0; j < kTileWarps; ++j) {
            const int w = Direction > 0 ? j : kTileWarps - 1 - j;
            if (maps.reset[w]) {
                H = maps.H[w][k];
                reset = true;
            } else {
                H = fma(maps.A[w][k], H, (double)maps.H[w][k]);
                A *= maps.A[w][k];
            }
        }
        // Does a story cross into the tile, and which tile holds its other end?
        const uint32_t words = (a.tables.tokens + 31) / 32;
        uint32_t holder = tile;
        if (a.tiles > 1) {
            if (Direction > 0)
                holder = __ldg(&a.tables.words[tile * (kTile / 32)].begin) / kTile;
            else
                holder = (__ldg(&a.tables.words[min((tile + 1) * (kTile / 32), words) - 1].end) - 1) / kTile;
        }
        const bool last = Direction > 0 ? tile + 1 == a.tiles : tile == 0;
        const bool state_tile = Direction > 0 ? (tile + 1) % kGroup == 0 : tile % kGroup == 0;
        if (!last && (reset || !state_tile)) publish(a.scratch, tile, flag_at, a.channels, c, active, A, H);
        if (holder != tile) {
            carry = carry_into<Direction>(a.scratch, tile, holder, flag_at, a.channels, c, active);
            if (!last && !reset && state_tile)
                publish(a.scratch, tile, flag_at, a.channels, c, active, 0.0, fma(A, carry, H));
        } else if (!last && !reset && state_tile) {
            publish(a.scratch, tile, flag_at, a.channels, c, active, 0.0, H);
        }
        double before = carry;
#pragma unroll
        for (int j = 0; j < kTileWarps; ++j) {
            const int w = Direction > 0 ? j : kTileWarps - 1 - j;
            maps.before[w][k] = (float)before;
            before = maps.reset[w] ? (double)maps.H[w][k] : fma(maps.A[w][k], before, (double)maps.H[w][k]);
        }
    }
    return carry;
}

// Stories without a token keep their initial (forward) or final (backward) row.
__device__ __forceinline__ void copy_empty(const LeoB200StoryTables& t, uint32_t channels, uint32_t c0, uint32_t width,
                                           const float* from, float* to) {
    for (uint32_t e = t.full; e < t.stories; ++e) {
        const size_t row = (size_t)t.order[e] * channels;
        for (uint32_t c = c0 + threadIdx.x; c < min(c0 + width, channels); c += kTileThreads)
            to[row + c] = from ? from[row + c] : 0.0f;
    }
}

template <typename T, typename G, int V, bool Shared>
__global__ void __launch_bounds__(kTileThreads, 3) scan_forward_kernel(const __grid_constant__ ScanArgs a) {
    __shared__ TileMaps<V> maps;
    const uint32_t ticket = take_ticket<V>(a, maps);
    const uint32_t tile = ticket / a.groups, group = ticket % a.groups;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t c = group * 32 * V + lane * V;
    const bool active = c < a.channels;
    const uint32_t first = tile * kTile + warp * kSegment;

    typename Packed<T, V>::Raw x[kSegment];
    typename Packed<G, V>::Raw gate[Shared ? 1 : kSegment];
    const Segment s = segment_at(a.tables, first);
    const T* xp = static_cast<const T*>(a.drive) + (int64_t)first * a.drive_stride + c;
    const G* gp = static_cast<const G*>(a.decay) + (Shared ? 0 : (int64_t)first * a.decay_stride) + c;
    float unit[V], none[V];
#pragma unroll
    for (int k = 0; k < V; ++k) unit[k] = 1.0f, none[k] = 0.0f;
    if (Shared) gate[0] = active ? read_once<G, V>(gp) : Packed<G, V>::pack(unit);
#pragma unroll
    for (int i = 0; i < kSegment; ++i) {
        const bool in = active && i < s.count;
        x[i] = in ? read_once<T, V>(xp + i * a.drive_stride) : Packed<T, V>::pack(none);
        if (!Shared) gate[i] = in ? read_once<G, V>(gp + i * a.decay_stride) : Packed<G, V>::pack(unit);
    }

    Product A[V];
    float H[V];
#pragma unroll
    for (int k = 0; k < V; ++k) H[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kSegment; ++i) {
        float xi[V], gi[V];
        Packed<T, V>::unpack(x[i], xi);
        Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
        if (s.starts >> i & 1u) row_or_zero<V>(a.initial, story_starting(a.tables, s, i), a.channels, c, active, H);
        const bool past = Shared && i >= s.count;  // a shared gate does not stop at the batch's end by itself
#pragma unroll
        for (int k = 0; k < V; ++k) {
            H[k] = past ? H[k] : fmaf(gi[k], H[k], xi[k]);
            if (!past) A[k].times(gi[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        maps.A[warp][lane * V + k] = A[k].value();
        maps.H[warp][lane * V + k] = H[k];
    }
    if (lane == 0) maps.reset[warp] = s.starts != 0;
    __syncthreads();
    const double carry = compose_tile<V, 1>(a, maps, tile, group);
    if (a.carries && warp < V && group * 32 * V + threadIdx.x < a.channels)
        a.carries[(size_t)tile * a.channels + group * 32 * V + threadIdx.x] = (float)carry;
    __syncthreads();

    float h[V];
#pragma unroll
    for (int k = 0; k < V; ++k) h[k] = maps.before[warp][lane * V + k];
    T* out = static_cast<T*>(a.states) + (size_t)first * a.channels + c;
#pragma unroll
    for (int i = 0; i < kSegment; ++i) {
        float xi[V], gi[V];
        Packed<T, V>::unpack(x[i], xi);
        Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
        if (s.starts >> i & 1u) row_or_zero<V>(a.initial, story_starting(a.tables, s, i), a.channels, c, active, h);
#pragma unroll
        for (int k = 0; k < V; ++k) h[k] = fmaf(gi[k], h[k], xi[k]);
        if (active && i < s.count) write_once<T, V>(out + (size_t)i * a.channels, h);
        if (s.ends >> i & 1u) {
            const size_t row = (size_t)story_ending(a.tables, s, i) * a.channels + c;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (active) a.final_states[row + k] = h[k];
        }
    }
    if (tile == 0 && a.tables.full < a.tables.stories)
        copy_empty(a.tables, a.channels, group * 32 * V, 32 * V, a.initial, a.final_states);
}

template <typename T, typename G, int V, bool Shared>
__global__ void __launch_bounds__(kTileThreads, 2) scan_backward_kernel(const __grid_constant__ ScanArgs a) {
    __shared__ TileMaps<V> maps;
    const uint32_t ticket = take_ticket<V>(a, maps);
    const uint32_t tile = a.tiles - 1 - ticket / a.groups, group = ticket % a.groups;
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5;
    const uint32_t c = group * 32 * V + lane * V;
    const bool active = c < a.channels;
    const uint32_t first = tile * kTile + warp * kSegment;

    typename Packed<T, V>::Raw x[kSegment], g[kSegment];
    typename Packed<G, V>::Raw gate[Shared ? 1 : kSegment];
    const Segment s = segment_at(a.tables, first);
    const T* xp = static_cast<const T*>(a.drive) + (int64_t)first * a.drive_stride + c;
    const T* sp = static_cast<const T*>(a.grad_states) + (int64_t)first * a.grad_states_stride + c;
    const G* gp = static_cast<const G*>(a.decay) + (Shared ? 0 : (int64_t)first * a.decay_stride) + c;
    float unit[V], none[V];
#pragma unroll
    for (int k = 0; k < V; ++k) unit[k] = 1.0f, none[k] = 0.0f;
    if (Shared) gate[0] = active ? read_once<G, V>(gp) : Packed<G, V>::pack(unit);
#pragma unroll
    for (int i = 0; i < kSegment; ++i) {
        const bool in = active && i < s.count;
        x[i] = in ? read_once<T, V>(xp + i * a.drive_stride) : Packed<T, V>::pack(none);
        if (!Shared) gate[i] = in ? read_once<G, V>(gp + i * a.decay_stride) : Packed<G, V>::pack(unit);
        g[i] = in ? read_once<T, V>(sp + i * a.grad_states_stride) : Packed<T, V>::pack(none);
    }

    // The segment's map from the left.
    Product A[V];
    float H[V];
#pragma unroll
    for (int k = 0; k < V; ++k) H[k] = 0.0f;
#pragma unroll
    for (int i = 0; i < kSegment; ++i) {
        float xi[V], gi[V];
        Packed<T, V>::unpack(x[i], xi);
        Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
        if (s.starts >> i & 1u) row_or_zero<V>(a.initial, story_starting(a.tables, s, i), a.channels, c, active, H);
        const bool past = Shared && i >= s.count;
#pragma unroll
        for (int k = 0; k < V; ++k) {
            H[k] = past ? H[k] : fmaf(gi[k], H[k], xi[k]);
            if (!past) A[k].times(gi[k]);
        }
    }
#pragma unroll
    for (int k = 0; k < V; ++k) {
        maps.A[warp][lane * V + k] = A[k].value();
        maps.H[warp][lane * V + k] = H[k];
    }
    if (lane == 0) maps.reset[warp] = s.starts != 0;
    __syncthreads();

    // The state before each token: from the tile's carry through the segments before this one.
    float h[kSegment][V];
    {
        float before[V];
#pragma unroll
        for (int k = 0; k < V; ++k) {
            double b = active && s.count > 0 ? (double)__ldcs(a.carries + (size_t)tile * a.channels + c + k) : 0.0;
            for (uint32_t w = 0; w < warp; ++w)
                b = maps.reset[w] ? (double)maps.H[w][lane * V + k]
                                  : fma(maps.A[w][lane * V + k], b, (double)maps.H[w][lane * V + k]);
            before[k] = (float)b;
        }
#pragma unroll
        for (int i = 0; i < kSegment; ++i) {
            float xi[V], gi[V];
            Packed<T, V>::unpack(x[i], xi);
            Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
            if (s.starts >> i & 1u)
                row_or_zero<V>(a.initial, story_starting(a.tables, s, i), a.channels, c, active, before);
#pragma unroll
            for (int k = 0; k < V; ++k) {
                h[i][k] = before[k];
                before[k] = fmaf(gi[k], before[k], xi[k]);
            }
        }
    }
    __syncthreads();

    // The segment's map from the right: m[t] = a[t] (g[t] + m[t + 1]).
#pragma unroll
    for (int k = 0; k < V; ++k) H[k] = 0.0f;
#pragma unroll
    for (int i = kSegment - 1; i >= 0; --i) {
        float si[V], gi[V];
        Packed<T, V>::unpack(g[i], si);
        Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
        if (s.ends >> i & 1u) row_or_zero<V>(a.grad_final, story_ending(a.tables, s, i), a.channels, c, active, H);
        const bool past = Shared && i >= s.count;
#pragma unroll
        for (int k = 0; k < V; ++k) H[k] = past ? H[k] : gi[k] * (si[k] + H[k]);
    }
#pragma unroll
    for (int k = 0; k < V; ++k) maps.H[warp][lane * V + k] = H[k];
    if (lane == 0) maps.reset[warp] = s.ends != 0;
    __syncthreads();
    compose_tile<V, -1>(a, maps, tile, group);
    __syncthreads();

    float m[V], sum[V];
#pragma unroll
    for (int k = 0; k < V; ++k) m[k] = maps.before[warp][lane * V + k], sum[k] = 0.0f;
    T* out = static_cast<T*>(a.grad_drive) + (size_t)first * a.channels + c;
    G* out_gate = static_cast<G*>(a.grad_decay) + (size_t)first * a.channels + c;
#pragma unroll
    for (int i = kSegment - 1; i >= 0; --i) {
        float si[V], gi[V], term[V];
        Packed<T, V>::unpack(g[i], si);
        Packed<G, V>::unpack(gate[Shared ? 0 : i], gi);
        if (s.ends >> i & 1u) row_or_zero<V>(a.grad_final, story_ending(a.tables, s, i), a.channels, c, active, m);
#pragma unroll
        for (int k = 0; k < V; ++k) {
            si[k] += m[k];
            term[k] = si[k] * h[i][k];
            m[k] = gi[k] * si[k];
        }
        if (i < s.count) {
            if (active) write_once<T, V>(out + (size_t)i * a.channels, si);
            if (!Shared) {
                if (active) write_once<G, V>(out_gate + (size_t)i * a.channels, term);
            } else {
#pragma unroll
                for (int k = 0; k < V; ++k) sum[k] += term[k];
            }
        }
        if (a.grad_initial && (s.starts >> i & 1u)) {
            const size_t row = (size_t)story_starting(a.tables, s, i) * a.channels + c;
#pragma unroll
            for (int k = 0; k < V; ++k)
                if (active) a.grad_initial[row + k] = m[k];
        }
    }
    if (Shared) {
        // The tile's sum, its segments in order.
#pragma unroll
        for (int k = 0; k < V; ++k) maps.H[warp][lane * V + k] = sum[k];
        __syncthreads();
        if (warp < V && group * 32 * V + threadIdx.x < a.channels) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kTileWarps; ++w) total += maps.H[w][threadIdx.x];
            if (a.tiles == 1)
                store(static_cast<G*>(a.grad_decay) + group * 32 * V + threadIdx.x, total);
            else
                a.scratch.partials[(size_t)tile * a.channels + group * 32 * V + threadIdx.x] = total;
        }
    }
    if (tile == 0 && a.grad_initial && a.tables.full < a.tables.stories)
        copy_empty(a.tables, a.channels, group * 32 * V, 32 * V, a.grad_final, a.grad_initial);
}

// The gradient of a shared row of gates: the tiles' sums in double, a column of
// 32 channels a block, every fourth tile a warp.
template <typename G>
__global__ void __launch_bounds__(kThreads) shared_decay_kernel(const float* partials, uint32_t tiles,
                                                                uint32_t channels, G* out) {
    __shared__ double sums[kThreads / 32][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    double sum = 0.0;
    if (c < channels)
#pragma unroll 8
        for (uint32_t t = warp; t < tiles; t += kThreads / 32) sum += (double)partials[(size_t)t * channels + c];
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || c >= channels) return;
    for (uint32_t w = 1; w < kThreads / 32; ++w) sum += sums[w][lane];
    store(out + c, (float)sum);
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
    require(t->tokens < (1u << 31), "too many tokens for one scan");
    require(t->full <= t->stories && (t->full > 0) == (t->tokens > 0), "story tables are inconsistent");
    require(t->order != nullptr && (t->tokens == 0 || t->words != nullptr), "story tables are null");
    require(channels > 0 && channels < (1u << 31), "channels must be positive");
}

uint32_t tiles_of(uint32_t tokens) { return tokens == 0 ? 1 : (tokens - 1) / kTile + 1; }

// The parts of a call's scratch; returns its size.
size_t lay_out(uint32_t tokens, uint32_t channels, void* base, Scratch* s) {
    const size_t tiles = tiles_of(tokens);
    if (tiles == 1) return 0;  // nothing crosses tiles
    const size_t flag_row = ((size_t)channels + 63) / 64 * 2;
    const size_t flags = 256, slots = (flags + tiles * flag_row * sizeof(uint32_t) + 255) / 256 * 256;
    const size_t partials = slots + tiles * channels * sizeof(double2);
    if (s) {
        char* p = static_cast<char*>(base);
        s->ticket = reinterpret_cast<uint32_t*>(p);
        s->flags = reinterpret_cast<uint32_t*>(p + flags);
        s->slots = reinterpret_cast<double2*>(p + slots);
        s->partials = reinterpret_cast<float*>(p + partials);
        s->flag_row = (uint32_t)flag_row;
    }
    return partials + tiles * channels * sizeof(float);
}

// Whether rows of `channels` elements of `size` bytes can be moved two at a time.
bool in_pairs(const void* p, int64_t stride, size_t size) {
    return reinterpret_cast<uintptr_t>(p) % (2 * size) == 0 && stride % 2 == 0;
}

// Fills the tiling of `a`, clears the scratch on `stream`; the number of blocks.
uint32_t begin_scan(ScanArgs& a, int V, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    a.tiles = tiles_of(a.tables.tokens);
    a.groups = (a.channels + 32 * V - 1) / (32 * V);
    require((uint64_t)a.tiles * a.groups < (1ull << 31), "too many tokens and channels for one scan");
    const size_t size = lay_out(a.tables.tokens, a.channels, workspace, &a.scratch);
    if (size > 0) {
        require(workspace != nullptr && workspace_bytes >= size, "the workspace is too small");
        require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be aligned to 16 bytes");
        check(cudaMemsetAsync(workspace, 0, 256 + (size_t)a.tiles * a.scratch.flag_row * sizeof(uint32_t), stream),
              "clear scan flags");
    }
    return a.tiles * a.groups;
}

// Calls body(V, Shared) as types.
template <typename Body>
void dispatch_shape(bool pairs, bool shared, Body&& body) {
    using One = std::integral_constant<int, 1>;
    using Two = std::integral_constant<int, 2>;
    if (pairs && shared) body(Two{}, std::true_type{});
    else if (pairs) body(Two{}, std::false_type{});
    else if (shared) body(One{}, std::true_type{});
    else body(One{}, std::false_type{});
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

size_t leo_b200_gated_scan_workspace(uint32_t tokens, uint32_t channels) {
    return lay_out(tokens, channels, nullptr, nullptr);
}

size_t leo_b200_gated_scan_carry_count(uint32_t tokens, uint32_t channels) {
    return (size_t)tiles_of(tokens) * channels;
}

int leo_b200_gated_scan(int device, const LeoB200StoryTables* tables, uint32_t channels, int dtype,
                        const void* drive, int64_t drive_stride, int decay_dtype, const void* decay,
                        int64_t decay_stride, int decay_shared, const float* initial, void* states,
                        float* final_states, float* carries, void* workspace, size_t workspace_bytes, void* stream) {
    return guarded([&] {
        check_tables(tables, channels);
        require(tables->tokens == 0 || (drive && decay && states), "scan arrays are null");
        require(final_states != nullptr, "final states are null");
        ScanArgs a{};
        a.tables = *tables;
        a.channels = channels;
        a.drive = drive;
        a.drive_stride = drive_stride;
        a.decay = decay;
        a.decay_stride = decay_stride;
        a.initial = initial;
        a.states = states;
        a.final_states = final_states;
        a.carries = carries;
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            const bool pairs = channels % 2 == 0 && in_pairs(drive, drive_stride, sizeof(T)) &&
                               in_pairs(decay, decay_shared ? 0 : decay_stride, sizeof(G)) &&
                               in_pairs(states, 0, sizeof(T));
            DeviceScope scope(device);
            dispatch_shape(pairs, decay_shared != 0 && tables->tokens > 0, [&](auto v, auto shared) {
                const uint32_t blocks = begin_scan(a, v(), workspace, workspace_bytes, (cudaStream_t)stream);
                scan_forward_kernel<T, G, v(), shared()><<<blocks, kTileThreads, 0, (cudaStream_t)stream>>>(a);
                check(cudaGetLastError(), "scan_forward_kernel");
            });
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
        ScanArgs a{};
        a.tables = *tables;
        a.channels = channels;
        a.drive = drive;
        a.drive_stride = drive_stride;
        a.decay = decay;
        a.decay_stride = decay_stride;
        a.initial = initial;
        a.carries = const_cast<float*>(carries);
        a.grad_states = grad_states;
        a.grad_states_stride = grad_states_stride;
        a.grad_final = grad_final;
        a.grad_drive = grad_drive;
        a.grad_decay = grad_decay;
        a.grad_initial = grad_initial;
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            const bool pairs = channels % 2 == 0 && in_pairs(drive, drive_stride, sizeof(T)) &&
                               in_pairs(decay, decay_shared ? 0 : decay_stride, sizeof(G)) &&
                               in_pairs(grad_states, grad_states_stride, sizeof(T)) &&
                               in_pairs(grad_drive, 0, sizeof(T)) && in_pairs(grad_decay, 0, sizeof(G));
            DeviceScope scope(device);
            dispatch_shape(pairs, decay_shared != 0, [&](auto v, auto shared) {
                const uint32_t blocks = begin_scan(a, v(), workspace, workspace_bytes, (cudaStream_t)stream);
                scan_backward_kernel<T, G, v(), shared()><<<blocks, kTileThreads, 0, (cudaStream_t)stream>>>(a);
                check(cudaGetLastError(), "scan_backward_kernel");
                if (decay_shared && a.tiles > 1) {
                    shared_decay_kernel<G><<<(channels + 31) / 32, kThreads, 0, (cudaStream_t)stream>>>(
                        a.scratch.partials, a.tiles, channels, static_cast<G*>(grad_decay));
                    check(cudaGetLastError(), "shared_decay_kernel");
                }
            });
        });
    });
}

int leo_b200_gated_scan_status(int device, uint32_t* gave_up) {
    return guarded([&] {
        require(gave_up != nullptr, "status is null");
        DeviceScope scope(device);
        check(cudaDeviceSynchronize(), "gated scan status");
        check(cudaMemcpyFromSymbol(gave_up, g_gave_up, sizeof(uint32_t)), "gated scan status");
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
