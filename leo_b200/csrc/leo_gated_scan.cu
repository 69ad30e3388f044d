// The gated linear recurrence over packed stories, its backward pass and its
// one-token step (include/leo_b200.h).
//
//   h[t] = a[t] h[t-1] + x[t]
//   slope[t] = g[t] + a[t+1] slope[t+1];  dx = slope, da[t] = slope[t] h[t-1]
//
// Maps.  A span of tokens maps the state before it to the state after it as
// h -> A h + H (A the product of the gates, H the state from zero), or as
// h -> H if a story starts inside, and such maps compose.  The batch is cut into
// tiles of 128 tokens or fewer (leo_b200_story_table): a block takes a tile of
// 64 channels, each thread a segment of 8 tokens of four channels (4 tokens in
// tiles of 64, where a stage of 128 would not fit).  The segments' maps give the
// tile's, the tiles' maps the state before a tile, and each thread then runs its
// tokens again and writes them.  The backward pass is the same from the right,
// with m -> A m + M for m[t] = a[t] slope[t]; h is formed anew from the states
// that the forward pass keeps every 64 tokens.
//
// Pipeline.  One block an SM works through tiles dealt by a ticket, every input
// read once.  Two teams of eight warps take tiles in turn: a team loads the tile
// after its next into shared memory (tiled loads where rows keep 16 bytes, each
// warp what it will use itself, so they need no barrier), maps its tile and
// writes it, and the other team's work fills its waits.  Four warps compose a
// tile's segments; four more scout, that is they do all the reading between
// tiles (slots, kept states, tickets, the schedule), since a warp with a load in
// flight waits for it with every read of shared memory.  Where four stages do
// not fit, one team with three maps tile i + 1 between the map and the writing
// of tile i.  81,920 tokens x 1,024 channels (bfloat16, float gates) in 64 stories:
// 141 us with one team and 127 us with two, 103 us at the rate of a copy; 20,480
// x 4,096 in 32 stories 141 and 260 us backward, 103 and 180 us at that rate.  A
// loop of the same loads and stores alone runs at a copy's rate, so the rest is
// the length of a tile's chain, from its loads to its map, the composing and the writes.
//
// Between tiles.  Each tile publishes its map, every kGroup-th the state after
// it instead, so a tile reads at most kGroup slots.  A slot and its mark are one
// 8-byte word, so a slot that is there costs one trip to L2.  Tickets deal the
// first tiles of all stories, then their second ones, and so on: a tile's
// predecessors have lower tickets, so they have started before it and every wait
// ends, and with many stories they are long done when it reads them.  (Tiles in
// the order of their tokens wait for neighbours that are mapped in the same
// moment, which took a quarter longer.)  Which slots are read, and in which
// order they are composed, depends on the layout alone: results are the same in
// every run.  Where a single long story leaves too few tiles side by side, the
// maps are found in a pass of their own (scan_map_kernel and on).
#include <cuda.h>
#include <cuda_bf16.h>
#include <cuda_fp16.h>
#include <cuda_runtime.h>
#include <math_constants.h>
#include <stdint.h>

#include <algorithm>
#include <cstring>
#include <type_traits>
#include <vector>

#include "../../include/leo_b200.h"
#include "leo_operator_device.cuh"
#include "leo_operator_host.h"

namespace {

using namespace leo_operator;

constexpr uint32_t kReduceThreads = 1024;

constexpr int kWarps = 8;                        // of a team, which maps and writes a tile
constexpr int kSegments = 2 * kWarps;            // of a tile, half a warp each
constexpr int kColumns = 64;                     // channels of a tile, four a thread
constexpr int kComposeWarps = kColumns / 16;     // that compose it, two lanes a channel
constexpr int kScoutWarps = kColumns / 16;       // that find the state before it, two lanes a channel
constexpr uint32_t kNone = 0xffffffffu;
constexpr size_t kSharedLimit = 227 * 1024;
constexpr uint32_t kKept = LEO_B200_TILE_TOKENS / 2;  // tokens between the states kept for the backward pass
constexpr int kGroup = 16;                       // tiles between published states
// Where fewer tiles than this can be worked on without waiting for one another
// (the stories' channel groups), they are mapped ahead, which reads the inputs
// twice.  One story of 65,536 tokens, bfloat16 with float gates, so and in one pass:
// 64 channels forward 29 and 61 us, backward 35 and 68 us; 512 channels (8 abreast)
// 121 and 135 us, 148 and 158 us; 1,024 channels (16) 213 and 211 us, 268 and 252 us.
constexpr uint32_t kAbreast = 12;
constexpr uint32_t kSpinLimit = 1u << 21;        // polls of a wait, a memory round trip and more apart

__device__ uint32_t g_gave_up;

// A thread's four channels.
struct Quad {
    Pair32 v[2] = {0, 0};
};

// N neighbours of a row as they lie in memory, and pairs of them as floats.
template <typename T, int N> struct Packed {
    using Raw = std::conditional_t<N * sizeof(T) == 16, uint4, std::conditional_t<N * sizeof(T) == 8, uint2, uint32_t>>;
};
// What a tile tells the tiles behind it, in one 8-byte word: its map (A, H),
// or the state after it as H.  All bits set: nothing yet (a NaN of that form
// is written as another one).
using Slot = unsigned long long;
__device__ __forceinline__ void write_slot(Slot* p, float A, float H) {
    uint32_t low = __float_as_uint(A);
    if (low == kNone) low = 0x7fffffffu;
    asm volatile("st.relaxed.gpu.global.u64 [%0], %1;" ::"l"(p), "l"((Slot)__float_as_uint(H) << 32 | low) : "memory");
}
__device__ __forceinline__ Slot read_slot(const Slot* p) {
    Slot s;
    asm volatile("ld.relaxed.gpu.global.u64 %0, [%1];" : "=l"(s) : "l"(p) : "memory");
    return s;
}

// The scratch of one call: a slot for every channel of a tile (all bits set
// before the launch), the ticket before them (set to -1 with them), and the
// partial sums of a shared gate's gradient.
struct Scratch {
    uint32_t* ticket;
    Slot* slots;      // [tiles][channels]
    float* partials;  // [tiles][channels]
};

struct ScanArgs {
    CUtensorMap drive_map, decay_map, grad_map;  // of the tiled loads
    LeoB200StoryTables tables;
    const LeoB200StoryTile* schedule;  // the tiles in the order of their tickets
    uint32_t channels, tiles, groups;  // groups: of 64 channels
    const void* drive;
    int64_t drive_stride;
    const void* decay;
    int64_t decay_stride;
    const float* initial;
    void* states;
    float* final_states;
    float* carries;  // [every 64 tokens][channels]: the state before them
    // backward
    const void* grad_states;
    int64_t grad_states_stride;
    const float* grad_final;
    void* grad_drive;
    void* grad_decay;
    float* grad_initial;
    Scratch scratch;
};

// A thread's tokens among the stories.
struct Segment {
    int count;        // tokens of the tile
    uint32_t starts;  // bit i: token i of the segment is the first of its story
    uint32_t ends;    // bit i: ... the last
    uint32_t rank;    // stories that start before the segment
};

// The two words of the story table that a segment's tokens lie in.
struct StoryBits {
    uint2 low, high;  // starts, rank
};
__device__ __forceinline__ StoryBits story_bits(const LeoB200StoryTables& t, uint32_t first) {
    const uint2* p = reinterpret_cast<const uint2*>(t.words) + (first >> 5);
    return {__ldg(p), __ldg(p + 1)};
}
__device__ __forceinline__ Segment segment_of(const StoryBits& b, uint32_t first, int count) {
    Segment s{count, 0, 0, 0};
    if (count <= 0) return s;
    const uint32_t shift = first & 31u, mask = (1u << count) - 1u;
    const uint32_t bits = (uint32_t)(((uint64_t)b.high.x << 32 | b.low.x) >> shift);
    s.starts = bits & mask;
    s.ends = bits >> 1 & mask;
    s.rank = b.low.y + __popc(b.low.x & ((1u << shift) - 1u));
    return s;
}
// The story that starts at, or ends with, token i of the segment.
__device__ __forceinline__ uint32_t story_starting(const LeoB200StoryTables& t, const Segment& s, int i) {
    return __ldg(t.order + s.rank + __popc(s.starts & ((1u << i) - 1u)));
}
__device__ __forceinline__ uint32_t story_ending(const LeoB200StoryTables& t, const Segment& s, int i) {
    return __ldg(t.order + s.rank + __popc(s.starts & ((2u << i) - 1u)) - 1u);
}

// A product of gates as hi + lo: the rounding of every factor is kept
// (p = hi a, e = hi a - p exactly), so that the map of a long span of slow
// gates is exact to float32 where a plain product would drift by a rounding a
// token, the same one in every span if the gates are constant.
struct Product4 {  // of four channels
    Pair32 hi[2] = {0x3f8000003f800000ull, 0x3f8000003f800000ull}, lo[2] = {0, 0};
    __device__ __forceinline__ void times(const Quad& a) {
#pragma unroll
        for (int q = 0; q < 2; ++q) {
            const Pair32 p = mul2(hi[q], a.v[q]);
            lo[q] = fma2(lo[q], a.v[q], fma2(hi[q], a.v[q], p ^ 0x8000000080000000ull));
            hi[q] = p;
        }
    }
};
__device__ __forceinline__ float2 product_of(float2 x, float2 y) {  // (hi, lo)
    const float p = x.x * y.x;
    return make_float2(p, fmaf(x.x, y.y, fmaf(x.y, y.x, fmaf(x.x, y.x, -p))));
}
__device__ __forceinline__ float value_of(float2 x) {
    return x.y == x.y ? x.x + x.y : x.x;  // an infinite product has no error term
}

// A product of segments' products that underflows has to leave an infinite state
// infinite: it becomes the smallest float of its sign.  (It adds at most 2^-149 of a
// finite state, as a rounding among the subnormals does.)  A segment's own product may
// be 0, by a gate of 0 or by gates below 2^-18, and makes an infinite state NaN.
__device__ __forceinline__ float smallest(float zero) { return __uint_as_float(__float_as_uint(zero) | 1u); }
__device__ __forceinline__ float times(float x, float y) {
    const float p = x * y;
    return p == 0.0f && x != 0.0f && y != 0.0f ? smallest(p) : p;
}
__device__ __forceinline__ float2 times(float2 x, float2 y) {
    const float2 p = product_of(x, y);
    return p.x == 0.0f ? make_float2(times(x.x, y.x), 0.0f) : p;
}

// The state before a tile, out of the slots between it and the tile that holds
// the near end of the story that crosses into it, or the nearest one that
// published a state.  Direction +1: from the left; -1: from the right.
template <int Direction>
struct Lookback {
    uint32_t from;  // tile whose slot is a state
    int maps;       // tiles between it and this one; -1: no story crosses in
    __device__ __forceinline__ Lookback(uint32_t tile, uint32_t holder) {
        maps = -1;
        from = holder;
        if (holder == tile) return;
        // A state is published by the last tile of a group of kGroup in the direction of the scan.
        if (Direction > 0) {
            const uint32_t p = tile / kGroup * kGroup;
            if (p > holder + 1) from = p - 1;
            maps = (int)(tile - 1 - from);
        } else {
            const uint32_t p = (tile / kGroup + 1) * kGroup;
            if (p < holder) from = p;
            maps = (int)(from - tile - 1);
        }
    }
    // Half the slots of a channel: the state and the first seven maps (half 0),
    // or the other eight (half 1).
    __device__ __forceinline__ void load(const Slot* slots, uint32_t channels, uint32_t c, int half, Slot (&s)[8]) const {
        const int64_t step = (int64_t)Direction * channels;
        const int count = maps + 1 - half * 8;
        const Slot* p = slots + (size_t)from * channels + c + half * 8 * step;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) s[j] = read_slot(p + j * step);
    }
    // From the left: composes them as (A, H); false if one of them was not there yet.
    __device__ __forceinline__ bool compose(const Slot (&s)[8], int half, float& A, float& H) const {
        const int count = maps + 1 - half * 8;
        bool there = true;
        A = 1.0f, H = 0.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < count) {
                const uint32_t low = (uint32_t)s[j];
                const float value = __uint_as_float((uint32_t)(s[j] >> 32));
                there = there && low != kNone;
                H = j == 0 && half == 0 ? value : fmaf(__uint_as_float(low), H, value);
                A *= __uint_as_float(low);
            }
        return there;
    }
    // The product of half 1 again, kept from 0.
    __device__ __forceinline__ float product(const Slot (&s)[8]) const {
        float A = 1.0f;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < maps - 7) A = times(A, __uint_as_float((uint32_t)s[j]));
        return A;
    }
    // From the right: whether all are there.
    __device__ __forceinline__ bool there(const Slot (&s)[8], int half) const {
        bool all = true;
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < maps + 1 - half * 8) all = all && (uint32_t)s[j] != kNone;
        return all;
    }
    // The state after them; for half 1 from that after half 0.
    __device__ __forceinline__ float run(const Slot (&s)[8], int half, float state) const {
#pragma unroll
        for (int j = 0; j < 8; ++j)
            if (j < maps + 1 - half * 8) {
                const float value = __uint_as_float((uint32_t)(s[j] >> 32));
                state = j == 0 && half == 0 ? value : fmaf(__uint_as_float((uint32_t)s[j]), state, value);
            }
        return state;
    }
};

// A tile of a channel group.
struct Work {
    uint32_t first;   // token
    uint32_t count;   // tokens; kNone: no more work
    uint32_t tile;
    uint32_t group;
    uint32_t holder;  // the tile where the story that crosses into this one begins (forward) or ends; or this one
    uint32_t kept;    // the kept state before it
    uint32_t onward;  // whether a story crosses out of it
    uint32_t unused;
};

// The shape of a kernel: its tiles, and its shared memory.
template <typename T, typename G, bool Shared, bool Backward>
struct Shape {
    // A token of a tile takes this much of a stage.
    static constexpr int kRow = kColumns * (int)((Backward ? 2 : 1) * sizeof(T) + (Shared ? 0 : sizeof(G)));
    struct Maps {  // read and written up to 16 bytes at a time
        alignas(16) float2 A[Shared ? 1 : kSegments][kColumns];   // hi, lo; a shared gate's follow from the tokens
        alignas(16) float H[kSegments][kColumns];     // then the state before each segment
        alignas(16) float M[Backward ? kSegments : 1][kColumns];  // then the value before each segment from the right
        alignas(16) uint8_t starts[kSegments];
        alignas(16) uint8_t ends[kSegments];  // whether a story does in the segment
    };
    struct Control {
        Maps maps[2];
        alignas(16) float sums[Backward && Shared ? 2 : 1][Backward && Shared ? kSegments : 1][kColumns];
        Work ring[8];  // the block's work; an entry is rewritten when no warp reads it any more
        float scouted[2][Backward ? 2 : 1][kColumns];  // the value before the tile; the kept state before it
        uint64_t landed[4][kWarps];  // barriers of the tiled loads
    };
    static constexpr bool fits(int segment, int stages) {
        return (size_t)stages * segment * kSegments * kRow + sizeof(Control) <= kSharedLimit;
    }
    // Two teams with two stages each where they fit shared memory, one with three
    // where not; 8 tokens a thread, or 4 where not even those would.
    static constexpr int kTeams = fits(8, 4) || !fits(8, 3) ? 2 : 1;
    static constexpr int kStages = kTeams == 2 ? 4 : 3;
    static constexpr int kSegment = fits(8, kStages) ? 8 : 4;
    static constexpr uint32_t kTile = kSegment * kSegments;
    static constexpr size_t kStage = (size_t)kTile * kRow;
    static constexpr size_t kBytes = kStages * kStage + sizeof(Control);
    // Tickets are drawn so far ahead that a team finds the one whose loads it issues:
    // its own last turn is the newest that it knows to be over.
    static constexpr int kAhead = 2 + kTeams;
    static constexpr int kFirstComposer = kWarps * kTeams;
    static constexpr int kFirstScout = kFirstComposer + kComposeWarps;
    static constexpr uint32_t kThreads = 32 * (kFirstScout + kScoutWarps);
};

// Named barriers of a block, one of each kind for even and one for odd tiles.
enum Barrier {
    kMapped = 1,    // the segments' maps are written: mapping and composing warps
    kComposed = 3,  // the values before the segments are: the same
    kScouted = 5,   // the state before the tile is: scouting and composing warps
    kTaken = 7      // and it has been read: the same
};
template <int Kind>
constexpr int kThreadsOf = 32 * (kComposeWarps + (Kind < kScouted ? kWarps : kScoutWarps));
template <int Kind>
__device__ __forceinline__ void sync_of(uint32_t parity) {
    if (parity)
        asm volatile("bar.sync %0, %1;" ::"n"(Kind + 1), "n"(kThreadsOf<Kind>) : "memory");
    else
        asm volatile("bar.sync %0, %1;" ::"n"(Kind), "n"(kThreadsOf<Kind>) : "memory");
}
template <int Kind>
__device__ __forceinline__ void arrive_at(uint32_t parity) {
    if (parity)
        asm volatile("bar.arrive %0, %1;" ::"n"(Kind + 1), "n"(kThreadsOf<Kind>) : "memory");
    else
        asm volatile("bar.arrive %0, %1;" ::"n"(Kind), "n"(kThreadsOf<Kind>) : "memory");
}

template <int Bytes>
__device__ __forceinline__ void copy_async(void* shared, const void* global) {
    const uint32_t to = (uint32_t)__cvta_generic_to_shared(shared);
    asm volatile("cp.async.ca.shared.global [%0], [%1], %2;" ::"r"(to), "l"(global), "n"(Bytes) : "memory");
}

// Tiled loads of a warp's tokens, counted in bytes at a barrier of the warp.
__device__ __forceinline__ void expect_bytes(uint64_t* barrier, uint32_t bytes) {
    asm volatile("mbarrier.arrive.expect_tx.shared.b64 _, [%0], %1;" ::"r"((uint32_t)__cvta_generic_to_shared(barrier)),
                 "r"(bytes)
                 : "memory");
}
__device__ __forceinline__ void load_tile(void* to, const CUtensorMap* map, uint32_t channel, uint32_t token,
                                          uint64_t* barrier) {
    asm volatile(
        "cp.async.bulk.tensor.2d.shared::cluster.global.tile.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3}], [%4];" ::"r"(
            (uint32_t)__cvta_generic_to_shared(to)),
        "l"(map), "r"(channel), "r"(token), "r"((uint32_t)__cvta_generic_to_shared(barrier))
        : "memory");
}
__device__ __forceinline__ void wait_landed(uint64_t* barrier, uint32_t parity) {
    const uint32_t at = (uint32_t)__cvta_generic_to_shared(barrier);
    for (uint32_t n = 0; n < kSpinLimit; ++n) {
        uint32_t done;
        asm volatile(
            "{ .reg .pred p; mbarrier.try_wait.parity.shared.b64 p, [%1], %2; selp.u32 %0, 1, 0, p; }"
            : "=r"(done)
            : "r"(at), "r"(parity)
            : "memory");
        if (done) return;
    }
    atomicExch(&g_gave_up, 1u);
}

// A thread's four channels of a row, Unit of them neighbours: all four where
// rows are tiled loads (16-byte aligned), two where rows keep pairs aligned, or
// one.  Half a warp covers a row in 4 / Unit accesses.
template <int Unit>
struct Columns {
    uint32_t at0;       // first column of the tile
    uint32_t c;         // its channel
    uint32_t channels;
    __device__ __forceinline__ Columns(uint32_t group, uint32_t channels_) {
        at0 = (threadIdx.x & 15u) * Unit;
        c = group * kColumns + at0;
        channels = channels_;
    }
    // Offset of access u from the first column.
    static __device__ __forceinline__ constexpr uint32_t step(int u) { return u * 16u * Unit; }
    __device__ __forceinline__ bool in(int u) const { return c + step(u) < channels; }
    template <typename E>
    __device__ __forceinline__ void copy(E* tile_row, const E* row) const {
#pragma unroll
        for (int u = 0; u < 4 / Unit; ++u)
            if (in(u)) copy_async<Unit * sizeof(E)>(tile_row + at0 + step(u), row + step(u));
    }
    template <typename E>
    __device__ __forceinline__ Quad get(const E* tile_row) const {
        Quad q;
        if constexpr (Unit == 1) {
#pragma unroll
            for (int p = 0; p < 2; ++p)
                q.v[p] = pair_of(load(tile_row + at0 + step(2 * p)), load(tile_row + at0 + step(2 * p + 1)));
        } else {
            using Raw = typename Packed<E, Unit>::Raw;
            Raw raw[4 / Unit];
#pragma unroll
            for (int u = 0; u < 4 / Unit; ++u) raw[u] = *reinterpret_cast<const Raw*>(tile_row + at0 + step(u));
#pragma unroll
            for (int p = 0; p < 2; ++p)
                q.v[p] = PairOf<E>::unpack(reinterpret_cast<const uint32_t*>(raw) + p * (sizeof(E) / 2));
        }
        return q;
    }
    // A thread's channels of a row in global memory, as they lie there; `row` at its first
    // channel.  Loaded to stay in L2, for it will be read again.
    template <typename E>
    struct Rows {
        alignas(16) uint32_t words[sizeof(E) == 4 || Unit == 1 ? 4 : 2];
    };
    template <typename E>
    __device__ __forceinline__ Rows<E> read(const E* row) const {
        Rows<E> r = {};
#pragma unroll
        for (int u = 0; u < 4 / Unit; ++u)
            if (in(u)) {
                if constexpr (Unit == 1) {
                    if constexpr (sizeof(E) == 4)
                        r.words[u] = __ldg(reinterpret_cast<const uint32_t*>(row + step(u)));
                    else
                        r.words[u] = __ldg(reinterpret_cast<const unsigned short*>(row + step(u)));
                } else {
                    using Raw = typename Packed<E, Unit>::Raw;
                    *reinterpret_cast<Raw*>(r.words + u * (Unit * sizeof(E) / 4)) =
                        __ldg(reinterpret_cast<const Raw*>(row + step(u)));
                }
            }
        return r;
    }
    template <typename E>
    __device__ __forceinline__ Quad unpack(const Rows<E>& r) const {
        Quad q;
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            if constexpr (Unit == 1 && sizeof(E) == 2) {
                const uint32_t word = r.words[2 * p] | r.words[2 * p + 1] << 16;
                q.v[p] = PairOf<E>::unpack(&word);
            } else {
                q.v[p] = PairOf<E>::unpack(r.words + p * (sizeof(E) / 2));
            }
        }
        return q;
    }
    template <typename E>
    __device__ __forceinline__ void put(E* row, const Quad& q) const {
        if constexpr (Unit == 1) {
#pragma unroll
            for (int p = 0; p < 2; ++p) {
                const float2 f = parts(q.v[p]);
                if (in(2 * p)) store(row + step(2 * p), f.x);
                if (in(2 * p + 1)) store(row + step(2 * p + 1), f.y);
            }
        } else {
            using Raw = typename Packed<E, Unit>::Raw;
            Raw raw[4 / Unit];
#pragma unroll
            for (int p = 0; p < 2; ++p)
                PairOf<E>::pack(q.v[p], reinterpret_cast<uint32_t*>(raw) + p * (sizeof(E) / 2));
#pragma unroll
            for (int u = 0; u < 4 / Unit; ++u)
                if (in(u)) __stcs(reinterpret_cast<Raw*>(row + step(u)), raw[u]);
        }
    }
    // Column of element e of the four.
    static __device__ __forceinline__ constexpr uint32_t offset(int e) { return step(e / Unit) + e % Unit; }
    // Of a row in global memory, one element at a time; zero where there is none.
    template <typename E>
    __device__ __forceinline__ Quad get_row(const E* row) const {
        float f[4];
#pragma unroll
        for (int e = 0; e < 4; ++e) f[e] = row && c + offset(e) < channels ? load(row + c + offset(e)) : 0.0f;
        Quad q;
        q.v[0] = pair_of(f[0], f[1]), q.v[1] = pair_of(f[2], f[3]);
        return q;
    }
    __device__ __forceinline__ Quad get_row(const float* rows, uint32_t row) const {
        return get_row(rows ? rows + (size_t)row * channels : nullptr);
    }
    __device__ __forceinline__ void put_row(float* rows, uint32_t row, const Quad& q) const {
        float* p = rows + (size_t)row * channels + c;
        const float2 x = parts(q.v[0]), y = parts(q.v[1]);
        const float f[4] = {x.x, x.y, y.x, y.y};
#pragma unroll
        for (int e = 0; e < 4; ++e)
            if (c + offset(e) < channels) p[offset(e)] = f[e];
    }
    // A row of float in shared memory, this thread's columns.
    __device__ __forceinline__ Quad get_shared(const float* row) const { return get(row); }
    __device__ __forceinline__ void put_shared(float* row, const Quad& q) const {
        const float2 x = parts(q.v[0]), y = parts(q.v[1]);
        const float f[4] = {x.x, x.y, y.x, y.y};
        if constexpr (Unit == 4) {
            *reinterpret_cast<float4*>(row + at0) = make_float4(f[0], f[1], f[2], f[3]);
        } else {
#pragma unroll
            for (int e = 0; e < 4; ++e) row[at0 + offset(e)] = f[e];
        }
    }
};

// 16-bit elements of rows that no aligned copy reaches, on their way from
// global to shared memory through registers.
template <int Length>
struct Pending {
    unsigned short v[Length][4];
    template <typename E>
    __device__ __forceinline__ void read(const Columns<1>& col, int j, const E* row) {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            if (col.in(u)) v[j][u] = __ldcs(reinterpret_cast<const unsigned short*>(row + col.step(u)));
    }
    template <typename E>
    __device__ __forceinline__ void write(const Columns<1>& col, int j, E* tile_row) const {
#pragma unroll
        for (int u = 0; u < 4; ++u)
            reinterpret_cast<unsigned short*>(tile_row)[col.at0 + col.step(u)] = v[j][u];
    }
};

// Stories without a token keep their initial (forward) or final (backward) value.
__device__ __forceinline__ void copy_empty(const LeoB200StoryTables& t, uint32_t channels, uint32_t c,
                                           const float* from, float* to) {
    if (c >= channels) return;
    for (uint32_t e = t.full; e < t.stories; ++e) {
        const size_t at = (size_t)t.order[e] * channels + c;
        to[at] = from ? from[at] : 0.0f;
    }
}

template <typename T, typename G, int Unit, bool Shared, bool Backward>
__global__ void __launch_bounds__(Shape<T, G, Shared, Backward>::kThreads, 1) scan_kernel(const __grid_constant__ ScanArgs a) {
    using S = Shape<T, G, Shared, Backward>;
    constexpr int Length = S::kSegment;
    constexpr uint32_t kTile = S::kTile;
    constexpr bool Tiled = Unit == 4;
    constexpr int kStages = S::kStages, kTeams = S::kTeams;
    extern __shared__ __align__(128) unsigned char dynamic[];
    typename S::Control& control = *reinterpret_cast<typename S::Control*>(dynamic + kStages * S::kStage);
    const uint32_t block_warp = threadIdx.x >> 5;
    const uint32_t total = a.tiles * a.groups;
    const auto work_of = [&](uint32_t ticket) {
        Work w{0, kNone, 0, 0, 0, 0, 0, 0};
        if (ticket >= total) return w;
        const uint32_t place = ticket / a.groups;
        const uint4* entry = reinterpret_cast<const uint4*>(a.schedule + place);
        const uint4 x = __ldg(entry), y = __ldg(entry + 1);  // first, count, tile, kept; holder, onward
        return Work{x.x, x.y, x.z, ticket - place * a.groups, y.x, x.w, y.y, 0};
    };
    // The first tickets: one if there is a block for each, or a few, drawn one
    // after the other so that the blocks take turns: a block that held the next
    // three in a row would keep its neighbours waiting for its third.
    const bool one_each = gridDim.x == total;
    if (threadIdx.x == 0) {
        uint32_t t = a.tiles == 1 ? blockIdx.x : atomicAdd(a.scratch.ticket, 1u) + 1u;
        control.ring[0] = work_of(t);
#pragma unroll
        for (int j = 1; j < S::kAhead; ++j) {
            if (!one_each) t = atomicAdd(a.scratch.ticket + (t == kNone), 1u) + 1u;  // after the one before
            control.ring[j] = work_of(one_each ? total : t);
        }
        if constexpr (Tiled) {
            for (int j = 0; j < 4 * kWarps; ++j)
                asm volatile("mbarrier.init.shared.b64 [%0], 1;" ::"r"(
                    (uint32_t)__cvta_generic_to_shared(&control.landed[0][0] + j))
                             : "memory");
            asm volatile("fence.mbarrier_init.release.cluster;" ::: "memory");
        }
    }
    __syncthreads();
    const auto work_at = [&](uint32_t i) -> const Work& { return control.ring[i & 7u]; };

    if (block_warp < S::kFirstComposer) {
        // ------------------------------------------------ the teams that map and write, tiles in turn
        const uint32_t team = block_warp / kWarps, warp = block_warp % kWarps;
        const uint32_t lane = threadIdx.x & 31u, segment = warp * 2 + (lane >> 4);
        const auto stage = [&](uint32_t i) { return dynamic + (i % kStages) * S::kStage; };
        const auto stage_x = [&](uint32_t i, uint32_t seg) {
            return reinterpret_cast<T*>(stage(i)) + seg * Length * kColumns;
        };
        const auto stage_s = [&](uint32_t i, uint32_t seg) {
            return reinterpret_cast<T*>(stage(i)) + (kTile + seg * Length) * kColumns;
        };
        const auto stage_a = [&](uint32_t i, uint32_t seg) {
            return reinterpret_cast<G*>(stage(i) + (size_t)(Backward ? 2 : 1) * kTile * kColumns * sizeof(T)) +
                   seg * Length * kColumns;
        };
        constexpr bool Pends = Unit == 1 && sizeof(T) == 2, GatePends = Unit == 1 && sizeof(G) == 2 && !Shared;
        Pending<Pends ? Length : 1> pending_x, pending_s;
        Pending<GatePends ? Length : 1> pending_a;
        (void)pending_x, (void)pending_s, (void)pending_a;
        // What the issue before left in registers.
        const auto settle = [&](uint32_t i) {
            if constexpr (Pends) {
                const Columns<1> col(0, a.channels);
#pragma unroll
                for (int j = 0; j < Length; ++j) {
                    pending_x.write(col, j, stage_x(i, segment) + j * kColumns);
                    if constexpr (Backward) pending_s.write(col, j, stage_s(i, segment) + j * kColumns);
                    if constexpr (GatePends) pending_a.write(col, j, stage_a(i, segment) + j * kColumns);
                }
            }
        };
        // Tokens of the thread's segment.
        const auto tokens_of = [&](const Work& work) {
            return max(min((int)work.count - (int)segment * Length, Length), 0);
        };
        const auto issue = [&](uint32_t i) -> StoryBits {
            StoryBits bits{};
            const Work& work = work_at(i);
            if (Pends && i >= kTeams) settle(i - kTeams);
            if (work.count != kNone) {
                const uint32_t first = work.first + segment * Length, group = work.group;
                const int count = tokens_of(work);
                if (count) bits = story_bits(a.tables, first);
                if constexpr (Tiled) {
                    // The warp's stage was read by its own lanes only.
                    __syncwarp();
                    if (lane == 0) {
                        uint64_t* barrier = &control.landed[i % kStages][warp];
                        const uint32_t token = work.first + warp * 2 * Length;
                        const bool any = warp * 2 * Length < work.count;  // if not, the barrier still turns
                        expect_bytes(barrier, any ? 2 * Length * S::kRow : 0);
                        if (any) {
                            load_tile(stage_x(i, 2 * warp), &a.drive_map, group * kColumns, token, barrier);
                            if constexpr (Backward)
                                load_tile(stage_s(i, 2 * warp), &a.grad_map, group * kColumns, token, barrier);
                            if constexpr (!Shared)
                                load_tile(stage_a(i, 2 * warp), &a.decay_map, group * kColumns, token, barrier);
                        }
                    }
                } else {
                    const Columns<Unit> col(group, a.channels);
                    const T* x = static_cast<const T*>(a.drive) + (int64_t)first * a.drive_stride + col.c;
                    const T* s = static_cast<const T*>(a.grad_states) + (int64_t)first * a.grad_states_stride + col.c;
                    const G* g = static_cast<const G*>(a.decay) + (int64_t)first * a.decay_stride + col.c;
#pragma unroll
                    for (int j = 0; j < Length; ++j)
                        if (j < count) {
                            if constexpr (Pends) {
                                pending_x.read(col, j, x + j * a.drive_stride);
                                if constexpr (Backward) pending_s.read(col, j, s + j * a.grad_states_stride);
                            } else {
                                col.copy(stage_x(i, segment) + j * kColumns, x + j * a.drive_stride);
                                if constexpr (Backward)
                                    col.copy(stage_s(i, segment) + j * kColumns, s + j * a.grad_states_stride);
                            }
                            if constexpr (GatePends)
                                pending_a.read(col, j, g + j * a.decay_stride);
                            else if constexpr (!Shared)
                                col.copy(stage_a(i, segment) + j * kColumns, g + j * a.decay_stride);
                        }
                }
            }
            if constexpr (!Tiled) asm volatile("cp.async.commit_group;" ::: "memory");
            return bits;
        };
        // Waits for the loads of tile i, those of tile i + 1 being issued.
        const auto landed = [&](uint32_t i) {
            if constexpr (Tiled) {
                wait_landed(&control.landed[i % kStages][warp], i / kStages & 1u);
            } else {
                asm volatile("cp.async.wait_group 1;" ::: "memory");
            }
        };
        const auto map = [&](uint32_t i, const StoryBits& bits) {
            const Work& work = work_at(i);
            landed(i);
            const Columns<Unit> col(work.group, a.channels);
            const Segment s = segment_of(bits, work.first + segment * Length, tokens_of(work));
            const T* x = stage_x(i, segment);
            const T* sp = stage_s(i, segment);
            const G* ap = stage_a(i, segment);
            Product4 A;
            Quad H, M, gate;
            if constexpr (Shared) gate = col.get_row(static_cast<const G*>(a.decay));
            const auto forward = [&](int j) {
                if constexpr (!Shared) gate = col.get(ap + j * kColumns);
                const Quad v = col.get(x + j * kColumns);
#pragma unroll
                for (int q = 0; q < 2; ++q) H.v[q] = fma2(gate.v[q], H.v[q], v.v[q]);
                if constexpr (!Shared) A.times(gate);
            };
            const auto backward = [&](int j) {
                if constexpr (!Shared) gate = col.get(ap + j * kColumns);
                const Quad v = col.get(sp + j * kColumns);
#pragma unroll
                for (int q = 0; q < 2; ++q) M.v[q] = mul2(gate.v[q], add2(v.v[q], M.v[q]));
            };
            if (s.count == Length && (s.starts | s.ends) == 0) {
#pragma unroll
                for (int j = 0; j < Length; ++j) forward(j);
                if constexpr (Backward) {
#pragma unroll
                    for (int j = Length - 1; j >= 0; --j) backward(j);
                }
            } else {
#pragma unroll 1
                for (int j = 0; j < s.count; ++j) {
                    if (s.starts >> j & 1u) H = col.get_row(a.initial, story_starting(a.tables, s, j));
                    forward(j);
                }
                if constexpr (Backward) {
#pragma unroll 1
                    for (int j = s.count - 1; j >= 0; --j) {
                        if (s.ends >> j & 1u) M = col.get_row(a.grad_final, story_ending(a.tables, s, j));
                        backward(j);
                    }
                }
            }
            typename S::Maps& m = control.maps[i & 1u];
#pragma unroll
            for (int q = 0; q < (Shared ? 0 : 2); ++q) {
                const float2 hi = parts(A.hi[q]), lo = parts(A.lo[q]);
                float2* row = m.A[Shared ? 0 : segment] + col.at0;
                if constexpr (Unit == 1) {
                    row[col.offset(2 * q)] = make_float2(hi.x, lo.x);
                    row[col.offset(2 * q + 1)] = make_float2(hi.y, lo.y);
                } else {
                    *reinterpret_cast<float4*>(row + col.offset(2 * q)) = make_float4(hi.x, lo.x, hi.y, lo.y);
                }
            }
            col.put_shared(m.H[segment], H);
            if constexpr (Backward) col.put_shared(m.M[segment], M);
            if ((lane & 15u) == 0) m.starts[segment] = s.starts != 0, m.ends[segment] = s.ends != 0;
            arrive_at<kMapped>(i & 1u);
        };
        const auto write = [&](uint32_t i, const StoryBits& bits) {
            const Work& work = work_at(i);
            const Columns<Unit> col(work.group, a.channels);
            const uint32_t first = work.first + segment * Length;
            const Segment s = segment_of(bits, first, tokens_of(work));
            const T* x = stage_x(i, segment);
            const T* sp = stage_s(i, segment);
            const G* ap = stage_a(i, segment);
            const typename S::Maps& m = control.maps[i & 1u];
            Quad h = col.get_shared(m.H[segment]), gate;
            if constexpr (Shared) gate = col.get_row(static_cast<const G*>(a.decay));
            const size_t row = (size_t)first * a.channels + col.c;
            const bool plain = s.count == Length && (s.starts | s.ends) == 0;
            if constexpr (!Backward) {
                T* out = static_cast<T*>(a.states) + row;
                const auto step = [&](int j) {
                    if constexpr (!Shared) gate = col.get(ap + j * kColumns);
                    const Quad v = col.get(x + j * kColumns);
#pragma unroll
                    for (int q = 0; q < 2; ++q) h.v[q] = fma2(gate.v[q], h.v[q], v.v[q]);
                    col.put(out, h);
                    out += a.channels;
                };
                if (plain) {
#pragma unroll
                    for (int j = 0; j < Length; ++j) step(j);
                } else {
#pragma unroll 1
                    for (int j = 0; j < s.count; ++j) {
                        if (s.starts >> j & 1u) h = col.get_row(a.initial, story_starting(a.tables, s, j));
                        step(j);
                        if (s.ends >> j & 1u) col.put_row(a.final_states, story_ending(a.tables, s, j), h);
                    }
                }
            } else {
                // The state before each token, then the slopes from the right.
                Quad previous[Length];
#pragma unroll
                for (int j = 0; j < Length; ++j) {
                    if (!plain && (s.starts >> j & 1u)) h = col.get_row(a.initial, story_starting(a.tables, s, j));
                    if constexpr (!Shared) gate = col.get(ap + j * kColumns);
                    previous[j] = h;
                    const Quad v = col.get(x + j * kColumns);
#pragma unroll
                    for (int q = 0; q < 2; ++q) h.v[q] = fma2(gate.v[q], h.v[q], v.v[q]);
                }
                Quad n = col.get_shared(m.M[segment]), sum;
                T* out = static_cast<T*>(a.grad_drive) + row + (size_t)(Length - 1) * a.channels;
                G* out_gate = static_cast<G*>(a.grad_decay) + (Shared ? 0 : row + (size_t)(Length - 1) * a.channels);
#pragma unroll
                for (int j = Length - 1; j >= 0; --j) {
                    if (plain || j < s.count) {
                        if (!plain && (s.ends >> j & 1u))
                            n = col.get_row(a.grad_final, story_ending(a.tables, s, j));
                        if constexpr (!Shared) gate = col.get(ap + j * kColumns);
                        const Quad v = col.get(sp + j * kColumns);
                        Quad slope, term;
#pragma unroll
                        for (int q = 0; q < 2; ++q) {
                            slope.v[q] = add2(v.v[q], n.v[q]);
                            term.v[q] = mul2(slope.v[q], previous[j].v[q]);
                            n.v[q] = mul2(gate.v[q], slope.v[q]);
                            if constexpr (Shared) sum.v[q] = add2(sum.v[q], term.v[q]);
                        }
                        col.put(out, slope);
                        if constexpr (!Shared) col.put(out_gate, term);
                        if (!plain && a.grad_initial && (s.starts >> j & 1u))
                            col.put_row(a.grad_initial, story_starting(a.tables, s, j), n);
                    }
                    out -= a.channels;
                    if constexpr (!Shared) out_gate -= a.channels;
                }
                if constexpr (Shared) col.put_shared(control.sums[i & 1u][segment], sum);
            }
        };

        if constexpr (kTeams == 1) {
            // What is done between the maps of a tile and its writing is the map of the next one.
            StoryBits bits0 = issue(0), bits1 = issue(1);
            if (work_at(0).count != kNone) map(0, bits0);
            for (uint32_t i = 0; work_at(i).count != kNone; ++i) {
                const StoryBits bits2 = issue(i + 2);
                if (work_at(i + 1).count != kNone) map(i + 1, bits1);
                sync_of<kComposed>(i & 1u);
                write(i, bits0);
                bits0 = bits1;
                bits1 = bits2;
            }
        } else {
            // The other team's work fills the time between.
            StoryBits bits = issue(team);
            for (uint32_t i = team; work_at(i).count != kNone; i += 2) {
                const StoryBits bits_next = issue(i + 2);
                map(i, bits);
                sync_of<kComposed>(i & 1u);
                write(i, bits);
                bits = bits_next;
            }
        }
        if constexpr (Backward && Shared) arrive_at<kMapped>(team);  // the last sums are written
    } else if (block_warp >= S::kFirstScout) {
        // ------------------------------------------------ the warps that scout
        // Everything that is read from memory between tiles is read here, up to two
        // tiles ahead: beside a load in flight the warps that compose would wait for
        // it with every read of shared memory.  A lane takes half the slots of a
        // channel; its partner is 16 lanes away.
        constexpr int Direction = Backward ? -1 : 1;
        const uint32_t lane = threadIdx.x & 31u, half = lane >> 4;
        const uint32_t k = (block_warp - S::kFirstScout) * 16 + (lane & 15u);
        const bool leader = threadIdx.x == 32 * S::kFirstScout;
        const auto draw = [&] {
            uint32_t t = kNone - 1u;
            if (leader && !one_each)  // no use of the answer here, so that nothing waits for it
                asm volatile("atom.relaxed.gpu.global.add.u32 %0, [%1], 1;" : "=r"(t) : "l"(a.scratch.ticket) : "memory");
            return t;
        };
        uint32_t drawn = draw();
        for (uint32_t i = 0;; ++i) {
            const Work work = work_at(i);
            if (work.count == kNone) break;
            // The schedule's entry of the ticket drawn a turn ago, and another ticket.
            const uint32_t ticket = drawn + 1u, place = min(ticket / a.groups, a.tiles - 1u);
            const uint4* entry = reinterpret_cast<const uint4*>(a.schedule + place);
            const uint4 x = __ldg(entry), y = __ldg(entry + 1);  // first, count, tile, kept; holder, onward
            drawn = draw();
            const uint32_t c = work.group * kColumns + k;
            const bool active = c < a.channels;
            const Lookback<Direction> back(work.tile, work.holder);
            Slot slots[8];
            if (back.maps >= 0 && active) back.load(a.scratch.slots, a.channels, c, (int)half, slots);
            float kept = 0.0f;
            if (Backward && active && half == 0 && work.count > 0)
                kept = __ldcs(a.carries + (size_t)work.kept * a.channels + c);
            float carry = 0.0f;
            if (back.maps >= 0) {
                // Forward, the halves are composed at the same time, since tiles wait for the state; backward, with
                // more to do elsewhere, one after the other, which needs no product (20,480 tokens x 4,096: 144 and
                // 266 us; 146 and 271 us the other way round).
                float A = 1.0f, H = 0.0f;
                const auto look = [&] {
                    if constexpr (Direction > 0)
                        return back.compose(slots, (int)half, A, H);
                    else
                        return back.there(slots, (int)half);
                };
                bool there = !active || look(), gave_up = false;
                for (uint32_t n = 0; !__all_sync(kNone, there); ++n) {
                    if (n >= kSpinLimit) {
                        if (lane == 0) atomicExch(&g_gave_up, 1u);
                        gave_up = true;
                        break;
                    }
                    if (active) {
                        back.load(a.scratch.slots, a.channels, c, (int)half, slots);
                        there = look();
                    }
                }
                if constexpr (Direction > 0) {
                    const float other_A = __shfl_xor_sync(kNone, A, 16), other_H = __shfl_xor_sync(kNone, H, 16);
                    // the far half's map of the near half's state; one slot is the state itself
                    if (back.maps < 8) {
                        carry = half ? other_H : H;
                    } else {
                        carry = half ? fmaf(A, other_H, H) : fmaf(other_A, H, other_H);
                        if (__any_sync(kNone, carry != carry)) {  // an infinite state, perhaps, times 0
                            if (half) A = back.product(slots);
                            const float kept_A = __shfl_xor_sync(kNone, A, 16);
                            carry = half ? fmaf(A, other_H, H) : fmaf(kept_A, H, other_H);
                        }
                    }
                } else {
                    if (active && half == 0) carry = back.run(slots, 0, 0.0f);
                    carry = __shfl_xor_sync(kNone, carry, 16);
                    if (active && half) carry = back.run(slots, 1, carry);
                }
                if (gave_up) carry = CUDART_NAN_F;
            }
            if (i >= 2) sync_of<kTaken>(i & 1u);
            if (half)
                control.scouted[i & 1u][0][k] = carry;
            else if constexpr (Backward)
                control.scouted[i & 1u][1][k] = kept;
            if (leader)
                control.ring[(i + S::kAhead) & 7u] =
                    Work{x.x, !one_each && ticket < total ? x.y : kNone, x.z, ticket - place * a.groups, y.x, x.w, y.y, 0};
            arrive_at<kScouted>(i & 1u);
        }
    } else {
        // ------------------------------------------------ the warps that compose
        // A lane takes half the segments of a channel, the nearer ones in the
        // direction of the scan first; its partner is 16 lanes away.
        constexpr int kHalf = kSegments / 2;
        const uint32_t lane = threadIdx.x & 31u, half = lane >> 4, k = (block_warp - S::kFirstComposer) * 16 + (lane & 15u);
        // A shared gate's product over a segment's tokens.
        const auto power = [&](uint32_t channel, int count) {
            float2 product = make_float2(1.0f, 0.0f);
            const float2 gate = make_float2(channel < a.channels ? load(static_cast<const G*>(a.decay) + channel) : 0.0f, 0.0f);
            for (int j = 0; j < count; ++j) product = product_of(product, gate);
            return product;
        };
        float2 whole = make_float2(1.0f, 0.0f);  // of a whole segment
        uint32_t whole_of = kNone;               // its channel
        (void)power, (void)whole, (void)whole_of;
        const auto add_sums = [&](uint32_t i, uint2 work) {  // (tile, group)
            const uint32_t c = work.y * kColumns + k;
            float sum = 0.0f;
#pragma unroll
            for (int w = 0; w < kSegments; ++w) sum += control.sums[i & 1u][w][k];
            if (c >= a.channels || half) return;
            if (a.tiles == 1)
                store(static_cast<G*>(a.grad_decay) + c, sum);
            else
                a.scratch.partials[(size_t)work.x * a.channels + c] = sum;
        };
        (void)add_sums;
        uint32_t i = 0;
        uint2 before1 = make_uint2(kNone, 0), before2 = before1;  // the last two tiles
        for (;; ++i) {
            const Work work = work_at(i);
            if (work.count == kNone) break;
            const uint32_t tile = work.tile, c = work.group * kColumns + k;
            const bool active = c < a.channels;
            sync_of<kMapped>(i & 1u);
            typename S::Maps& m = control.maps[i & 1u];
            if constexpr (Backward && Shared)
                if (before2.x != kNone) add_sums(i, before2);

            // The map of this half of the tile, then of the tile, in the direction of the scan.
            const uint2 cut_bytes =
                reinterpret_cast<const uint2*>(Backward ? m.ends : m.starts)[Backward ? 1 - half : half];
            const auto segment = [&](int j) { return (Backward ? kSegments - 1 - j : j) + (Backward ? -1 : 1) * (int)half * kHalf; };
            const auto cut_at = [&](int j) {  // of this half
                const int byte = Backward ? kHalf - 1 - j : j;
                return ((byte < 4 ? cut_bytes.x : cut_bytes.y) >> (byte & 3) * 8 & 1u) != 0;
            };
            if (Shared && whole_of != c) {
                whole = power(c, Length);
                whole_of = c;
            }
            const auto product_at = [&](int w) {
                if constexpr (Shared) {
                    const int count = max(min((int)work.count - w * Length, Length), 0);
                    return count == Length ? whole : power(c, count);
                } else {
                    return m.A[w][k];
                }
            };
            float2 product = make_float2(1.0f, 0.0f);
            float sum = 0.0f, A[kHalf], v[kHalf];
            bool zero = false;
#pragma unroll
            for (int j = 0; j < kHalf; ++j) {
                const int w = segment(j);
                const float2 p = product_at(w);
                A[j] = value_of(p);
                v[j] = Backward ? m.M[Backward ? w : 0][k] : m.H[w][k];
                sum = cut_at(j) ? v[j] : fmaf(A[j], sum, v[j]);
                product = product_of(product, p);
                zero |= A[j] == 0.0f;
            }
            if (product.x == 0.0f && !zero) product.x = smallest(product.x);
            const bool cut = (cut_bytes.x | cut_bytes.y) != 0;
            const bool other_cut = __shfl_xor_sync(kNone, cut, 16);
            const float other_sum = __shfl_xor_sync(kNone, sum, 16);
            const float2 other = make_float2(__shfl_xor_sync(kNone, product.x, 16), __shfl_xor_sync(kNone, product.y, 16));
            const bool cuts = cut || other_cut;
            // of the near and the far half
            const float near_A = value_of(half ? other : product), near_sum = half ? other_sum : sum;
            const bool near_cut = half ? other_cut : cut, far_cut = half ? cut : other_cut;
            const float far_A = value_of(half ? product : other), far_sum = half ? sum : other_sum;
            const float both = near_A * far_A;
            const float tile_A =
                both == 0.0f && near_A != 0.0f && far_A != 0.0f ? smallest(both) : value_of(product_of(product, other));
            const float tile_sum = far_cut ? far_sum : fmaf(far_A, near_sum, far_sum);
            const bool state_tile = Backward ? tile % kGroup == 0 : (tile + 1) % kGroup == 0;
            const bool writes = active && work.onward && half == 0;
            Slot* mine = a.scratch.slots + (size_t)tile * a.channels + c;
            if (writes && (cuts || !state_tile)) write_slot(mine, tile_A, tile_sum);

            sync_of<kScouted>(i & 1u);
            const float carry = control.scouted[i & 1u][0][k];
            const float kept = Backward ? control.scouted[i & 1u][Backward ? 1 : 0][k] : 0.0f;
            arrive_at<kTaken>(i & 1u);
            if (writes && !cuts && state_tile) write_slot(mine, 0.0f, fmaf(tile_A, carry, tile_sum));

            // The value before each segment, in place of its map.
            float before = half ? (near_cut ? near_sum : fmaf(near_A, carry, near_sum)) : carry;
#pragma unroll
            for (int j = 0; j < kHalf; ++j) {
                const int w = segment(j);
                if constexpr (Backward) {
                    m.M[w][k] = before;
                } else {
                    m.H[w][k] = before;
                    if (a.carries && active && w % (kKept / Length) == 0 && (uint32_t)w * Length < work.count)
                        a.carries[(size_t)(work.kept + w / (kKept / Length)) * a.channels + c] = before;
                }
                before = cut_at(j) ? v[j] : fmaf(A[j], before, v[j]);
            }
            if constexpr (Backward) {
                // The state before each segment: this lane's half from the right is the other one from the left.
                const uint2 starts = reinterpret_cast<const uint2*>(m.starts)[1 - half];
                float h[kHalf];
                float state = 0.0f;
#pragma unroll
                for (int j = 0; j < kHalf; ++j) h[j] = m.H[segment(kHalf - 1 - j)][k];
                const auto start_at = [&](int j) { return ((j < 4 ? starts.x : starts.y) >> (j & 3) * 8 & 1u) != 0; };
#pragma unroll
                for (int j = 0; j < kHalf; ++j) state = start_at(j) ? h[j] : fmaf(A[kHalf - 1 - j], state, h[j]);
                // Lanes of half 1 hold the segments on the left, and pass the state after them on.
                const bool left_cut = (starts.x | starts.y) != 0;
                const float after = half ? (left_cut ? state : fmaf(far_A, kept, state)) : 0.0f;
                const float from_left = __shfl_xor_sync(kNone, after, 16);
                float at = half ? kept : from_left;
#pragma unroll
                for (int j = 0; j < kHalf; ++j) {
                    m.H[segment(kHalf - 1 - j)][k] = at;
                    at = start_at(j) ? h[j] : fmaf(A[kHalf - 1 - j], at, h[j]);
                }
            }
            arrive_at<kComposed>(i & 1u);
            if (tile == 0 && a.tables.full < a.tables.stories && half == 0) {
                if constexpr (!Backward)
                    copy_empty(a.tables, a.channels, c, a.initial, a.final_states);
                else if (a.grad_initial)
                    copy_empty(a.tables, a.channels, c, a.grad_final, a.grad_initial);
            }
            before2 = before1;
            before1 = make_uint2(tile, work.group);
        }
        if constexpr (Backward && Shared) {
            sync_of<kMapped>(0);
            if constexpr (kTeams == 2) sync_of<kMapped>(1);
            if (before2.x != kNone) add_sums(i, before2);
            if (before1.x != kNone) add_sums(i + 1, before1);
        }
    }
}

// Few stories side by side: the tiles of one are then in the works at the same
// time, and each would wait for its neighbours.  Their maps are found first, in
// a pass over the inputs, and joined to the states after every tile; then the
// tiles are written by a block each, which reads the inputs once more and waits
// for nothing.  One document of 65,537 tokens x 257 channels, float32 with one gate
// a channel: 66 us forward and 90 us backward, 104 and 137 us in one pass (21 and 31 us
// at the rate of a copy; rows of 257 are read and written an element at a time).

// Calls body(true_type) for a segment that is whole and inside a story, as most
// are: nothing is asked of its tokens there.  body(false_type) for the others.
template <typename Body>
__device__ __forceinline__ void with_plain(const Segment& s, int length, Body&& body) {
    if (s.count == length && (s.starts | s.ends) == 0)
        body(std::true_type{});
    else
        body(std::false_type{});
}

// The map of a tile, the work divided as above, every row read at once.
template <typename T, typename G, int Unit, bool Shared, bool Backward>
__global__ void __launch_bounds__(16 * kSegments) scan_map_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int Length = LEO_B200_TILE_TOKENS / kSegments;
    __shared__ __align__(16) float2 products[kSegments][kColumns];
    __shared__ __align__(16) float values[kSegments][kColumns];
    __shared__ uint32_t cuts[kSegments];
    const uint32_t place = blockIdx.x / a.groups, group = blockIdx.x - place * a.groups;
    const LeoB200StoryTile tile = a.schedule[place];
    const uint32_t segment = threadIdx.x >> 4, first = tile.first + segment * Length;
    const int count = max(min((int)tile.count - (int)segment * Length, Length), 0);
    const Columns<Unit> col(group, a.channels);
    const int64_t stride = Backward ? a.grad_states_stride : a.drive_stride;
    const T* x = (Backward ? static_cast<const T*>(a.grad_states) : static_cast<const T*>(a.drive)) +
                 (int64_t)first * stride + col.c;
    const G* g = static_cast<const G*>(a.decay) + (Shared ? 0 : (int64_t)first * a.decay_stride) + col.c;
    typename Columns<Unit>::template Rows<T> xs[Length];
    typename Columns<Unit>::template Rows<G> gs[Shared ? 1 : Length];
#pragma unroll
    for (int j = 0; j < Length; ++j)
        if (j < count) {
            xs[j] = col.read(x + j * stride);
            if constexpr (!Shared) gs[j] = col.read(g + j * a.decay_stride);
        }
    const StoryBits bits = count ? story_bits(a.tables, first) : StoryBits{};
    const Segment s = segment_of(bits, first, count);
    Quad value, gate;
    Product4 product;
    if constexpr (Shared) gate = col.get_row(static_cast<const G*>(a.decay));
    with_plain(s, Length, [&](auto plain) {
        constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
        for (int k = 0; k < Length; ++k) {
            const int j = Backward ? Length - 1 - k : k;
            if (kPlain || j < count) {
                if (!kPlain && ((Backward ? s.ends : s.starts) >> j & 1u))
                    value = Backward ? col.get_row(a.grad_final, story_ending(a.tables, s, j))
                                     : col.get_row(a.initial, story_starting(a.tables, s, j));
                if constexpr (!Shared) gate = col.unpack(gs[j]);
                const Quad v = col.unpack(xs[j]);
#pragma unroll
                for (int q = 0; q < 2; ++q)
                    value.v[q] = Backward ? mul2(gate.v[q], add2(v.v[q], value.v[q])) : fma2(gate.v[q], value.v[q], v.v[q]);
                product.times(gate);
            }
        }
    });
    col.put_shared(values[segment], value);
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float2 hi = parts(product.hi[q]), lo = parts(product.lo[q]);
        products[segment][col.at0 + col.offset(2 * q)] = make_float2(hi.x, lo.x);
        products[segment][col.at0 + col.offset(2 * q + 1)] = make_float2(hi.y, lo.y);
    }
    if ((threadIdx.x & 15u) == 0) cuts[segment] = Backward ? s.ends : s.starts;
    __syncthreads();
    const uint32_t c = group * kColumns + threadIdx.x;
    if (threadIdx.x >= kColumns || c >= a.channels) return;
    float2 all = make_float2(1.0f, 0.0f);
    float sum = 0.0f;
    bool cut = false;
#pragma unroll
    for (int k = 0; k < kSegments; ++k) {
        const int w = Backward ? kSegments - 1 - k : k;
        const float2 A = products[w][threadIdx.x];
        sum = cuts[w] ? values[w][threadIdx.x] : fmaf(value_of(A), sum, values[w][threadIdx.x]);
        all = product_of(all, A);
        cut |= cuts[w] != 0;
    }
    if (all.x == 0.0f) {
        all = make_float2(1.0f, 0.0f);
#pragma unroll 1
        for (int w = 0; w < kSegments; ++w) all = times(all, products[w][threadIdx.x]);
    }
    // A map that a story starts in has no product; all bits set say so.
    uint32_t low = __float_as_uint(value_of(all));
    if (low == kNone) low = 0x7fffffffu;
    if (cut) low = kNone;
    a.scratch.slots[(size_t)tile.tile * a.channels + c] = (Slot)__float_as_uint(sum) << 32 | low;
}

// The states after all tiles out of their maps: a lane a run of tiles of a
// channel, its maps composed first and then walked from the state before it.  The
// time is that of the trips to memory, so runs are short, and the first eight
// maps are read at once and kept.
constexpr uint32_t kJoinChannels = 8, kJoinRuns = 4;  // of a warp
template <bool Backward>
__global__ void __launch_bounds__(1024) scan_join_kernel(const __grid_constant__ ScanArgs a) {
    struct Map {
        float A = 1.0f, H = 0.0f;
        bool cut = false;  // a story starts inside: H is the state after it
        __device__ __forceinline__ void then(Slot s) {
            const float value = __uint_as_float((uint32_t)(s >> 32)), product = __uint_as_float((uint32_t)s);
            const bool here = (uint32_t)s == kNone;
            H = here ? value : fmaf(product, H, value);
            A = times(A, product);
            cut |= here;
        }
        __device__ __forceinline__ float of(float state) const { return cut ? H : fmaf(A, state, H); }
    };
    __shared__ float products[32][kJoinChannels], values[32][kJoinChannels];
    __shared__ bool cuts[32][kJoinChannels];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, k = lane % kJoinChannels, sub = lane / kJoinChannels;
    const uint32_t c = blockIdx.x * kJoinChannels + k, runs = 32 * kJoinRuns;
    const uint32_t run = (a.tiles + runs - 1) / runs, begin = min((warp * kJoinRuns + sub) * run, a.tiles);
    const uint32_t end = c < a.channels ? min(begin + run, a.tiles) : begin;
    const auto slot = [&](uint32_t i) {
        return a.scratch.slots + (size_t)(Backward ? a.tiles - 1 - i : i) * a.channels + c;
    };
    const auto read = [&](uint32_t from, Slot (&s)[8]) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (from + j < end) s[j] = *slot(from + j);
    };
    Slot held[8], more[8];
    read(begin, held);
    Map mine;
#pragma unroll
    for (uint32_t j = 0; j < 8; ++j)
        if (begin + j < end) mine.then(held[j]);
    for (uint32_t from = begin + 8; from < end; from += 8) {
        read(from, more);
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (from + j < end) mine.then(more[j]);
    }
    // The maps of the warp's runs before this one, and of all of them.
    Map before, all;
#pragma unroll
    for (uint32_t r = 0; r < kJoinRuns; ++r) {
        const uint32_t from = r * kJoinChannels + k;
        const float A = __shfl_sync(kNone, mine.A, from), H = __shfl_sync(kNone, mine.H, from);
        const bool cut = __shfl_sync(kNone, mine.cut, from);
        if (r == sub) before = all;
        all.H = cut ? H : fmaf(A, all.H, H);
        all.A = times(all.A, A);
        all.cut |= cut;
    }
    if (sub == 0) products[warp][k] = all.A, values[warp][k] = all.H, cuts[warp][k] = all.cut;
    __syncthreads();
    float state = 0.0f;
#pragma unroll 4
    for (uint32_t w = 0; w < warp; ++w) state = cuts[w][k] ? values[w][k] : fmaf(products[w][k], state, values[w][k]);
    if (sub) state = before.of(state);
    const auto walk = [&](uint32_t from, const Slot (&s)[8]) {
#pragma unroll
        for (uint32_t j = 0; j < 8; ++j)
            if (from + j < end) {
                Map m;
                m.then(s[j]);
                state = m.of(state);
                *slot(from + j) = (Slot)__float_as_uint(state) << 32;
            }
    };
    walk(begin, held);
    for (uint32_t from = begin + 8; from < end; from += 8) {
        read(from, more);
        walk(from, more);
    }
}

// The tiles themselves, the state before each in the slot of the tile before it.
// Nothing is waited for, so a block a tile keeps its tokens in registers and
// the SM's blocks hide one another's loads.
template <typename T, typename G, int Unit, bool Shared, bool Backward>
__global__ void __launch_bounds__(16 * kSegments, 2) scan_tile_kernel(const __grid_constant__ ScanArgs a) {
    constexpr int Length = LEO_B200_TILE_TOKENS / kSegments;
    __shared__ __align__(16) float products[kSegments][kColumns];
    __shared__ __align__(16) float states[kSegments][kColumns];                     // of a segment from zero, then before it
    __shared__ __align__(16) float values[Backward ? kSegments : 1][kColumns];  // the same from the right
    __shared__ bool starts[kSegments], ends[kSegments];
    const uint32_t place = blockIdx.x / a.groups, group = blockIdx.x - place * a.groups;
    const LeoB200StoryTile tile = a.schedule[place];
    const uint32_t segment = threadIdx.x >> 4, first = tile.first + segment * Length;
    const int count = max(min((int)tile.count - (int)segment * Length, Length), 0);
    const Columns<Unit> col(group, a.channels);
    typename Columns<Unit>::template Rows<T> xs[Length], ss[Backward ? Length : 1];
    typename Columns<Unit>::template Rows<G> gs[Shared ? 1 : Length];
    {
        const T* x = static_cast<const T*>(a.drive) + (int64_t)first * a.drive_stride + col.c;
        const T* s = static_cast<const T*>(a.grad_states) + (Backward ? (int64_t)first * a.grad_states_stride + col.c : 0);
        const G* g = static_cast<const G*>(a.decay) + (Shared ? 0 : (int64_t)first * a.decay_stride) + col.c;
#pragma unroll
        for (int j = 0; j < Length; ++j)
            if (j < count) {
                xs[j] = col.read(x + j * a.drive_stride);
                if constexpr (Backward) ss[j] = col.read(s + j * a.grad_states_stride);
                if constexpr (!Shared) gs[j] = col.read(g + j * a.decay_stride);
            }
    }
    // Of the threads that join the segments, a channel each: 64 from the left, and 64 more from the right.
    const uint32_t k = threadIdx.x % kColumns, c = group * kColumns + k, side = threadIdx.x / kColumns;
    const bool joins = side < (Backward ? 2 : 1), leftward = Backward && side == 0;
    float before = 0.0f;
    if (joins && c < a.channels) {
        if (Backward && !leftward)
            before = a.carries[(size_t)tile.kept * a.channels + c];
        else if (tile.holder != tile.tile)
            before = __uint_as_float((uint32_t)(
                a.scratch.slots[(size_t)(Backward ? tile.tile + 1 : tile.tile - 1) * a.channels + c] >> 32));
    }
    const StoryBits bits = count ? story_bits(a.tables, first) : StoryBits{};
    const Segment s = segment_of(bits, first, count);
    Quad h, n, gate;
    Product4 product;
    if constexpr (Shared) gate = col.get_row(static_cast<const G*>(a.decay));
    with_plain(s, Length, [&](auto plain) {
        constexpr bool kPlain = decltype(plain)::value;
#pragma unroll
        for (int j = 0; j < Length; ++j)
            if (kPlain || j < count) {
                if (!kPlain && (s.starts >> j & 1u)) h = col.get_row(a.initial, story_starting(a.tables, s, j));
                if constexpr (!Shared) gate = col.unpack(gs[j]);
                const Quad v = col.unpack(xs[j]);
#pragma unroll
                for (int q = 0; q < 2; ++q) h.v[q] = fma2(gate.v[q], h.v[q], v.v[q]);
                product.times(gate);
            }
        if constexpr (Backward) {
#pragma unroll
            for (int j = Length - 1; j >= 0; --j)
                if (kPlain || j < count) {
                    if (!kPlain && (s.ends >> j & 1u)) n = col.get_row(a.grad_final, story_ending(a.tables, s, j));
                    if constexpr (!Shared) gate = col.unpack(gs[j]);
                    const Quad v = col.unpack(ss[j]);
#pragma unroll
                    for (int q = 0; q < 2; ++q) n.v[q] = mul2(gate.v[q], add2(v.v[q], n.v[q]));
                }
        }
    });
    if constexpr (Backward) col.put_shared(values[segment], n);
    col.put_shared(states[segment], h);
    Quad A;
#pragma unroll
    for (int q = 0; q < 2; ++q) {
        const float2 hi = parts(product.hi[q]), lo = parts(product.lo[q]);
        A.v[q] = pair_of(value_of(make_float2(hi.x, lo.x)), value_of(make_float2(hi.y, lo.y)));
    }
    col.put_shared(products[segment], A);
    if ((threadIdx.x & 15u) == 0) starts[segment] = s.starts != 0, ends[segment] = s.ends != 0;
    __syncthreads();
    if (joins && !leftward) {
#pragma unroll
        for (int w = 0; w < kSegments; ++w) {
            const float v = states[w][k];
            states[w][k] = before;
            if constexpr (!Backward)
                if (a.carries && c < a.channels && w % (kKept / Length) == 0 && (uint32_t)w * Length < tile.count)
                    a.carries[(size_t)(tile.kept + w / (kKept / Length)) * a.channels + c] = before;
            before = starts[w] ? v : fmaf(products[w][k], before, v);
        }
    } else if (joins) {
#pragma unroll
        for (int w = kSegments - 1; w >= 0; --w) {
            const float v = values[Backward ? w : 0][k];
            values[Backward ? w : 0][k] = before;
            before = ends[w] ? v : fmaf(products[w][k], before, v);
        }
    }
    __syncthreads();
    const size_t row = (size_t)first * a.channels + col.c;
    h = col.get_shared(states[segment]);
    Quad sum;
    with_plain(s, Length, [&](auto plain) {
        constexpr bool kPlain = decltype(plain)::value;
        if constexpr (!Backward) {
            T* out = static_cast<T*>(a.states) + row;
#pragma unroll
            for (int j = 0; j < Length; ++j)
                if (kPlain || j < count) {
                    if (!kPlain && (s.starts >> j & 1u)) h = col.get_row(a.initial, story_starting(a.tables, s, j));
                    if constexpr (!Shared) gate = col.unpack(gs[j]);
                    const Quad v = col.unpack(xs[j]);
#pragma unroll
                    for (int q = 0; q < 2; ++q) h.v[q] = fma2(gate.v[q], h.v[q], v.v[q]);
                    col.put(out + (size_t)j * a.channels, h);
                    if (!kPlain && (s.ends >> j & 1u)) col.put_row(a.final_states, story_ending(a.tables, s, j), h);
                }
        } else {
            // The state before each token, then the slopes from the right.
            Quad previous[Length];
#pragma unroll
            for (int j = 0; j < Length; ++j)
                if (kPlain || j < count) {
                    if (!kPlain && (s.starts >> j & 1u)) h = col.get_row(a.initial, story_starting(a.tables, s, j));
                    if constexpr (!Shared) gate = col.unpack(gs[j]);
                    previous[j] = h;
                    const Quad v = col.unpack(xs[j]);
#pragma unroll
                    for (int q = 0; q < 2; ++q) h.v[q] = fma2(gate.v[q], h.v[q], v.v[q]);
                }
            n = col.get_shared(values[segment]);
            T* out = static_cast<T*>(a.grad_drive) + row;
            G* out_gate = static_cast<G*>(a.grad_decay) + (Shared ? 0 : row);
            (void)out_gate;
#pragma unroll
            for (int j = Length - 1; j >= 0; --j)
                if (kPlain || j < count) {
                    if (!kPlain && (s.ends >> j & 1u)) n = col.get_row(a.grad_final, story_ending(a.tables, s, j));
                    if constexpr (!Shared) gate = col.unpack(gs[j]);
                    const Quad v = col.unpack(ss[j]);
                    Quad slope, term;
#pragma unroll
                    for (int q = 0; q < 2; ++q) {
                        slope.v[q] = add2(v.v[q], n.v[q]);
                        term.v[q] = mul2(slope.v[q], previous[j].v[q]);
                        n.v[q] = mul2(gate.v[q], slope.v[q]);
                        if constexpr (Shared) sum.v[q] = add2(sum.v[q], term.v[q]);
                    }
                    col.put(out + (size_t)j * a.channels, slope);
                    if constexpr (!Shared) col.put(out_gate + (size_t)j * a.channels, term);
                    if (!kPlain && a.grad_initial && (s.starts >> j & 1u))
                        col.put_row(a.grad_initial, story_starting(a.tables, s, j), n);
                }
        }
    });
    if constexpr (Backward && Shared) {
        col.put_shared(states[segment], sum);  // only these threads' columns, which they have read
        __syncthreads();
        if (threadIdx.x < kColumns && c < a.channels) {
            float total = 0.0f;
#pragma unroll
            for (int w = 0; w < kSegments; ++w) total += states[w][k];
            a.scratch.partials[(size_t)tile.tile * a.channels + c] = total;
        }
    }
    if (tile.tile == 0 && a.tables.full < a.tables.stories && side == 0) {
        if constexpr (!Backward)
            copy_empty(a.tables, a.channels, c, a.initial, a.final_states);
        else if (a.grad_initial)
            copy_empty(a.tables, a.channels, c, a.grad_final, a.grad_initial);
    }
}

// The gradient of a shared row of gates: the tiles' sums in double, a column of
// 32 channels a block, every 32nd tile a warp.
template <typename G>
__global__ void __launch_bounds__(kReduceThreads) shared_decay_kernel(const float* partials, uint32_t tiles,
                                                                uint32_t channels, G* out) {
    __shared__ double sums[kReduceThreads / 32][32];
    const uint32_t lane = threadIdx.x & 31u, warp = threadIdx.x >> 5, c = blockIdx.x * 32 + lane;
    double sum = 0.0;
    if (c < channels)
#pragma unroll 8
        for (uint32_t t = warp; t < tiles; t += kReduceThreads / 32) sum += (double)partials[(size_t)t * channels + c];
    sums[warp][lane] = sum;
    __syncthreads();
    if (warp || c >= channels) return;
    for (uint32_t w = 1; w < kReduceThreads / 32; ++w) sum += sums[w][lane];
    store(out + c, (float)sum);
}

// One token of every lane: Unit neighbouring channels a thread.  Bound by memory
// (two reads, the state's read and write, one write a channel): 4,096 x 4,096 in
// bfloat16 with float32 gates move 268 MB in 43 us, 96 % of a copy's rate.
template <typename T, typename G, int Unit>
__global__ void __launch_bounds__(256)
    step_kernel(uint32_t lanes, uint32_t channels, const T* drive, int64_t drive_stride, const G* decay,
                int64_t decay_stride, float* state, int64_t state_stride, T* output) {
    const uint32_t units = channels / Unit;
    const uint64_t at = (uint64_t)blockIdx.x * 256 + threadIdx.x;
    if (at >= (uint64_t)lanes * units) return;
    const uint64_t lane = at >> 32 ? at / units : (uint32_t)at / units;
    const uint32_t c = (uint32_t)(at - lane * units) * Unit;
    const T* x = drive + (int64_t)lane * drive_stride + c;
    const G* g = decay + (int64_t)lane * decay_stride + c;
    float* h = state + (int64_t)lane * state_stride + c;
    T* out = output + lane * channels + c;
    if constexpr (Unit == 4) {
        using X = typename Packed<T, 4>::Raw;
        using A = typename Packed<G, 4>::Raw;
        X rx = __ldcs(reinterpret_cast<const X*>(x));
        const A ra = decay_stride ? __ldcs(reinterpret_cast<const A*>(g)) : __ldg(reinterpret_cast<const A*>(g));
        uint4 rh = *reinterpret_cast<const uint4*>(h);
        uint32_t* wh = reinterpret_cast<uint32_t*>(&rh);
        uint32_t* wx = reinterpret_cast<uint32_t*>(&rx);
#pragma unroll
        for (int p = 0; p < 2; ++p) {
            const Pair32 v = fma2(PairOf<G>::unpack(reinterpret_cast<const uint32_t*>(&ra) + p * (sizeof(G) / 2)),
                                  PairOf<float>::unpack(wh + 2 * p), PairOf<T>::unpack(wx + p * (sizeof(T) / 2)));
            PairOf<float>::pack(v, wh + 2 * p);
            PairOf<T>::pack(v, wx + p * (sizeof(T) / 2));
        }
        *reinterpret_cast<uint4*>(h) = rh;
        __stcs(reinterpret_cast<X*>(out), rx);
    } else {
        const float v = fmaf(load(g), *h, load(x));
        *h = v;
        store(out, v);
    }
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
    require(t->words && t->order && t->schedule[0][0] && t->schedule[0][1] && t->schedule[1][0] && t->schedule[1][1],
            "story tables are null");
    require(t->tiles[0] > 0 && t->tiles[1] >= t->tiles[0] && t->longest[0] > 0 && t->longest[1] > 0,
            "story tables are inconsistent");
    require(channels > 0 && channels < (1u << 31), "channels must be positive");
}

// The parts of a call's scratch, for the shortest tiles; returns its size.
size_t lay_out(const LeoB200StoryTables& t, uint32_t channels, void* base, Scratch* s) {
    const size_t tiles = t.tiles[1];
    if (tiles == 1) return 0;  // nothing crosses tiles
    const size_t slots = 256, partials = slots + tiles * channels * sizeof(Slot);
    if (s) {
        char* p = static_cast<char*>(base);
        s->ticket = reinterpret_cast<uint32_t*>(p);
        s->slots = reinterpret_cast<Slot*>(p + slots);
        s->partials = reinterpret_cast<float*>(p + partials);
    }
    return partials + tiles * channels * sizeof(float);
}

// Where the parts of a story table lie, in bytes.
struct TableLayout {
    size_t words, order, schedule[2][2], size;
    TableLayout(uint32_t tokens, uint32_t stories, const uint32_t (&tiles)[2]) {
        schedule[0][0] = 0;
        schedule[0][1] = schedule[0][0] + tiles[0] * sizeof(LeoB200StoryTile);
        schedule[1][0] = schedule[0][1] + tiles[0] * sizeof(LeoB200StoryTile);
        schedule[1][1] = schedule[1][0] + tiles[1] * sizeof(LeoB200StoryTile);
        words = schedule[1][1] + tiles[1] * sizeof(LeoB200StoryTile);
        order = words + ((size_t)tokens / LEO_B200_STORY_WORD_TOKENS + 2) * sizeof(LeoB200StoryWord);
        size = order + stories * sizeof(uint32_t);
    }
};

// The tiles of a batch, in the order of their tokens.  A story that does not
// fit the rest of the tile before it begins a tile of its own, so that only
// the tiles of one story depend on one another; short stories share one.
std::vector<LeoB200StoryTile> cut(const uint64_t* offsets, uint32_t stories) {
    std::vector<LeoB200StoryTile> tiles;
    for (uint32_t s = 0; s < stories; ++s) {
        const uint32_t begin = (uint32_t)offsets[s], length = (uint32_t)(offsets[s + 1] - offsets[s]);
        if (length == 0) continue;
        if (!tiles.empty() && tiles.back().count + length <= LEO_B200_TILE_TOKENS) {
            tiles.back().count += length;
            continue;
        }
        for (uint32_t at = 0; at < length; at += LEO_B200_TILE_TOKENS) {
            LeoB200StoryTile t{};
            t.first = begin + at;
            t.count = std::min(length - at, LEO_B200_TILE_TOKENS);
            tiles.push_back(t);
        }
    }
    if (tiles.empty()) tiles.push_back({});  // a batch without tokens
    return tiles;
}

// Numbers the tiles and finds, for every one, the tiles where the stories that
// cross its ends begin and end.  `starts(t)`: a story starts at token t (the
// batch's end counts as one).
template <typename Starts>
void link(std::vector<LeoB200StoryTile>& tiles, std::vector<uint32_t>& begins, std::vector<uint32_t>& ends,
          Starts&& starts) {
    const uint32_t n = (uint32_t)tiles.size();
    begins.resize(n);
    ends.resize(n);
    const auto starts_in = [&](const LeoB200StoryTile& t) {  // after its first token too
        for (uint32_t i = 0; i < t.count; ++i)
            if (starts(t.first + i)) return true;
        return false;
    };
    for (uint32_t i = 0; i < n; ++i) {
        tiles[i].tile = i;
        const bool crossed = i > 0 && !starts(tiles[i].first);
        // the story that crosses in began in the tile before, or crossed into that one too
        begins[i] = !crossed ? i : starts_in(tiles[i - 1]) ? i - 1 : begins[i - 1];
    }
    for (uint32_t i = n; i-- > 0;) {
        const bool crossed = i + 1 < n && !starts(tiles[i + 1].first);
        const auto ends_in = [&](const LeoB200StoryTile& t) {
            for (uint32_t k = 0; k < t.count; ++k)
                if (starts(t.first + k + 1)) return true;
            return false;
        };
        ends[i] = !crossed ? i : ends_in(tiles[i + 1]) ? i + 1 : ends[i + 1];
    }
}

// The tiles in the order of their tickets: by their distance from `holders`,
// so that a tile follows every tile it reads from.
uint32_t schedule(const std::vector<LeoB200StoryTile>& tiles, const std::vector<uint32_t>& holders,
              const std::vector<uint32_t>& onward, LeoB200StoryTile* out, bool backward) {
    const uint32_t n = (uint32_t)tiles.size();
    std::vector<uint32_t> rank(n), first;
    for (uint32_t k = 0; k < n; ++k) {
        const uint32_t i = backward ? n - 1 - k : k;
        rank[i] = holders[i] == i ? 0 : rank[backward ? i + 1 : i - 1] + 1;
        if (rank[i] + 2 > first.size()) first.resize(rank[i] + 2, 0);
        ++first[rank[i] + 1];
    }
    for (size_t r = 1; r < first.size(); ++r) first[r] += first[r - 1];
    for (uint32_t k = 0; k < n; ++k) {
        const uint32_t i = backward ? n - 1 - k : k;
        LeoB200StoryTile& t = out[first[rank[i]]++];
        t = tiles[i];
        t.holder = holders[i];
        t.onward = onward[i] != i;
    }
    return (uint32_t)first.size() - 1;  // the longest row of tiles that depend on one another
}

// Neighbours of a row that can be moved at once, going by its address and stride.
int unit_of(const void* p, int64_t stride, size_t size) {
    const auto fits = [&](size_t bytes) {
        return reinterpret_cast<uintptr_t>(p) % bytes == 0 && stride * (int64_t)size % (int64_t)bytes == 0;
    };
    return fits(16) ? 4 : fits(2 * size) ? 2 : 1;
}

using EncodeTiled = CUresult (*)(CUtensorMap*, CUtensorMapDataType, cuuint32_t, void*, const cuuint64_t*,
                                 const cuuint64_t*, const cuuint32_t*, const cuuint32_t*, CUtensorMapInterleave,
                                 CUtensorMapSwizzle, CUtensorMapL2promotion, CUtensorMapFloatOOBfill);

EncodeTiled encode_tiled() {
    static const EncodeTiled found = [] {
        void* entry = nullptr;
        cudaDriverEntryPointQueryResult result{};
        check(cudaGetDriverEntryPoint("cuTensorMapEncodeTiled", &entry, cudaEnableDefault, &result),
              "cuTensorMapEncodeTiled");
        require(entry != nullptr && result == cudaDriverEntryPointSuccess, "cuTensorMapEncodeTiled is missing");
        return reinterpret_cast<EncodeTiled>(entry);
    }();
    return found;
}

// Boxes of `rows` tokens of kColumns channels.
template <typename E>
void describe(CUtensorMap* map, const void* p, int64_t stride, uint32_t tokens, uint32_t channels, uint32_t rows) {
    const CUtensorMapDataType type = std::is_same_v<E, float>    ? CU_TENSOR_MAP_DATA_TYPE_FLOAT32
                                     : std::is_same_v<E, __half> ? CU_TENSOR_MAP_DATA_TYPE_FLOAT16
                                                                 : CU_TENSOR_MAP_DATA_TYPE_BFLOAT16;
    const cuuint64_t sizes[2] = {channels, tokens}, strides[1] = {(cuuint64_t)stride * sizeof(E)};
    const cuuint32_t box[2] = {kColumns, rows}, steps[2] = {1, 1};
    const CUresult r = encode_tiled()(map, type, 2, const_cast<void*>(p), sizes, strides, box, steps,
                                      CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_NONE,
                                      CU_TENSOR_MAP_L2_PROMOTION_L2_256B, CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    require(r == CUDA_SUCCESS, "cuTensorMapEncodeTiled refused a tensor");
}

// Launches one scan on `stream`: one block an SM, or one a tile if there are few.
template <typename T, typename G, int Unit, bool Shared, bool Backward>
void launch_scan(ScanArgs& a, void* workspace, size_t workspace_bytes, cudaStream_t stream) {
    using S = Shape<T, G, Shared, Backward>;
    static_assert(S::kBytes <= kSharedLimit && kKept % S::kSegment == 0, "shape");
    static_assert(S::kTile == LEO_B200_TILE_TOKENS || S::kTile == LEO_B200_TILE_TOKENS / 2, "tiles of the story table");
    constexpr int halves = S::kTile < LEO_B200_TILE_TOKENS;
    a.tiles = a.tables.tiles[halves];
    a.schedule = a.tables.schedule[halves][Backward];
    a.groups = (a.channels + kColumns - 1) / kColumns;
    const uint64_t total = (uint64_t)a.tiles * a.groups;
    require(total < (1ull << 31) - 65536, "too many tokens and channels for one scan");
    const size_t size = lay_out(a.tables, a.channels, workspace, &a.scratch);
    if (size > 0) {
        require(workspace != nullptr && workspace_bytes >= size, "the workspace is too small");
        require(reinterpret_cast<uintptr_t>(workspace) % 16 == 0, "the workspace must be aligned to 16 bytes");
    }
    // Whole tiles that may be worked on side by side without waiting for one another, of those in the longest row.
    const uint64_t whole = (uint64_t)a.tables.tiles[0] * a.groups;
    if (a.tables.longest[0] > kGroup && whole / a.tables.longest[0] < kAbreast) {
        a.tiles = a.tables.tiles[0];
        a.schedule = a.tables.schedule[0][Backward];
        constexpr uint32_t threads = 16 * kSegments;
        scan_map_kernel<T, G, Unit, Shared, Backward><<<(uint32_t)whole, threads, 0, stream>>>(a);
        check(cudaGetLastError(), "scan_map_kernel");
        scan_join_kernel<Backward><<<(a.channels + kJoinChannels - 1) / kJoinChannels, 1024, 0, stream>>>(a);
        check(cudaGetLastError(), "scan_join_kernel");
        scan_tile_kernel<T, G, Unit, Shared, Backward><<<(uint32_t)whole, threads, 0, stream>>>(a);
        check(cudaGetLastError(), "scan_tile_kernel");
        return;
    }
    const int sms = sm_count();
    const auto kernel = scan_kernel<T, G, Unit, Shared, Backward>;
    static std::atomic<uint64_t> allowed{0};
    allow_shared(kernel, S::kBytes, allowed);
    if constexpr (Unit == 4) {
        const uint32_t rows = 2 * S::kSegment;
        describe<T>(&a.drive_map, a.drive, a.drive_stride, a.tables.tokens, a.channels, rows);
        if constexpr (!Shared) describe<G>(&a.decay_map, a.decay, a.decay_stride, a.tables.tokens, a.channels, rows);
        if constexpr (Backward)
            describe<T>(&a.grad_map, a.grad_states, a.grad_states_stride, a.tables.tokens, a.channels, rows);
    }
    if (a.tiles > 1) {
        check(cudaMemsetAsync(workspace, 0xff, 256 + (size_t)a.tiles * a.channels * sizeof(Slot), stream), "clear scan slots");
    }
    const uint32_t blocks = a.tiles == 1 || total <= 2u * (uint32_t)sms ? (uint32_t)total : (uint32_t)sms;
    kernel<<<blocks, S::kThreads, S::kBytes, stream>>>(a);
    check(cudaGetLastError(), "scan_kernel");
}

// Calls body(Unit, Shared) as types.
template <typename Body>
void dispatch_shape(int unit, bool shared, Body&& body) {
    const auto with = [&](auto u) { shared ? body(u, std::true_type{}) : body(u, std::false_type{}); };
    if (unit == 4) with(std::integral_constant<int, 4>{});
    else if (unit == 2) with(std::integral_constant<int, 2>{});
    else with(std::integral_constant<int, 1>{});
}

// Tiled loads and rows of neighbours need every tensor of the call to allow
// them; rows that overlap have no tiled form.
int unit_of_call(uint32_t channels, uint32_t tokens, int64_t stride0, int64_t stride1, int64_t stride2, int least) {
    int unit = std::min(least, channels % 4 == 0 ? 4 : channels % 2 == 0 ? 2 : 1);
    const bool strided = stride0 >= channels && stride1 >= channels && stride2 >= channels;
    if (unit == 4 && (!strided || tokens == 0)) unit = 2;
    return unit;
}

}  // namespace

extern "C" {

size_t leo_b200_story_table_bytes(const uint64_t* offsets, uint32_t stories) {
    size_t bytes = 0;
    guarded([&] {
        require(offsets != nullptr && stories > 0, "a batch needs at least one story");
        require(offsets[0] == 0, "story offsets must start at 0");
        for (uint32_t s = 0; s < stories; ++s)
            require(offsets[s + 1] >= offsets[s], "story offsets must be non-decreasing");
        require(offsets[stories] < (1ull << 31), "too many tokens for one batch");
        uint32_t tiles[2] = {0, 0};
        for (const LeoB200StoryTile& t : cut(offsets, stories)) {
            ++tiles[0];
            tiles[1] += t.count > LEO_B200_TILE_TOKENS / 2 ? 2 : 1;
        }
        bytes = TableLayout((uint32_t)offsets[stories], stories, tiles).size;
    });
    return bytes;
}

int leo_b200_story_table(const uint64_t* offsets, uint32_t stories, void* table, size_t bytes, const void* device_table,
                         LeoB200StoryTables* out) {
    return guarded([&] {
        const size_t needed = leo_b200_story_table_bytes(offsets, stories);
        if (needed == 0) throw Failure(leo_b200_last_error());
        require(table != nullptr && out != nullptr, "story table arrays are null");
        require(bytes >= needed, "the story table is too small");
        require(reinterpret_cast<uintptr_t>(table) % 16 == 0 && reinterpret_cast<uintptr_t>(device_table) % 16 == 0,
                "the story table must be aligned to 16 bytes");
        const uint32_t tokens = (uint32_t)offsets[stories];
        // Whole tiles, and their halves; a state is kept before each half.
        std::vector<LeoB200StoryTile> whole = cut(offsets, stories), halves;
        for (LeoB200StoryTile& t : whole) {
            t.kept = (uint32_t)halves.size();
            for (uint32_t at = 0; at == 0 || at < t.count; at += LEO_B200_TILE_TOKENS / 2) {
                LeoB200StoryTile h = t;
                h.first += at;
                h.count = std::min(t.count - at, LEO_B200_TILE_TOKENS / 2);
                h.kept = (uint32_t)halves.size();
                halves.push_back(h);
            }
        }
        const uint32_t tiles[2] = {(uint32_t)whole.size(), (uint32_t)halves.size()};
        const TableLayout at(tokens, stories, tiles);
        std::memset(table, 0, at.size);
        char* base = static_cast<char*>(table);
        auto* words = reinterpret_cast<LeoB200StoryWord*>(base + at.words);
        auto* order = reinterpret_cast<uint32_t*>(base + at.order);
        uint32_t n = 0;
        for (uint32_t s = 0; s < stories; ++s)
            if (offsets[s + 1] > offsets[s]) {
                words[offsets[s] / LEO_B200_STORY_WORD_TOKENS].starts |= 1u << offsets[s] % LEO_B200_STORY_WORD_TOKENS;
                order[n++] = s;
            }
        const uint32_t full = n;
        for (uint32_t s = 0; s < stories; ++s)
            if (offsets[s + 1] == offsets[s]) order[n++] = s;
        words[tokens / LEO_B200_STORY_WORD_TOKENS].starts |= 1u << tokens % LEO_B200_STORY_WORD_TOKENS;
        uint32_t rank = 0;
        for (size_t w = 0; w < (size_t)tokens / LEO_B200_STORY_WORD_TOKENS + 2; ++w) {
            words[w].rank = rank;
            for (uint32_t b = words[w].starts; b; b &= b - 1) ++rank;
        }
        const auto starts = [&](uint32_t t) {
            return (words[t / LEO_B200_STORY_WORD_TOKENS].starts >> t % LEO_B200_STORY_WORD_TOKENS & 1u) != 0;
        };
        uint32_t longest[2];
        for (int k = 0; k < 2; ++k) {
            std::vector<LeoB200StoryTile>& list = k ? halves : whole;
            std::vector<uint32_t> begins, ends;
            link(list, begins, ends, starts);
            for (int d = 0; d < 2; ++d)
                longest[k] = schedule(list, d ? ends : begins, d ? begins : ends,
                                      reinterpret_cast<LeoB200StoryTile*>(base + at.schedule[k][d]), d != 0);
        }
        const char* device = static_cast<const char*>(device_table);
        LeoB200StoryTables t{};
        t.words = reinterpret_cast<const LeoB200StoryWord*>(device + at.words);
        t.order = reinterpret_cast<const uint32_t*>(device + at.order);
        for (int k = 0; k < 2; ++k) {
            t.tiles[k] = tiles[k];
            t.longest[k] = longest[k];
            for (int d = 0; d < 2; ++d)
                t.schedule[k][d] = reinterpret_cast<const LeoB200StoryTile*>(device + at.schedule[k][d]);
        }
        t.tokens = tokens;
        t.stories = stories;
        t.full = full;
        *out = t;
    });
}

size_t leo_b200_gated_scan_workspace(const LeoB200StoryTables* tables, uint32_t channels) {
    return tables ? lay_out(*tables, channels, nullptr, nullptr) : 0;
}

size_t leo_b200_gated_scan_carry_count(const LeoB200StoryTables* tables, uint32_t channels) {
    return tables ? (size_t)tables->tiles[1] * channels : 0;
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
            const bool shared = decay_shared != 0 && tables->tokens > 0;
            int unit = std::min(unit_of(drive, drive_stride, sizeof(T)), unit_of(states, channels, sizeof(T)));
            if (!shared) unit = std::min(unit, unit_of(decay, decay_stride, sizeof(G)));
            unit = unit_of_call(channels, tables->tokens, drive_stride, shared ? channels : decay_stride, channels, unit);
            DeviceScope scope(device);
            dispatch_shape(unit, shared, [&](auto u, auto is_shared) {
                launch_scan<T, G, u(), is_shared(), false>(a, workspace, workspace_bytes, (cudaStream_t)stream);
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
        require((decay && grad_decay) || (tables->tokens == 0 && !decay_shared), "scan arrays are null");
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
            const bool shared = decay_shared != 0;
            int unit = std::min(unit_of(drive, drive_stride, sizeof(T)),
                                unit_of(grad_states, grad_states_stride, sizeof(T)));
            unit = std::min(unit, unit_of(grad_drive, channels, sizeof(T)));
            if (!shared)
                unit = std::min({unit, unit_of(decay, decay_stride, sizeof(G)), unit_of(grad_decay, channels, sizeof(G))});
            unit = unit_of_call(channels, tables->tokens, drive_stride, shared ? channels : decay_stride, grad_states_stride, unit);
            DeviceScope scope(device);
            dispatch_shape(unit, shared, [&](auto u, auto is_shared) {
                launch_scan<T, G, u(), is_shared(), true>(a, workspace, workspace_bytes, (cudaStream_t)stream);
                if (decay_shared && a.tiles > 1) {
                    shared_decay_kernel<G><<<(channels + 31) / 32, kReduceThreads, 0, (cudaStream_t)stream>>>(
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
        require(channels > 0, "channels must be positive");
        require(((uint64_t)lanes * channels >> 8) < (1ull << 31) - 1, "too many lanes and channels for one step");
        dispatch(dtype, decay_dtype, [&](auto* t, auto* g) {
            using T = std::remove_pointer_t<decltype(t)>;
            using G = std::remove_pointer_t<decltype(g)>;
            if (lanes == 0) return;
            require(drive && decay && state && output, "step arrays are null");
            const int64_t gate_stride = decay_shared ? 0 : decay_stride;
            const auto fits = [](const void* p, int64_t stride, size_t size) {
                return reinterpret_cast<uintptr_t>(p) % (4 * size) == 0 && stride % 4 == 0;
            };
            const bool fours = channels % 4 == 0 && fits(drive, drive_stride, sizeof(T)) &&
                               fits(decay, gate_stride, sizeof(G)) && fits(state, state_stride, sizeof(float)) &&
                               fits(output, 0, sizeof(T));
            DeviceScope scope(device);
            const uint64_t threads = (uint64_t)lanes * (fours ? channels / 4 : channels);
            const uint32_t blocks = (uint32_t)((threads + 255) / 256);
            const auto kernel = fours ? step_kernel<T, G, 4> : step_kernel<T, G, 1>;
            kernel<<<blocks, 256, 0, (cudaStream_t)stream>>>(lanes, channels, static_cast<const T*>(drive), drive_stride,
                                                             static_cast<const G*>(decay), gate_stride, state,
                                                             state_stride, static_cast<T*>(output));
            check(cudaGetLastError(), "step_kernel");
        });
    });
}

}  // extern "C"
