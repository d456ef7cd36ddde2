// Gated linear recurrence over a batch of sequences, its gradient, and its
// one-token form.
//
//   p = [x | r | z] along the last axis (z optional), f = sigmoid(r), k = 1 - f
//   h_t = f_t h_{t-1} + k_t x_t
//   y_t = h_t * z_t * sigmoid(z_t)             (y_t = h_t without z)
//
// A long memory has k near 0, where 1 - k in 32 bits has lost k's digits; a token that
// lets the state go has f = 1 - k near 0, where k has lost f's. So a gate is kept as the
// smaller of the two, and which it is (gs_gate). Every state is held in 32 bits; only y
// and dp are rounded, once, to the type of p.
//
// A wave owns 64 * V channels (V neighbours a lane) and takes GS_R tokens at a
// time: all their loads are issued before the first is used, so that enough
// bytes are in flight, and the recurrence then runs in registers.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include <cfloat>

#include "checkpoint8.h"
#include "launchers.h"

#define GS_R 16  // tokens of a tile, and between two kept states

namespace {

__device__ __forceinline__ float gs_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
// exp overflows to +inf for x far below 0, whose reciprocal is the right 0
__device__ __forceinline__ float gs_sigmoid(float x) { return gs_rcp(1.f + __expf(-x)); }

// A gate of r in one register: the smaller of k = sigmoid(-r) and f = sigmoid(r), with all
// its digits, as +k where r >= 0 and the state is held, as -f where it is let go. The
// other one is 1 less the smaller, with all its digits too, and k f the product of both.
__device__ __forceinline__ float gs_gate(float r) {
    const float e = __expf(-fabsf(r));
    return copysignf(e * gs_rcp(1.f + e), r);
}
// where the gate holds, else lets go
__device__ __forceinline__ float gs_pick(float gate, float holds, float lets_go) { return (int)__float_as_uint(gate) >= 0 ? holds : lets_go; }
// f v
__device__ __forceinline__ float gs_passes(float gate, float v) { return fmaf(-gate, v, gs_pick(gate, v, 0.f)); }
// the state after a token, as two products: x - h may be more than the largest number
__device__ __forceinline__ float gs_next(float& gate, float x, float h) {
    asm("" : "+v"(gate));  // what was made of it before is made anew: kept, it takes registers
    const float most = gs_pick(gate, h, x), rest = gs_pick(gate, x, h), small = fabsf(gate);
    return fmaf(small, rest, fmaf(-small, most, most));
}

// V neighbouring elements of type E as the register that a load fills. They stay
// packed until they are used: 16-bit pairs as 32-bit floats would take twice the
// registers, and how many tokens a wave holds is what decides the speed here.
template <class E, int V>
struct GsPack {
    typedef typename E::store store;
    static_assert(sizeof(store) * V <= 4, "a register");
    unsigned int w;
    __device__ __forceinline__ void load(const store* from) {
        if constexpr (sizeof(store) * V == 2) w = *(const unsigned short*)from;
        else w = *(const unsigned int*)from;
    }
    __device__ __forceinline__ float get(int v) const {
        if constexpr (sizeof(store) == 4) return __uint_as_float(w);
        else if constexpr (std::is_same<E, C8Bf16>::value) return __uint_as_float(v == 0 ? w << 16 : w & 0xffff0000u);
        else return E::up((unsigned short)(v == 0 ? w : w >> 16));
    }
    // what was unpacked before this is not kept for what comes after
    __device__ __forceinline__ void pin() { asm("" : "+v"(w)); }
    static __device__ __forceinline__ void put(store* to, const float (&f)[V]) {
        if constexpr (V == 1) to[0] = E::down(f[0]);
        else *(unsigned int*)to = pair(f[0], f[1]);
    }
    static __device__ __forceinline__ unsigned int pair(float a, float b) {
        return (unsigned int)E::down(a) | ((unsigned int)E::down(b) << 16);
    }
};

// A token behind its sequence's end: whatever p holds there is gone before it is used, and
// its gate is f = 1 as such, which passes every state and gradient on as it is (an infinite
// one too: 1 less a share of 0 would be no number). The loops over a tile need no masks.
template <class E, int V, int P, int R>
__device__ __forceinline__ void gs_mask(GsPack<E, V> (&raw)[P][R], int i, bool out) {
#pragma unroll
    for (int q = 0; q < P; ++q) raw[q][i].w = out ? 0u : raw[q][i].w;
}

// Where waves share a CU by registers, a scheduler that interleaves many tokens to
// hide latencies spills: two tokens at a time are enough beside the other waves.
template <int W>
__device__ __forceinline__ void gs_fence(int i) {
    if (W > 1 && i % 2 == 0) __builtin_amdgcn_sched_barrier(0);
}

// The gates of a tile's tokens. whole: no token of the wave's lanes is behind its end.
template <int W, class E, int V, int R>
__device__ __forceinline__ void gs_gates(const GsPack<E, V> (&r)[R], float (&gate)[R][V], bool whole, int t0, int len) {
#pragma unroll
    for (int i = 0; i < R; ++i) {
#pragma unroll
        for (int v = 0; v < V; ++v) gate[i][v] = gs_gate(r[i].get(v));
        gs_fence<W>(i);
    }
    if (!whole) {
#pragma unroll
        for (int i = 0; i < R; ++i)
#pragma unroll
            for (int v = 0; v < V; ++v) gate[i][v] = t0 + i >= len ? -1.f : gate[i][v];
    }
}

struct GsArgs {
    const void* p;          // [B][T][P*D], rows at sb, st
    int64_t sb, st;
    void* y;                // [B][T][D]
    const float* h0;        // [B][D] or null
    float* h_last;          // [B][D]
    float* states;          // [B][nT][D]: h before every GS_R-th token, or null
    const void* lengths;    // [B] or null
    int lengths64;
    signed char* codes;     // [B][T][P][Dp] or null
    unsigned char* scales;  // [B][nT][P][Dp / 32][GS_R]: a tile's scales of a group lie together
    // backward
    const void* dy;         // [B][T][D], rows at dsb, dst
    int64_t dsb, dst;
    const float* dh_last;   // [B][D] or null
    void* dp;               // [B][T][P*D]
    float* dh0;             // [B][D] or null
    int B, T, D, Dp;
    int tps;                // lanes of one sequence
    int nJ;                 // blocks' tiles along T
    int groups;             // 64-lane groups of channels
    int seqs;               // staged: sequences of a wave
    int pitch_p, pitch_y;   // staged: bytes of a sequence's tile of p and of y in LDS
    // chained blocks (null: a block walks all its tiles)
    unsigned int* ticket;
    unsigned long long* agg;  // [nJ][groups][V][64]: a tile's (A, H), all ones until it is there
    unsigned int* prefix;     // [nJ / lb][groups][V][64]: state after a run of lb tiles
    int lb;                   // tiles of a link
};

__device__ __forceinline__ int gs_len(const GsArgs& a, int b) {
    if (a.lengths == nullptr) return a.T;
    int64_t n = a.lengths64 ? ((const int64_t*)a.lengths)[b] : (int64_t)((const int*)a.lengths)[b];
    return n < 0 ? 0 : (n > a.T ? a.T : (int)n);
}

// what a lane works on
struct GsLane {
    int b, d, len;
    bool live;  // has a channel
    int seq;    // staged: which of the wave's sequences
};

// staged: a wave has whole sequences
template <int V>
__device__ __forceinline__ GsLane gs_lane_staged(const GsArgs& a, int64_t cg, int lane) {
    GsLane l;
    l.seq = lane / a.tps;
    l.d = (lane - l.seq * a.tps) * V;
    const int64_t b = cg * a.seqs + l.seq;
    l.live = l.seq < a.seqs && b < a.B && l.d < a.D;
    l.seq = min(l.seq, a.seqs - 1);
    l.b = (int)min(b, (int64_t)a.B - 1);
    l.d = min(l.d, a.D - V);
    l.len = l.live ? gs_len(a, l.b) : a.T;
    return l;
}

// ---------------------------------------------------------------------------
// Staging of narrow rows. Rows of 25 or 50 channels start and end inside a memory
// sector; written row by row, every sector is written in pieces (backward 2.8 TB/s at 25
// channels against 4.6 at 32). But a sequence's tile of GS_R rows is one run of bytes:
// it goes through LDS, and memory sees whole words of the run, 256 bytes at a time.
// A run starts at any 2-byte address; in LDS it keeps its place within a word, so a
// word of memory is a word of LDS. A load may take the other half of the run's first
// or last word along (memory of the same aligned 4 bytes); a store leaves it alone.
// ---------------------------------------------------------------------------
__device__ __forceinline__ void gs_stage_in(const char* run, int bytes, char* lds, int lane) {
    const int n = ((int)((uintptr_t)run & 3) + bytes + 3) >> 2;
    const unsigned int* from = (const unsigned int*)(run - ((uintptr_t)run & 3));
    for (int w = 0; w < n; w += 64)
        if (w + lane < n)
            __builtin_amdgcn_global_load_lds((const __attribute__((address_space(1))) void*)(from + w + lane),
                                             (__attribute__((address_space(3))) void*)(lds + 4 * w), 4, 0, 0);
}

__device__ __forceinline__ void gs_stage_out(char* run, int bytes, const char* lds, int lane) {
    const int skip = (int)((uintptr_t)run & 3), end = skip + bytes, n = (end + 3) >> 2;
    char* to = run - skip;
    for (int w = lane; w < n; w += 64) {
        const unsigned int v = *(const unsigned int*)(lds + 4 * w);
        if (4 * w >= skip && 4 * w + 4 <= end) *(unsigned int*)(to + 4 * w) = v;
        else if (4 * w < skip) *(unsigned short*)(to + 4 * w + 2) = (unsigned short)(v >> 16);
        else *(unsigned short*)(to + 4 * w) = (unsigned short)v;
    }
}

// What was loaded into LDS is there, and what was read from it is in registers, for the
// one wave of the block. Said outright: a barrier of one wave waits for nothing.
__device__ __forceinline__ void gs_staged() { asm volatile("s_waitcnt vmcnt(0)" ::: "memory"); }
__device__ __forceinline__ void gs_taken() { asm volatile("s_waitcnt lgkmcnt(0)" ::: "memory"); }

template <int V>
__device__ __forceinline__ GsLane gs_lane(const GsArgs& a, int64_t id) {
    GsLane l;
    int64_t b = id / a.tps;
    l.d = (int)(id - b * a.tps) * V;
    l.live = b < a.B && l.d < a.D;
    l.seq = 0;
    l.b = b < a.B ? (int)b : a.B - 1;   // lanes without a channel read one that exists
    l.d = l.d < a.D ? l.d : a.D - V;
    l.len = l.live ? gs_len(a, l.b) : a.T;
    return l;
}

// ---------------------------------------------------------------------------
// Blocks of W waves take W tiles side by side in time. A tile maps the state
// before it to the state after it by h -> A h + H; the waves put their (A, H)
// into LDS, and each folds those before it, in their order.
//
// With few channels, time is split over blocks too. Block j needs the state
// after tile j - 1, and gets it without a second pass over the data: every block
// publishes its (A, H) as soon as it has it, and every LB-th block, which folds the
// LB - 1 before it, the state after itself. So a block reads at most LB words a
// channel, the serial chain has nJ / LB links of some 0.9 us, and the order of the
// folds is fixed: the same inputs give the same bits.
//
// (A, H) is one 64-bit word, the prefix one 32-bit word: a word is there when it
// is no longer all ones (a NaN is published as the canonical one), so data and
// flag arrive together and no fence is needed; accesses are at agent scope, since
// the blocks of a chain run on XCDs with L2 caches of their own. Blocks take their
// place in the chain from a ticket, so each waits only for blocks that run
// already: every wait ends. The bound on the spins is there so that a broken
// workspace gives NaN and no hang.
// ---------------------------------------------------------------------------
#define GS_LB 32  // tiles of a link at most
#define GS_SPINS (1 << 22)  // some seconds

__device__ __forceinline__ unsigned int gs_word(float f) { return f != f ? 0x7fc00000u : __float_as_uint(f); }

__device__ __forceinline__ void gs_publish(unsigned long long* to, float2 m) {
    __hip_atomic_store(to, ((unsigned long long)gs_word(m.y) << 32) | gs_word(m.x), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
}

__device__ __forceinline__ float2 gs_then(float2 first, float2 second) {
    return float2{first.x * second.x, fmaf(second.x, first.y, second.y)};
}

// another look at a word that was not there; false: give up
__device__ __forceinline__ bool gs_again(int& spins) {
    __builtin_amdgcn_s_sleep(1);
    return ++spins < GS_SPINS;
}

template <int V, int W>
struct GsChain {
    float2 part[2][W][V][64];
    float2 pred[W > 1 ? GS_LB : 1][V][64];
    float start[V][64];
    unsigned int ticket;
};

// A block's place: its group of channels, its tile, counted in the order of the
// chain, and the first tile that it does not do.
template <int V, int W>
__device__ __forceinline__ void gs_place(const GsArgs& a, GsChain<V, W>& s, int& cg, int& j, int& end) {
    cg = blockIdx.x;
    j = 0;
    end = a.nJ;
    if constexpr (W > 1) {
        if (a.ticket != nullptr) {
            if (threadIdx.x == 0) s.ticket = atomicAdd(a.ticket, 1u) + 1u;  // it starts at all ones
            __syncthreads();
            const unsigned int t = __builtin_amdgcn_readfirstlane(s.ticket);
            j = (int)(t / (unsigned int)a.groups);
            cg = (int)(t - (unsigned int)j * a.groups);
            end = j + 1;
        }
    }
}

// The state that enters this wave's tile, from `carry` (the state that enters the
// block's first tile; of the chain's first block where blocks are chained), and,
// where a block walks on, in `carry` the state after its last tile. `mine`: this
// wave's map; `order`: this wave's place in the block, 0 first. j counts tiles in the
// chain's order.
// `meanwhile` is done after this block's map is out and before others' are waited for.
template <int V, int W, class F>
__device__ __forceinline__ void gs_join(const GsArgs& a, GsChain<V, W>& s, int cg, int j, int order, int lane,
                                        const float2 (&mine)[V], float (&carry)[V], float (&in)[V], F&& meanwhile) {
    if constexpr (W == 1) {
        meanwhile();
#pragma unroll
        for (int v = 0; v < V; ++v) in[v] = carry[v];
        return;
    }
    const int par = j & 1;
#pragma unroll
    for (int v = 0; v < V; ++v) s.part[par][order][v][lane] = mine[v];
    __syncthreads();
    // the map from the block's first state to this wave's, and to the one after the block
    float2 to[V], all[V];
#pragma unroll
    for (int v = 0; v < V; ++v) all[v] = float2{1.f, 0.f};
    const auto parts = [&] {
#pragma unroll
        for (int v = 0; v < V; ++v) {
#pragma unroll 2
            for (int w = 0; w < W; ++w) {
                if (w == order) to[v] = all[v];
                all[v] = gs_then(all[v], s.part[par][w][v][lane]);
            }
        }
    };
    const int lb = a.lb, i = j % lb, g = j / lb;
    const bool more = j + 1 < a.nJ;
    if (a.ticket != nullptr && order == W - 1 && i < lb - 1 && more) {
        parts();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            gs_publish(a.agg + (((int64_t)j * a.groups + cg) * V + v) * 64 + lane, all[v]);
            all[v] = float2{1.f, 0.f};
        }
    }
    meanwhile();
    if (a.ticket == nullptr) {
        parts();
#pragma unroll
        for (int v = 0; v < V; ++v) {
            in[v] = fmaf(to[v].x, carry[v], to[v].y);
            carry[v] = fmaf(all[v].x, carry[v], all[v].y);
        }
        return;
    }
    // the wave's share of the blocks before, since the last link
    int spins = 0;
    for (int q = order; q < i; q += W) {
        unsigned long long word[V];
        const unsigned long long* from = a.agg + ((int64_t)(g * lb + q) * a.groups + cg) * V * 64 + lane;
        bool there;
        do {
            there = true;
#pragma unroll
            for (int v = 0; v < V; ++v) word[v] = __hip_atomic_load(from + v * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
            for (int v = 0; v < V; ++v) there &= (unsigned int)word[v] != ~0u;
        } while (!__all(there) && gs_again(spins));
#pragma unroll
        for (int v = 0; v < V; ++v)
            s.pred[q][v][lane] = float2{__uint_as_float((unsigned int)word[v]), __uint_as_float((unsigned int)(word[v] >> 32))};
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) {
#pragma unroll 2
        for (int q = 0; q < i; ++q) all[v] = gs_then(all[v], s.pred[q][v][lane]);
    }
    parts();
    // All maps are ready before the state that they are applied to is there: from a
    // link to the next it is one load, one operation and one store.
    if (order == W - 1) {
        float start[V];
#pragma unroll
        for (int v = 0; v < V; ++v) start[v] = carry[v];
        if (g > 0) {
            unsigned int word[V];
            const unsigned int* from = a.prefix + ((int64_t)(g - 1) * a.groups + cg) * V * 64 + lane;
            bool there;
            do {
                there = true;
#pragma unroll
                for (int v = 0; v < V; ++v) word[v] = __hip_atomic_load(from + v * 64, __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
#pragma unroll
                for (int v = 0; v < V; ++v) there &= word[v] != ~0u;
            } while (!__all(there) && gs_again(spins));
#pragma unroll
            for (int v = 0; v < V; ++v) start[v] = __uint_as_float(word[v]);
        }
        if (i == lb - 1 && more) {
#pragma unroll
            for (int v = 0; v < V; ++v)
                __hip_atomic_store(a.prefix + (((int64_t)g * a.groups + cg) * V + v) * 64 + lane,
                                   gs_word(fmaf(all[v].x, start[v], all[v].y)), __ATOMIC_RELAXED, __HIP_MEMORY_SCOPE_AGENT);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) s.start[v][lane] = start[v];
    }
    __syncthreads();
#pragma unroll
    for (int v = 0; v < V; ++v) in[v] = fmaf(to[v].x, s.start[v][lane], to[v].y);
}

// all ones: no word of the chain is there yet, and the next ticket is 0
__global__ __launch_bounds__(256) void gs_clear(uint4* to, int64_t n) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) to[i] = uint4{~0u, ~0u, ~0u, ~0u};
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------

// The codes and scales of a tile of one part. The 32 values of a group are pairs
// in 16 lanes (V = 2) or one in each of 32 (V = 1). A tile has 16 tokens: lane i of
// 16 (fewer in a short one) takes the largest magnitude of token i, so the scales of all tokens are made
// at once and stored once, and come back to the lanes by a broadcast.
template <class E, int V, int R>
__device__ __forceinline__ void gs_encode(const GsArgs& a, const GsPack<E, V> (&raw)[R], bool live, bool mine, int64_t row,
                                          int64_t step, int64_t group, int left, int dd, int lane) {
    unsigned int top = 0;
#pragma unroll
    for (int i = 0; i < R; ++i) {
        unsigned int t = c8_mag(raw[i].get(0));
        if constexpr (V == 2) t = max(t, c8_mag(raw[i].get(1)));
        t = c8_max16(live ? t : 0u);
        if constexpr (V == 1) t = max(t, (unsigned int)__shfl_xor((int)t, 16, 64));
        top = (lane & 15) == i ? t : top;
    }
    const unsigned int scale = c8_scale(top);
    const float mine_inv = c8_inv(scale);
    signed char* to = a.codes + row * a.Dp + dd;
    c8_for<R>([&](auto n) {
        constexpr int i = decltype(n)::value;
        // row_newbcast: lane i's value to its 16 lanes
        const float inv = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(mine_inv), 0x150 + i, 0xF, 0xF, true));
        unsigned int c = c8_code_byte(live ? raw[i].get(0) : 0.f, inv);
        if constexpr (V == 2) c |= c8_code_byte(live ? raw[i].get(1) : 0.f, inv) << 8;
        if (mine && i < left) {
            if constexpr (V == 2) *(unsigned short*)to = (unsigned short)c;
            else *(unsigned char*)to = (unsigned char)c;
        }
        to += step * a.Dp;
        if constexpr (i % 2 == 1) __builtin_amdgcn_sched_barrier(0);
    });
    // 64 bytes in a row from a wave: a scale at its token's place would be a 4-byte write
    if (mine && (V == 2 || (lane & 16) == 0)) a.scales[(group + dd / C8_GROUP) * GS_R + (lane & 15)] = (unsigned char)scale;
}

template <class E, int V, int P, bool KEEP, int W, bool STAGE = false, int R = GS_R>
__global__ __launch_bounds__(64 * W, W == 1 ? 2 : W == 4 ? 3 : 4) void gs_fwd(GsArgs a) {
    typedef GsPack<E, V> pack;
    static_assert(!STAGE || W == 1, "staged: a wave alone");
    extern __shared__ __attribute__((aligned(16))) char gs_lds[];
    __shared__ GsChain<V, W> chain;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the same in all lanes: scalar
    int cg, j, end;
    gs_place<V, W>(a, chain, cg, j, end);
    const int64_t id = (int64_t)cg * 64 + lane;
    const GsLane l = STAGE ? gs_lane_staged<V>(a, cg, lane) : gs_lane<V>(a, id);
    const int nT = (a.T + GS_R - 1) / GS_R;  // kept states
    static_assert(R == GS_R || W == 1, "shorter tiles are for sequences of one tile");
    const typename E::store* p = (const typename E::store*)a.p + l.b * a.sb + l.d;
    typename E::store* y = (typename E::store*)a.y + (int64_t)l.b * a.T * a.D + l.d;

    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = a.h0 != nullptr ? a.h0[(int64_t)l.b * a.D + l.d + v] : 0.f;

    constexpr int ES = sizeof(typename E::store);
    char* const lds_y = gs_lds + a.seqs * a.pitch_p;
    // this lane's place in a sequence's tile, p's and y's
    const char* mine_p = nullptr;
    char* mine_y = nullptr;
    if constexpr (STAGE) {
        // a tile is R rows: its start within a word is the sequence's own, tile after tile
        mine_p = gs_lds + l.seq * a.pitch_p + (int)((uintptr_t)((const typename E::store*)a.p + l.b * a.sb) & 3) + l.d * ES;
        mine_y = lds_y + l.seq * a.pitch_y + (int)((uintptr_t)((const typename E::store*)a.y + (int64_t)l.b * a.T * a.D) & 3) + l.d * ES;
    }
    auto stage = [&](int tile) {
        for (int s = 0; s < a.seqs; ++s) {
            const int64_t b = cg * (int64_t)a.seqs + s, t0 = (int64_t)tile * R;
            if (b < a.B && t0 < a.T)
                gs_stage_in((const char*)((const typename E::store*)a.p + b * a.sb + t0 * a.st), min(R, a.T - (int)t0) * P * a.D * ES,
                            gs_lds + s * a.pitch_p, lane);
        }
    };
    if constexpr (STAGE) stage(0);

    for (; j < end; ++j) {
        const int tile = j * W + wid, t0 = tile * R;
        pack raw[P][R];
        if constexpr (STAGE) {
            gs_staged();
#pragma unroll
            for (int i = 0; i < R; ++i)
#pragma unroll
                for (int q = 0; q < P; ++q) raw[q][i].load((const typename E::store*)(mine_p + (i * P + q) * a.D * ES));
            gs_taken();
            stage(tile + 1);
        } else {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = min(t0 + i, a.T - 1);
#pragma unroll
                for (int q = 0; q < P; ++q) raw[q][i].load(p + (int64_t)t * a.st + q * a.D);
            }
        }
        const bool whole = __all(l.len >= t0 + R);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < R; ++i) gs_mask<E, V, P, R>(raw, i, t0 + i >= l.len);
        }
        float gate[R][V], h[V];
        float2 m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = float2{1.f, 0.f};
        if constexpr (W > 1) {
            gs_gates<W>(raw[1], gate, whole, t0, l.len);
#pragma unroll
            for (int i = 0; i < R; ++i) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    m[v].y = gs_next(gate[i][v], raw[0][i].get(v), m[v].y);
                    m[v].x = gs_passes(gate[i][v], m[v].x);
                }
                gs_fence<W>(i);
            }
        }
        // the codes are made while the state is on its way
        gs_join<V, W>(a, chain, cg, j, wid, lane, m, carry, h, [&] {
            if constexpr (KEEP) {
                const int64_t row = ((int64_t)l.b * a.T + t0) * P;
                // channel, padding included, and whether it is one
                const int dd = (STAGE ? lane % a.tps : (int)(id % a.tps)) * V;
                const bool kept = STAGE ? lane / a.tps < a.seqs && cg * (int64_t)a.seqs + lane / a.tps < a.B : id < (int64_t)a.B * a.tps;
#pragma unroll
                for (int q = 0; q < P; ++q) {
#pragma unroll
                    for (int i = 0; i < R; ++i) raw[q][i].pin();
                    gs_encode<E, V, R>(a, raw[q], l.live, kept && tile < nT, row + q, P, (((int64_t)l.b * nT + tile) * P + q) * (a.Dp / C8_GROUP), a.T - t0, dd, lane);
                }
            }
        });
        if constexpr (W == 1) gs_gates<W>(raw[1], gate, whole, t0, l.len);  // here: packed, r takes fewer registers
        if (a.states != nullptr && l.live && tile < nT) {
#pragma unroll
            for (int v = 0; v < V; ++v) a.states[((int64_t)l.b * nT + tile) * a.D + l.d + v] = h[v];
        }
        // h_last comes from the wave that has the last token: what is behind it in its tile
        // is padding, which passes the state on
        const bool last = l.live && tile == max(l.len - 1, 0) / R;
        const int rows = l.live ? l.len - t0 : 0;  // tokens of the tile that are there, if more than 0
#pragma unroll
        for (int i = 0; i < R; ++i) {
            float out[V];
            raw[0][i].pin();
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = gs_next(gate[i][v], raw[0][i].get(v), h[v]);
                out[v] = h[v];
                if constexpr (P == 3) {
                    const float z = raw[2][i].get(v);
                    out[v] *= z * gs_sigmoid(z);
                }
            }
            if constexpr (STAGE) {
                if (l.live) pack::put((typename E::store*)(mine_y + i * a.D * ES), out);
            } else if (i < rows) {
                pack::put(y + (int64_t)(t0 + i) * a.D, out);
            }
            gs_fence<W>(i);
        }
        if constexpr (STAGE) {
            if (!whole && l.live) {
                const float zero[V] = {};
                for (int i = max(rows, 0); i < min(R, a.T - t0); ++i) pack::put((typename E::store*)(mine_y + i * a.D * ES), zero);
            }
            gs_taken();
            for (int s = 0; s < a.seqs; ++s) {
                const int64_t b = cg * (int64_t)a.seqs + s;
                if (b < a.B)
                    gs_stage_out((char*)((typename E::store*)a.y + (b * a.T + t0) * a.D), min(R, a.T - t0) * a.D * ES, lds_y + s * a.pitch_y, lane);
            }
        } else if (l.live) {
            const float zero[V] = {};
            for (int t = max(t0, l.len); t < min(t0 + R, a.T); ++t) pack::put(y + (int64_t)t * a.D, zero);
        }
        if (last) {
#pragma unroll
            for (int v = 0; v < V; ++v) a.h_last[(int64_t)l.b * a.D + l.d + v] = h[v];
        }
        if constexpr (W == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = h[v];
        }
    }
}

// ---------------------------------------------------------------------------
// backward: tiles from the last to the first. The states of a tile are computed
// again from the one kept before it, then
//   g_t = dy_t silu(z_t) + c,  c = f_t g_t for the token before
//   dx = g k, dr = g (h_{t-1} - x) k f, dz = dy h silu'(z)
// The chain carries c, from the last tile to the first. Kept codes are decoded as
// they are loaded, to bf16, in which they are exact.
// ---------------------------------------------------------------------------
// A lane of one 16-bit channel fits 128 registers: held to it, four waves a SIMD (with codes,
// 8192 sequences of 144 tokens, 25 channels: 112 us, with a few registers more 140).
template <class E, int V, int P, bool KEEP, int W, bool STAGE = false, int R = GS_R>
__global__ __launch_bounds__(64 * W, W == 1 ? (V == 1 && sizeof(typename E::store) == 2 ? 4 : 2) : W == 4 ? 3 : 4) void gs_bwd(GsArgs a) {
    typedef GsPack<E, V> pack;
    extern __shared__ __attribute__((aligned(16))) char gs_lds[];
    typedef typename std::conditional<KEEP, C8Bf16, E>::type K;  // type of the kept projection in registers
    __shared__ GsChain<V, W> chain;
    const int lane = threadIdx.x & 63, wid = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);  // the same in all lanes: scalar
    int cg, j, end;
    gs_place<V, W>(a, chain, cg, j, end);
    const int64_t id = (int64_t)cg * 64 + lane;
    const GsLane l = STAGE ? gs_lane_staged<V>(a, cg, lane) : gs_lane<V>(a, id);
    const int nT = (a.T + GS_R - 1) / GS_R;  // kept states
    static_assert(R == GS_R || W == 1, "shorter tiles are for sequences of one tile");
    const int64_t row0 = (int64_t)l.b * a.T;
    const typename E::store* p = (const typename E::store*)a.p + l.b * a.sb + l.d;
    const typename E::store* dy = (const typename E::store*)a.dy + l.b * a.dsb + l.d;
    typename E::store* dp = (typename E::store*)a.dp + row0 * P * a.D + l.d;

    float carry[V];
#pragma unroll
    for (int v = 0; v < V; ++v) carry[v] = a.dh_last != nullptr ? a.dh_last[(int64_t)l.b * a.D + l.d + v] : 0.f;

    // LDS, staged: a tile of p (not of codes: their rows are whole sectors), one of dy, and
    // one of dp to go out
    constexpr int ES = sizeof(typename E::store);
    char* const lds_dy = gs_lds + (KEEP ? 0 : a.seqs * a.pitch_p);
    char* const lds_dp = lds_dy + a.seqs * a.pitch_y;
    const char *mine_p = nullptr, *mine_dy = nullptr;
    char* mine_dp = nullptr;
    if constexpr (STAGE) {
        mine_p = gs_lds + l.seq * a.pitch_p + (int)((uintptr_t)((const typename E::store*)a.p + l.b * a.sb) & 3) + l.d * ES;
        mine_dy = lds_dy + l.seq * a.pitch_y + (int)((uintptr_t)((const typename E::store*)a.dy + l.b * a.dsb) & 3) + l.d * ES;
        mine_dp = lds_dp + l.seq * a.pitch_p + (int)((uintptr_t)((const typename E::store*)a.dp + row0 * P * a.D) & 3) + l.d * ES;
    }
    auto stage = [&](int tile) {
        if (tile < 0) return;
        const int t0 = tile * R, rows = min(R, a.T - t0);
        for (int s = 0; s < a.seqs; ++s) {
            const int64_t b = cg * (int64_t)a.seqs + s;
            if (b >= a.B) break;
            if constexpr (!KEEP)
                gs_stage_in((const char*)((const typename E::store*)a.p + b * a.sb + t0 * a.st), rows * P * a.D * ES, gs_lds + s * a.pitch_p, lane);
            gs_stage_in((const char*)((const typename E::store*)a.dy + b * a.dsb + t0 * a.dst), rows * a.D * ES, lds_dy + s * a.pitch_y, lane);
        }
    };
    if constexpr (STAGE) stage(a.nJ - 1);

    for (; j < end; ++j) {
        const int tile = (a.nJ - 1 - j) * W + wid, t0 = tile * R;
        GsPack<K, V> raw[P][R];
        pack up[R];
        if constexpr (STAGE) {
            gs_staged();
#pragma unroll
            for (int i = 0; i < R; ++i) {
                up[i].load((const typename E::store*)(mine_dy + i * a.D * ES));
                if constexpr (!KEEP)
#pragma unroll
                    for (int q = 0; q < P; ++q) raw[q][i].load((const typename E::store*)(mine_p + (i * P + q) * a.D * ES));
            }
            gs_taken();
            stage(tile - 1);
        }
        if constexpr (KEEP) {
            // lane i of 16 has the scale of token i
            float step[P];
            const int64_t group = ((int64_t)l.b * nT + min(tile, nT - 1)) * P * (a.Dp / C8_GROUP);
            // the group's lanes stay together, padding included
            const int dd = (STAGE ? lane % a.tps : (int)(id % a.tps)) * V;
#pragma unroll
            for (int q = 0; q < P; ++q) step[q] = c8_step(a.scales[(group + (q * a.Dp + dd) / C8_GROUP) * GS_R + (lane & 15)]);
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = min(t0 + i, a.T - 1);
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    const signed char* from = a.codes + ((row0 + t) * P + q) * a.Dp + dd;
                    if constexpr (V == 2) raw[q][i].w = *(const unsigned short*)from;
                    else raw[q][i].w = *(const unsigned char*)from;
                }
            }
            if constexpr (!STAGE)
#pragma unroll
                for (int i = 0; i < R; ++i) up[i].load(dy + (int64_t)min(t0 + i, a.T - 1) * a.dst);
            c8_for<R>([&](auto n) {
                constexpr int i = decltype(n)::value;
#pragma unroll
                for (int q = 0; q < P; ++q) {
                    raw[q][i].pin();
                    // row_newbcast: lane i's value to its 16 lanes
                    const float s = __int_as_float(__builtin_amdgcn_mov_dpp(__float_as_int(step[q]), 0x150 + i, 0xF, 0xF, true));
                    const unsigned int w = raw[q][i].w;
                    const float f0 = (float)(signed char)(w & 0xff) * s;
                    if constexpr (V == 2) raw[q][i].w = (__float_as_uint(f0) >> 16) | (__float_as_uint((float)(signed char)(w >> 8) * s) & 0xffff0000u);
                    else raw[q][i].w = __float_as_uint(f0) >> 16;
                }
            });
        } else if constexpr (!STAGE) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                const int t = min(t0 + i, a.T - 1);
                up[i].load(dy + (int64_t)t * a.dst);
#pragma unroll
                for (int q = 0; q < P; ++q) raw[q][i].load(p + (int64_t)t * a.st + q * a.D);
            }
        }
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = a.states[((int64_t)l.b * nT + min(tile, nT - 1)) * a.D + l.d + v];
        const bool whole = __all(l.len >= t0 + R);
        if (!whole) {
#pragma unroll
            for (int i = 0; i < R; ++i) {
                gs_mask<K, V, P, R>(raw, i, t0 + i >= l.len);
                up[i].w = t0 + i >= l.len ? 0u : up[i].w;
            }
        }
        float gate[R][V], c[V];
        gs_gates<W>(raw[1], gate, whole, t0, l.len);
        float2 m[V];
#pragma unroll
        for (int v = 0; v < V; ++v) m[v] = float2{1.f, 0.f};
        if constexpr (W > 1) {
#pragma unroll
            for (int i = R - 1; i >= 0; --i) {
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    float g = up[i].get(v);
                    if constexpr (P == 3) {
                        const float z = raw[2][i].get(v);
                        g *= z * gs_sigmoid(z);
                    }
                    m[v].y = gs_passes(gate[i][v], g + m[v].y);
                    m[v].x = gs_passes(gate[i][v], m[v].x);
                }
                gs_fence<W>(i);
            }
        }
        gs_join<V, W>(a, chain, cg, j, W - 1 - wid, lane, m, carry, c, [] {});
        // Beside other waves, and where codes take registers too, the states of half a tile at
        // a time: the first half's are computed twice. A wave alone keeps all of them (8192
        // sequences of 144 tokens, 70 channels: 356 us, in halves 384; 25 channels as codes,
        // where they would cost a wave a SIMD: 142, in halves 112).
        constexpr int SPAN = W == 1 && !KEEP ? R : R / 2;
        const int rows = l.live ? l.len - t0 : 0;  // tokens of the tile that are there, if more than 0
        float first[V], before[SPAN][V];
#pragma unroll
        for (int v = 0; v < V; ++v) first[v] = h[v];
#pragma unroll
        for (int i = 0; i < R - SPAN; ++i) {
            raw[0][i].pin();
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = gs_next(gate[i][v], raw[0][i].get(v), h[v]);
        }
#pragma unroll
        for (int half = R / SPAN - 1; half >= 0; --half) {
#pragma unroll
            for (int n = 0; n < SPAN; ++n) {
                const int i = half * SPAN + n;
                raw[0][i].pin();
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    before[n][v] = h[v];
                    h[v] = gs_next(gate[i][v], raw[0][i].get(v), h[v]);
                }
            }
            gs_fence<W>(0);
#pragma unroll
            for (int n = SPAN - 1; n >= 0; --n) {
                const int i = half * SPAN + n;
                float out[P][V];
                raw[P - 1][i].pin();
                up[i].pin();
#pragma unroll
                for (int v = 0; v < V; ++v) {
                    asm("" : "+v"(gate[i][v]));
                    const float x = raw[0][i].get(v), small = fabsf(gate[i][v]), hp = before[n][v];
                    float g = up[i].get(v);
                    if constexpr (P == 3) {
                        const float z = raw[2][i].get(v);
                        const float s = gs_sigmoid(z), zs = z * s;
                        out[2][v] = g * fmaf(zs, 1.f - s, s) * (n == SPAN - 1 ? h[v] : before[(n + 1) % SPAN][v]);
                        g *= zs;
                    }
                    g += c[v];
                    // k g and f g, or f g and k g. An infinite g stays so: 1 less a share is more than 0.
                    const float less = small * g, more = fmaf(-small, __builtin_amdgcn_fmed3f(g, -FLT_MAX, FLT_MAX), g);
                    c[v] = gs_pick(gate[i][v], more, less);
                    out[0][v] = gs_pick(gate[i][v], less, more);
                    out[1][v] = fmaf(small, hp, -(small * x)) * more;  // small is at most 1/2: the difference does not overflow
                }
                if constexpr (STAGE) {
                    if (l.live) {
#pragma unroll
                        for (int q = 0; q < P; ++q) pack::put((typename E::store*)(mine_dp + (i * P + q) * a.D * ES), out[q]);
                    }
                } else if (i < rows) {
#pragma unroll
                    for (int q = 0; q < P; ++q) pack::put(dp + ((int64_t)(t0 + i) * P + q) * a.D, out[q]);
                }
                gs_fence<W>(i);
            }
#pragma unroll
            for (int v = 0; v < V; ++v) h[v] = first[v];
        }
        if constexpr (STAGE) {
            if (!whole && l.live) {
                const float zero[V] = {};
                for (int i = max(rows, 0); i < min(R, a.T - t0); ++i)
#pragma unroll
                    for (int q = 0; q < P; ++q) pack::put((typename E::store*)(mine_dp + (i * P + q) * a.D * ES), zero);
            }
            gs_taken();
            for (int s = 0; s < a.seqs; ++s) {
                const int64_t b = cg * (int64_t)a.seqs + s;
                if (b < a.B)
                    gs_stage_out((char*)((typename E::store*)a.dp + (b * a.T + t0) * P * a.D), min(R, a.T - t0) * P * a.D * ES, lds_dp + s * a.pitch_p, lane);
            }
        } else if (l.live) {
            const float zero[V] = {};
            for (int t = max(t0, l.len); t < min(t0 + R, a.T); ++t)
#pragma unroll
                for (int q = 0; q < P; ++q) pack::put(dp + ((int64_t)t * P + q) * a.D, zero);
        }
        if (l.live && a.dh0 != nullptr && tile == 0) {
#pragma unroll
            for (int v = 0; v < V; ++v) a.dh0[(int64_t)l.b * a.D + l.d + v] = c[v];
        }
        if constexpr (W == 1) {
#pragma unroll
            for (int v = 0; v < V; ++v) carry[v] = c[v];
        }
    }
}

// ---------------------------------------------------------------------------
// one token. A block takes one row of p, all its channels. Rows with the same
// slot are applied in their order: the block of the first one does them all,
// the blocks of the others leave. Every state word is read and written by one
// lane only, so `out` may be `state` itself.
// ---------------------------------------------------------------------------
struct GsStepArgs {
    const void* p;
    int64_t sb;
    const float* state;  // [S][D]
    float* out;          // [S][D]
    const void* slots;   // [B] or null: row b has slot b
    int slots64;
    void* y;             // [B][D]
    int B, D;
    int64_t S;
};

__device__ __forceinline__ int64_t gs_slot(const GsStepArgs& a, int b) {
    return a.slots64 ? ((const int64_t*)a.slots)[b] : (int64_t)((const int*)a.slots)[b];
}

template <class E, int V, int P>
__global__ __launch_bounds__(256) void gs_step(GsStepArgs a) {
    typedef GsPack<E, V> pack;
    __shared__ int found[4];
    const int row = blockIdx.x, step = blockDim.x * V;
    const int64_t slot = a.slots != nullptr ? gs_slot(a, row) : row;
    typename E::store* y = (typename E::store*)a.y;
    if (slot < 0 || slot >= a.S) {  // no state: a row of padding
        const float zero[V] = {};
        for (int d = threadIdx.x * V; d < a.D; d += step) pack::put(y + (int64_t)row * a.D + d, zero);
        return;
    }
    pack raw[P];
    float h[V];
    auto load = [&](int b, int d) {
        const typename E::store* p = (const typename E::store*)a.p + b * a.sb + d;
#pragma unroll
        for (int q = 0; q < P; ++q) raw[q].load(p + (int64_t)q * a.D);
    };
    auto state = [&](int d) {
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = a.state[slot * a.D + d + v];
    };
    int d = threadIdx.x * V;
    if (d < a.D) {  // under way while the slots are looked through
        load(row, d);
        state(d);
    }
    int later = 0;
    if (a.slots != nullptr) {
        int other = 0;  // 1: an earlier row has the slot, 2: a later one
        auto look = [&](int b, int64_t s) {
            if (s == slot && b != row) other |= b < row ? 1 : 2;
        };
        int from = 0;
        if (!a.slots64 && ((uintptr_t)a.slots & 15) == 0) {  // four at a time
            from = a.B & ~3;
            for (int b = threadIdx.x * 4; b < from; b += blockDim.x * 4) {
                const int4 four = *(const int4*)((const int*)a.slots + b);
                look(b, four.x);
                look(b + 1, four.y);
                look(b + 2, four.z);
                look(b + 3, four.w);
            }
        }
        for (int b = from + threadIdx.x; b < a.B; b += blockDim.x) look(b, gs_slot(a, b));
        const int both = (__any(other & 1) ? 1 : 0) | (__any(other & 2) ? 2 : 0);
        if ((threadIdx.x & 63) == 0) found[threadIdx.x >> 6] = both;
        __syncthreads();
        for (int w = 0; w < (int)blockDim.x >> 6; ++w) later |= found[w];
        if (later & 1) return;
    }
    for (; d < a.D; d += step) {
        if (d >= step) {
            load(row, d);
            state(d);
        }
        for (int b = row;;) {
            float out[V];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                float gate = gs_gate(raw[1].get(v));
                h[v] = gs_next(gate, raw[0].get(v), h[v]);
                out[v] = h[v];
                if constexpr (P == 3) {
                    const float z = raw[2].get(v);
                    out[v] *= z * gs_sigmoid(z);
                }
            }
            pack::put(y + (int64_t)b * a.D + d, out);
            if (!later) break;
            do ++b;
            while (b < a.B && gs_slot(a, b) != slot);
            if (b >= a.B) break;
            load(b, d);
        }
#pragma unroll
        for (int v = 0; v < V; ++v) a.out[slot * a.D + d + v] = h[v];
    }
}

// a lane takes two neighbouring channels where that is one aligned 32-bit access
bool gs_pairs(const torch::Tensor& t) { return t.element_size() == 2 && (uintptr_t)t.data_ptr() % 4 == 0; }

// calls f.template operator()<E, V, P>()
template <class F>
void gs_types(at::ScalarType dt, bool pair, int64_t parts, F&& f) {
    auto with = [&](auto e) {
        typedef decltype(e) E;
        if constexpr (sizeof(typename E::store) == 2) {
            if (pair) {
                if (parts == 3) f.template operator()<E, 2, 3>();
                else f.template operator()<E, 2, 2>();
                return;
            }
        }
        {
            if (parts == 3) f.template operator()<E, 1, 3>();
            else f.template operator()<E, 1, 2>();
        }
    };
    if (dt == at::kBFloat16) with(C8Bf16{});
    else if (dt == at::kHalf) with(C8Fp16{});
    else if (dt == at::kFloat) with(C8Fp32{});
    else TORCH_CHECK(false, "gated_scan: p must be float32, bfloat16 or float16");
}

void gs_f32(const torch::Tensor& t, int64_t n, const torch::Tensor& p, const char* what) {
    TORCH_CHECK(t.device() == p.device() && t.scalar_type() == at::kFloat && t.is_contiguous() && t.numel() == n,
                "gated_scan: ", what, " must be contiguous float32 with ", n, " values on the device of p");
}

// How a scan is laid out. One wave a block that walks all tokens (W = 1) needs no
// exchange, and fills the chip from 2048 groups of channels on (8 waves a CU). With
// fewer, `many` waves share the tokens; with fewer than two such blocks a CU,
// and more than a few tiles, blocks are chained along time. Forward without codes
// fits 128 registers a lane: blocks of 8 waves, 4 waves a SIMD. The codes and the
// backward pass need up to 168: blocks of 4, 3 waves a SIMD.
// Staging: where a wave walks alone, narrow rows that are not whole sectors (64 bytes) go
// through LDS: 8192 sequences of 144 tokens, 25 channels in bf16, take 49 + 78 us that way,
// forward and backward, and 50 + 108 row by row. Rows of up to 64 channels have a lane for
// each: more waves, more loads under way (144 tokens, 50 channels, x | r | z: 119 + 210 us,
// 151 + 292 in pairs). In tiles of 4 tokens a wave has little to do, and pairs, which give
// it two rows, are faster (200000 of 3 tokens, 50 channels: 91 + 133, and 126 + 162 a lane
// each). Rows of 66 to 128 channels go in pairs (8192 x 144 x 70: 163 + 349, row by row 191
// + 384), but not into codes (16384 x 40 x 100: 234 + 250, row by row 192 + 185), not in
// tiles of 4 (200000 x 3 x 100: 154 + 238, row by row 142 + 251), and not where tiles
// have over an eighth more tokens than there are: LDS has room for two waves a SIMD, which
// walk them all the same (30000 x 40 x 70: 189 + 415, row by row 190 + 358).
// Sequences of up to 4 tokens have tiles of 4 (32768 of one token, 1024 channels:
// forward 284 us in tiles of 16, 117 in tiles of 4).
struct GsPlan {
    int W, R;
    unsigned int blocks;
    torch::Tensor space;
    int staged;  // channels of a lane, 0: not staged
    size_t lds;
};

// A launch takes fewer than 2^32 threads.
unsigned int gs_blocks(int64_t blocks, int threads, const char* what) {
    TORCH_CHECK(blocks * threads <= UINT32_MAX, what, ": sizes of p out of range");
    return (unsigned int)blocks;
}

GsPlan gs_plan(GsArgs& a, int V, int many, int parts, const torch::Tensor& p, hipStream_t stream) {
    GsPlan plan{};
    const int64_t groups = ((int64_t)a.B * a.tps + 63) / 64;
    TORCH_CHECK(groups <= INT_MAX && a.T <= (1 << 30), "gated_scan: sizes of p out of range");
    plan.W = a.T <= GS_R || groups >= 2048 ? 1 : many;
    plan.R = a.T <= 4 ? 4 : GS_R;
    a.lb = 1;  // no chain
    const int es = (int)p.element_size();
    const bool narrow = a.D <= 64, brief = plan.R < GS_R;
    const int stage = V == 2 && narrow == brief ? 2 : 1;
    const bool full = ((int64_t)a.T + plan.R - 1) / plan.R * plan.R * 8 <= (int64_t)a.T * 9;
    const bool fits = narrow || (a.D <= 128 && stage == 2 && a.codes == nullptr && full);
    if (plan.W == 1 && fits && a.D * es % 64 != 0 && (a.T == 1 || (a.st == (int64_t)parts * a.D && (a.dy == nullptr || a.dst == a.D)))) {
        plan.staged = stage;
        a.tps = (a.codes != nullptr ? a.Dp : a.D) / stage;
        a.seqs = 64 / a.tps;
        a.pitch_p = (plan.R * parts * a.D * es + 7) / 4 * 4;
        a.pitch_y = (plan.R * a.D * es + 7) / 4 * 4;
        a.nJ = (a.T + plan.R - 1) / plan.R;
        plan.blocks = gs_blocks(((int64_t)a.B + a.seqs - 1) / a.seqs, 64, "gated_scan");
        const int p_in = a.dy != nullptr && a.codes != nullptr ? 0 : a.pitch_p;
        plan.lds = (size_t)a.seqs * (p_in + a.pitch_y + (a.dy != nullptr ? a.pitch_p : 0));
        return plan;
    }
    a.groups = (int)groups;
    a.nJ = (a.T + plan.W * plan.R - 1) / (plan.W * plan.R);
    const bool chained = plan.W > 1 && groups < 512 && a.nJ > 4;
    const int64_t blocks = chained ? groups * a.nJ : groups;
    plan.blocks = gs_blocks(blocks, 64 * plan.W, "gated_scan");
    if (chained) {
        // Links of 16 tiles, where those take as long as a link by their bytes; else 32
        // (1 sequence of 131072 tokens, 64 channels: 61 + 108 us in links of 16, 47 + 75 of 32;
        // of 65536 tokens, 768 channels: 106 + 174 of 16, 108 + 198 of 32).
        a.lb = groups * plan.W * V < 32 ? GS_LB : 16;
        const int64_t words = blocks * V * 64, links = (int64_t)((a.nJ + a.lb - 1) / a.lb) * groups * V * 64;
        const int64_t n = (words * 8 + links * 4 + 16 + 15) / 16;
        plan.space = torch::empty({n * 16}, p.options().dtype(at::kByte));
        char* at = (char*)plan.space.data_ptr();
        a.ticket = (unsigned int*)at;
        a.agg = (unsigned long long*)(at + 16);
        a.prefix = (unsigned int*)(at + 16 + words * 8);
        hipLaunchKernelGGL(gs_clear, dim3((unsigned)std::min<int64_t>((n + 255) / 256, 2048)), dim3(256), 0, stream, (uint4*)at, n);
    }
    return plan;
}

struct GsFwdCall {
    const GsArgs& a;
    const GsPlan& plan;
    hipStream_t stream;
    void go(void (*staged)(GsArgs)) { hipLaunchKernelGGL(staged, dim3(plan.blocks), dim3(64), plan.lds, stream, a); }
    template <class E, int V, int P, bool KEEP>
    void with() {
        if (plan.staged) {
            if constexpr (V == 2) {
                if (plan.R == 4) go(gs_fwd<E, 2, P, KEEP, 1, true, 4>);
                else if constexpr (!KEEP)
                    if (plan.staged == 2) go(gs_fwd<E, 2, P, KEEP, 1, true>);
            } else if (plan.R == 4) {
                go(gs_fwd<E, 1, P, KEEP, 1, true, 4>);
            }
            if (plan.R == GS_R && plan.staged == 1) go(gs_fwd<E, 1, P, KEEP, 1, true>);
            return;
        }
        if (plan.R == 4) hipLaunchKernelGGL((gs_fwd<E, V, P, KEEP, 1, false, 4>), dim3(plan.blocks), dim3(64), 0, stream, a);
        else if (plan.W == 1) hipLaunchKernelGGL((gs_fwd<E, V, P, KEEP, 1>), dim3(plan.blocks), dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((gs_fwd<E, V, P, KEEP, KEEP ? 4 : 8>), dim3(plan.blocks), dim3(KEEP ? 256 : 512), 0, stream, a);
    }
    template <class E, int V, int P>
    void operator()() {
        if (a.codes != nullptr) with<E, V, P, true>();
        else with<E, V, P, false>();
    }
};

struct GsBwdCall {
    const GsArgs& a;
    const GsPlan& plan;
    hipStream_t stream;
    void go(void (*staged)(GsArgs)) { hipLaunchKernelGGL(staged, dim3(plan.blocks), dim3(64), plan.lds, stream, a); }
    template <class E, int V, int P, bool KEEP>
    void with() {
        if (plan.staged) {
            if constexpr (V == 2) {
                if (plan.R == 4) go(gs_bwd<E, 2, P, KEEP, 1, true, 4>);
                else if constexpr (!KEEP)
                    if (plan.staged == 2) go(gs_bwd<E, 2, P, KEEP, 1, true>);
            } else if (plan.R == 4) {
                go(gs_bwd<E, 1, P, KEEP, 1, true, 4>);
            }
            if (plan.R == GS_R && plan.staged == 1) go(gs_bwd<E, 1, P, KEEP, 1, true>);
            return;
        }
        if (plan.R == 4) hipLaunchKernelGGL((gs_bwd<E, V, P, KEEP, 1, false, 4>), dim3(plan.blocks), dim3(64), 0, stream, a);
        else if (plan.W == 1) hipLaunchKernelGGL((gs_bwd<E, V, P, KEEP, 1>), dim3(plan.blocks), dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((gs_bwd<E, V, P, KEEP, 4>), dim3(plan.blocks), dim3(256), 0, stream, a);
    }
    template <class E, int V, int P>
    void operator()() {
        if (a.codes != nullptr) with<E, V, P, true>();
        else with<E, V, P, false>();
    }
};

struct GsStepCall {
    const GsStepArgs& a;
    int threads;
    hipStream_t stream;
    template <class E, int V, int P>
    void operator()() {
        hipLaunchKernelGGL((gs_step<E, V, P>), dim3(gs_blocks(a.B, threads, "gated_step")), dim3(threads), 0, stream, a);
    }
};

void gs_shape(GsArgs& a, const torch::Tensor& p, int64_t dim) {
    TORCH_CHECK(p.is_cuda() && p.dim() == 3 && p.stride(2) == 1, "gated_scan: p must be [B, T, parts * dim] on the GPU, unit stride last");
    TORCH_CHECK(dim > 0 && (p.size(2) == 2 * dim || p.size(2) == 3 * dim), "gated_scan: p's last axis must be 2 or 3 times dim");
    TORCH_CHECK(p.size(0) > 0 && p.size(1) > 0 && p.size(0) <= INT_MAX && p.size(1) <= INT_MAX && p.size(2) <= INT_MAX, "gated_scan: sizes of p out of range");
    a.p = p.data_ptr();
    a.sb = p.stride(0);
    a.st = p.stride(1);
    a.B = (int)p.size(0);
    a.T = (int)p.size(1);
    a.D = (int)dim;
    a.Dp = (int)((dim + C8_GROUP - 1) / C8_GROUP * C8_GROUP);
}

void gs_lengths(GsArgs& a, const c10::optional<torch::Tensor>& lengths, const torch::Tensor& p) {
    if (!lengths.has_value()) return;
    TORCH_CHECK(lengths->device() == p.device() && lengths->is_contiguous() && lengths->numel() == p.size(0) &&
                    (lengths->scalar_type() == at::kInt || lengths->scalar_type() == at::kLong),
                "gated_scan: lengths must be contiguous int32 or int64 [B] on the device of p");
    a.lengths = lengths->data_ptr();
    a.lengths64 = lengths->scalar_type() == at::kLong;
}

void gs_codes(GsArgs& a, const c10::optional<torch::Tensor>& codes, const c10::optional<torch::Tensor>& scales,
              const torch::Tensor& p, int64_t parts) {
    if (!codes.has_value()) return;
    const int64_t rows = p.size(0) * p.size(1) * parts, groups = p.size(0) * ((a.T + GS_R - 1) / GS_R) * parts * (a.Dp / C8_GROUP);
    TORCH_CHECK(scales.has_value() && codes->device() == p.device() && scales->device() == p.device() &&
                    codes->scalar_type() == at::kChar && scales->scalar_type() == at::kByte &&
                    codes->is_contiguous() && scales->is_contiguous() &&
                    codes->numel() == rows * a.Dp && scales->numel() == groups * GS_R,
                "gated_scan: codes and scales do not match p");
    a.codes = (signed char*)codes->data_ptr();
    a.scales = (unsigned char*)scales->data_ptr();
}

}  // namespace

void gated_scan_fwd_launch(torch::Tensor p, int64_t dim, c10::optional<torch::Tensor> h0,
                           c10::optional<torch::Tensor> lengths, torch::Tensor y, torch::Tensor h_last,
                           c10::optional<torch::Tensor> states, c10::optional<torch::Tensor> codes,
                           c10::optional<torch::Tensor> scales) {
    GsArgs a{};
    gs_shape(a, p, dim);
    const int64_t parts = p.size(2) / dim, n = (int64_t)a.B * a.D;
    TORCH_CHECK(y.device() == p.device() && y.scalar_type() == p.scalar_type() && y.is_contiguous() &&
                    y.numel() == n * a.T, "gated_scan: y does not match p");
    gs_f32(h_last, n, p, "h_last");
    a.y = y.data_ptr();
    a.h_last = h_last.data_ptr<float>();
    if (h0.has_value()) {
        gs_f32(*h0, n, p, "h0");
        a.h0 = h0->data_ptr<float>();
    }
    if (states.has_value()) {
        gs_f32(*states, n * ((a.T + GS_R - 1) / GS_R), p, "states");
        a.states = states->data_ptr<float>();
    }
    gs_lengths(a, lengths, p);
    gs_codes(a, codes, scales, p, parts);
    const bool pair = a.D % 2 == 0 && a.sb % 2 == 0 && a.st % 2 == 0 && gs_pairs(p) && gs_pairs(y);
    const int V = pair ? 2 : 1;
    a.tps = a.codes != nullptr ? a.Dp / V : a.D / V;
    const c10::DeviceGuard guard(p.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    const GsPlan plan = gs_plan(a, V, a.codes != nullptr ? 4 : 8, (int)parts, p, stream);
    GsFwdCall call{a, plan, stream};
    gs_types(p.scalar_type(), pair, parts, call);
    C10_HIP_KERNEL_LAUNCH_CHECK();
}

void gated_scan_bwd_launch(torch::Tensor p, int64_t dim, c10::optional<torch::Tensor> lengths,
                           torch::Tensor states, c10::optional<torch::Tensor> codes,
                           c10::optional<torch::Tensor> scales, torch::Tensor dy,
                           c10::optional<torch::Tensor> dh_last, torch::Tensor dp,
                           c10::optional<torch::Tensor> dh0) {
    // with codes, p is not read: dp says its shape
    GsArgs a{};
    gs_shape(a, p, dim);
    const int64_t parts = p.size(2) / dim, n = (int64_t)a.B * a.D;
    TORCH_CHECK(dp.device() == p.device() && dp.scalar_type() == p.scalar_type() && dp.is_contiguous() &&
                    dp.numel() == n * a.T * parts, "gated_scan: dp does not match p");
    TORCH_CHECK(dy.device() == p.device() && dy.scalar_type() == p.scalar_type() && dy.dim() == 3 &&
                    dy.size(0) == a.B && dy.size(1) == a.T && dy.size(2) == a.D && (a.D == 1 || dy.stride(2) == 1),
                "gated_scan: dy does not match p");
    gs_f32(states, n * ((a.T + GS_R - 1) / GS_R), p, "states");
    a.states = states.data_ptr<float>();
    a.dy = dy.data_ptr();
    a.dsb = dy.stride(0);
    a.dst = dy.stride(1);
    a.dp = dp.data_ptr();
    if (dh_last.has_value()) {
        gs_f32(*dh_last, n, p, "dh_last");
        a.dh_last = dh_last->data_ptr<float>();
    }
    if (dh0.has_value()) {
        gs_f32(*dh0, n, p, "dh0");
        a.dh0 = dh0->data_ptr<float>();
    }
    gs_lengths(a, lengths, p);
    gs_codes(a, codes, scales, p, parts);
    const bool pair = a.D % 2 == 0 && a.dsb % 2 == 0 && a.dst % 2 == 0 && gs_pairs(dy) && gs_pairs(dp) &&
                      (a.codes != nullptr || (a.sb % 2 == 0 && a.st % 2 == 0 && gs_pairs(p)));
    const int V = pair ? 2 : 1;
    a.tps = a.codes != nullptr ? a.Dp / V : a.D / V;
    const c10::DeviceGuard guard(p.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    const GsPlan plan = gs_plan(a, V, 4, (int)parts, p, stream);
    GsBwdCall call{a, plan, stream};
    gs_types(p.scalar_type(), pair, parts, call);
    C10_HIP_KERNEL_LAUNCH_CHECK();
}

torch::Tensor gated_step_launch(torch::Tensor p, torch::Tensor state, c10::optional<torch::Tensor> slots,
                                torch::Tensor out) {
    TORCH_CHECK(state.dim() == 2, "gated_step: state must be [slots, dim]");
    for (const auto& t : {p, state, out}) TORCH_CHECK_VALUE(!t._fw_grad(/*level=*/0).defined(), "gated_step has no gradient, no forward mode either");
    const int64_t dim = state.size(1);
    TORCH_CHECK(p.is_cuda() && p.dim() == 2 && p.stride(1) == 1 && dim > 0 &&
                    (p.size(1) == 2 * dim || p.size(1) == 3 * dim) && p.size(0) > 0 && p.size(0) <= INT_MAX && p.size(1) <= INT_MAX,
                "gated_step: p must be [B, 2 or 3 times dim] on the GPU, unit stride last");
    GsStepArgs a{};
    a.B = (int)p.size(0);
    a.D = (int)dim;
    a.S = state.size(0);
    gs_f32(state, a.S * dim, p, "state");
    gs_f32(out, a.S * dim, p, "out");
    torch::Tensor y = at::empty({a.B, dim}, p.options());
    if (slots.has_value()) {
        TORCH_CHECK(slots->device() == p.device() && slots->is_contiguous() && slots->numel() == a.B &&
                        (slots->scalar_type() == at::kInt || slots->scalar_type() == at::kLong),
                    "gated_step: slots must be contiguous int32 or int64 [B] on the device of p");
        a.slots = slots->data_ptr();
        a.slots64 = slots->scalar_type() == at::kLong;
    } else {
        TORCH_CHECK(a.S == a.B, "gated_step: without slots, state has one row for each row of p");
    }
    a.p = p.data_ptr();
    a.sb = p.stride(0);
    a.state = state.data_ptr<float>();
    a.out = out.data_ptr<float>();
    a.y = y.data_ptr();
    const bool pair = dim % 2 == 0 && a.sb % 2 == 0 && gs_pairs(p) && gs_pairs(y);
    const int64_t lanes = dim / (pair ? 2 : 1);
    const int threads = lanes >= 256 ? 256 : (int)((lanes + 63) / 64 * 64);
    const c10::DeviceGuard guard(p.device());
    GsStepCall call{a, threads, at::hip::getCurrentHIPStream().stream()};
    gs_types(p.scalar_type(), pair, p.size(1) / dim, call);
    C10_HIP_KERNEL_LAUNCH_CHECK();
    // a graph that has kept what was in `out` is told that it changed
    if (!out.is_inference()) out.unsafeGetTensorImpl()->bump_version();
    return y;
}
