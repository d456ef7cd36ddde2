// 8-bit activation checkpoints: writing them, restoring them, and the weight
// gradient of a linear layer from them. Format: checkpoint8.h.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "checkpoint8.h"
#include "launchers.h"

namespace {

typedef __bf16 c8_bf16x8 __attribute__((ext_vector_type(8)));
typedef _Float16 c8_f16x8 __attribute__((ext_vector_type(8)));
typedef float c8_f32x4 __attribute__((ext_vector_type(4)));

// ---------------------------------------------------------------------------
// save8: a group of 32 is eight values in each of four lanes, so that a lane reads 16
// or 32 bytes and writes 8; a lane takes WORK such eights, all loads before the first
// use. load8: the reverse.
// ---------------------------------------------------------------------------
#define C8_WORK 4

template <class E>
struct alignas(16) C8Eight {
    typename E::store v[8];
};

// Eight values of a row of F from column `col` on, 0 behind the row. The hardware loads
// and stores 16 bytes from any address of an element; only the eight at a row's end, if
// it is short, goes value by value.
template <class E>
__device__ __forceinline__ C8Eight<E> c8_take(const typename E::store* row, int col, int F, bool in) {
    C8Eight<E> v;
    if (in && col + 8 <= F) {
        __builtin_memcpy(&v, row + col, sizeof(v));
    } else {
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = in && col + e < F ? row[col + e] : (typename E::store)0;
    }
    return v;
}

// VEC: rows start at 16-byte words and F is a multiple of 8
template <class E, bool VEC>
__global__ __launch_bounds__(256) void c8_save(const typename E::store* x, int64_t sx, signed char* codes,
                                               unsigned char* scales, int64_t N, int F, int Fp) {
    // eights of the padded rows; a multiple of 4, so the lanes of a group stay together
    const unsigned int each = Fp / 8;
    const int64_t all = N * each, from = (int64_t)blockIdx.x * 256 * C8_WORK + threadIdx.x;
    C8Eight<E> v[C8_WORK];
    int64_t row[C8_WORK];
    int col[C8_WORK];
#pragma unroll
    for (int k = 0; k < C8_WORK; ++k) {
        const int64_t i = from + k * 256;
        row[k] = i < all ? i / each : 0;
        col[k] = i < all ? (int)(i - row[k] * each) * 8 : 0;
        const typename E::store* at = x + row[k] * sx;
        if constexpr (VEC) {
            if (i < all && col[k] < F) v[k] = *(const C8Eight<E>*)(at + col[k]);
            else
#pragma unroll
                for (int e = 0; e < 8; ++e) v[k].v[e] = 0;
        } else {
            v[k] = c8_take<E>(at, col[k], F, i < all);
        }
    }
#pragma unroll
    for (int k = 0; k < C8_WORK; ++k) {
        const int64_t i = from + k * 256;
        unsigned int top = 0;
#pragma unroll
        for (int e = 0; e < 8; ++e) top = max(top, c8_mag(E::up(v[k].v[e])));
        const unsigned int s = c8_scale(c8_max4(top));
        const float inv = c8_inv(s);
        unsigned int w[8];
#pragma unroll
        for (int e = 0; e < 8; ++e) w[e] = c8_code_byte(E::up(v[k].v[e]), inv);
        if (i < all) {
            *(uint2*)(codes + row[k] * Fp + col[k]) = uint2{w[0] | w[1] << 8 | w[2] << 16 | w[3] << 24, w[4] | w[5] << 8 | w[6] << 16 | w[7] << 24};
            if (col[k] % C8_GROUP == 0) scales[row[k] * (Fp / C8_GROUP) + col[k] / C8_GROUP] = (unsigned char)s;
        }
    }
}

template <class E, bool VEC>
__global__ __launch_bounds__(256) void c8_load(const signed char* codes, const unsigned char* scales,
                                               typename E::store* x, int64_t N, int F, int Fp) {
    const unsigned int each = Fp / 8;
    const int64_t all = N * each, from = (int64_t)blockIdx.x * 256 * C8_WORK + threadIdx.x;
    uint2 c[C8_WORK];
    unsigned int s[C8_WORK];
    int64_t row[C8_WORK];
    int col[C8_WORK];
#pragma unroll
    for (int k = 0; k < C8_WORK; ++k) {
        const int64_t i = from + k * 256;
        row[k] = i < all ? i / each : 0;
        col[k] = i < all ? (int)(i - row[k] * each) * 8 : 0;
        c[k] = *(const uint2*)(codes + row[k] * Fp + col[k]);
        s[k] = scales[row[k] * (Fp / C8_GROUP) + col[k] / C8_GROUP];
    }
#pragma unroll
    for (int k = 0; k < C8_WORK; ++k) {
        if (from + k * 256 >= all || col[k] >= F) continue;
        const float step = c8_step(s[k]);
        C8Eight<E> v;
#pragma unroll
        for (int e = 0; e < 8; ++e) v.v[e] = E::down((float)(signed char)((e < 4 ? c[k].x : c[k].y) >> (e % 4 * 8)) * step);
        typename E::store* at = x + row[k] * F + col[k];
        if constexpr (VEC) {
            *(C8Eight<E>*)at = v;
        } else if (col[k] + 8 <= F) {
            __builtin_memcpy(at, &v, sizeof(v));
        } else {
#pragma unroll
            for (int e = 0; e < 8; ++e)
                if (col[k] + e < F) at[e] = v.v[e];
        }
    }
}

// ---------------------------------------------------------------------------
// weight gradient: dW[o][f] = sum_n dy[n][o] * x8[n][f], db[o] = sum_n dy[n][o].
//
// Both operands have the summed axis outermost, while a matrix instruction wants
// eight consecutive n of one o or f in a lane. The tiles go to LDS as they lie in
// memory, and the transposing LDS read (ds_read_b64_tr_b16: 16 lanes read four rows
// of 16 columns, each gets one column) turns them on the way to the registers.
// Codes become 16-bit numbers between memory and LDS, exactly, so the product reads
// one byte a value and nothing is restored in memory.
//
// 32-bit dy is taken as a sum of three bf16 numbers (8 + 8 + 8 bits: all of its
// 24), one product each; x8 is exact in bf16.
//
// Rows of a tile are cut into 32-byte chunks, and row k has its chunks permuted by
// (k & 3) + 4 * (k >> 3 & 1): the eight rows that half a wave's transposing read
// takes (0..3 and 8..11 of a fragment) lie in different banks, all 64 of them.
// ---------------------------------------------------------------------------
#define WG_K 64  // rows of dy and x8 that are in LDS at a time
#define WG_THREADS 512

struct WgArgs {
    const void* dy;  // [N][O], rows at sdy
    int64_t sdy;
    const signed char* codes;
    const unsigned char* scales;
    void* dw;      // [O][F] in the output type, or fp32 [splits][O][Fq], Fq = F rounded up to 4
    void* db;      // [O], or fp32 [splits][tiles_f][O rounded up to 4], or null
    int64_t N, per;  // rows, and rows of one split
    int O, F, Fp;
    int tiles_f, tiles_o, splits;
};

template <class E>
struct WgPieces { static const int n = 1; };
template <>
struct WgPieces<C8Fp32> { static const int n = 3; };

__device__ __forceinline__ unsigned int wg_pair(unsigned short a, unsigned short b) { return (unsigned int)a | ((unsigned int)b << 16); }

__device__ __forceinline__ int wg_mix(int k) { return (k & 3) | ((k >> 1) & 4); }

// place of 8 columns (16 bytes), number `c`, of row k in a tile with `pitch` bytes a row
__device__ __forceinline__ int wg_at(int k, int c, int pitch) { return k * pitch + ((((c >> 1) ^ wg_mix(k)) << 5) | ((c & 1) << 4)); }

typedef short wg_s16x4 __attribute__((ext_vector_type(4)));
typedef short wg_s16x8 __attribute__((ext_vector_type(8)));

__device__ __forceinline__ wg_s16x4 wg_turn(const char* at) {
    return __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) wg_s16x4*)at);
}

template <class E>
__device__ __forceinline__ c8_f32x4 wg_mfma(wg_s16x8 a, wg_s16x8 b, c8_f32x4 c) {
    union { wg_s16x8 u; c8_bf16x8 h; c8_f16x8 f; } x, y;
    x.u = a;
    y.u = b;
    if constexpr (std::is_same<E, C8Fp16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.f, y.f, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.h, y.h, c, 0, 0, 0);
}

// What is left of a number after its first piece: of an infinite one nothing. A NaN stays
// one, also where its bits are all in the lower half and the piece is infinite.
__device__ __forceinline__ float wg_rest(float f, float piece) { return __builtin_isinf(f) ? 0.f : f - piece; }

// an offset behind every buffer: for columns that do not exist (a tile's own are below 2^30)
#define WG_OUT 0x7ffffff0

// A buffer of the rows that are left, from this one on: what lies behind them reads as 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wg_rows(const void* at, int64_t left, int64_t row_bytes) {
    const int64_t bytes = left > 0 ? left * row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bytes < WG_OUT ? (int)bytes : WG_OUT, 0x00027000);
}

typedef unsigned int wg_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int wg_u32x2 __attribute__((ext_vector_type(2)));

// eight codes and their scale as 16-bit numbers
template <class E>
__device__ __forceinline__ uint4 wg_decode(uint2 codes, unsigned int scale) {
    const float s = c8_step(scale);
    unsigned int out[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned int w = h == 0 ? codes.x : codes.y;
        const float f0 = (float)(signed char)w * s, f1 = (float)(signed char)(w >> 8) * s;
        const float f2 = (float)(signed char)(w >> 16) * s, f3 = (float)(signed char)(w >> 24) * s;
        if constexpr (std::is_same<E, C8Fp16>::value) {
            out[2 * h] = wg_pair(C8Fp16::down(f0), C8Fp16::down(f1));
            out[2 * h + 1] = wg_pair(C8Fp16::down(f2), C8Fp16::down(f3));
        } else {  // exact: the upper halves are the numbers
            out[2 * h] = __builtin_amdgcn_perm(__float_as_uint(f1), __float_as_uint(f0), 0x07060302u);
            out[2 * h + 1] = __builtin_amdgcn_perm(__float_as_uint(f3), __float_as_uint(f2), 0x07060302u);
        }
    }
    return uint4{out[0], out[1], out[2], out[3]};
}

// four neighbouring values, as one access where rows allow it
template <class G>
__device__ __forceinline__ void wg_store(typename G::store* to, c8_f32x4 v, int f, int F) {
    if ((F & 3) == 0) {
        struct alignas(sizeof(typename G::store) * 4) Four { typename G::store v[4]; };
        *(Four*)to = Four{{G::down(v[0]), G::down(v[1]), G::down(v[2]), G::down(v[3])}};
    } else {
#pragma unroll
        for (int r = 0; r < 4; ++r)
            if (f + r < F) to[r] = G::down(v[r]);
    }
}

// E: type of dy; G: type of the gradient. Eight waves, 2 along O and 4 along F.
template <class E, class G, int BM, int BN, bool ALIGNED>
__global__ __launch_bounds__(WG_THREADS, 2) void c8_weight_grad(WgArgs a) {
    typedef typename std::conditional<std::is_same<E, C8Fp16>::value, C8Fp16, C8Bf16>::type C;  // type of the products
    constexpr int NP = WgPieces<E>::n;
    constexpr int PA = BM * 2, PB = BN * 2;                    // bytes of a tile row
    constexpr int SA = WG_K * PA, SB = WG_K * PB;              // bytes of a tile
    constexpr int CA = BM / 8, CB = BN / 8;                    // eights of a tile row
    constexpr int RA = WG_THREADS / CA, RB = WG_THREADS / CB;  // rows that the block takes at a time
    constexpr int NA = WG_K / RA, NB = WG_K / RB;
    constexpr int MI = BM / 32, NI = BN / 64;
    __shared__ __attribute__((aligned(16))) char lds[2][NP * SA + SB];

    const int tid = threadIdx.x, lane = tid & 63, wid = __builtin_amdgcn_readfirstlane(tid >> 6);
    // Blocks go to the eight XCDs in turn: neighbours in the order of the tiles, which
    // share rows of dy or x8, are given to one XCD and its L2.
    const int total = gridDim.x, each = total >> 3, rest = total & 7, xcd = blockIdx.x & 7;
    const int place = xcd * each + min(xcd, rest) + (blockIdx.x >> 3);
    const int tf = place % a.tiles_f, to = place / a.tiles_f % a.tiles_o, split = place / a.tiles_f / a.tiles_o;
    const int f0 = tf * BN, o0 = to * BM;
    const int64_t n0 = split * a.per, n1 = min(a.N, n0 + a.per);
    const int ng = a.Fp / C8_GROUP;

    const int ca = tid % CA, ra = tid / CA, cb = tid % CB, rb = tid / CB;
    const typename E::store* dy = (const typename E::store*)a.dy;
    constexpr int ES = sizeof(typename E::store);
    // ALIGNED: rows of dy are whole 16-byte words, so are a lane's eight values
    const int oa = o0 + ca * 8 < a.O ? (ra * (int)a.sdy + o0 + ca * 8) * ES : WG_OUT;
    const int fb8 = f0 + cb * 8;
    const int ob = fb8 < a.Fp ? rb * a.Fp + fb8 : WG_OUT;
    // the four lanes of a quad have one group of 32 codes in each of their NB rows: lane i
    // loads the scale of row i, and the others get it from there
    static_assert(NB <= 4, "a scale for each lane of a quad");
    const int os = fb8 < a.Fp ? (rb + (tid % NB) * RB) * ng + fb8 / C8_GROUP : WG_OUT;
    C8Eight<E> va[NA];
    uint2 vb[NB];
    int vs;
    auto load_a = [&](int i, int64_t n) {
        if constexpr (ALIGNED) {
            const auto rows = wg_rows(dy + n * a.sdy, n1 - n, a.sdy * ES);
            const int at = oa + i * RA * (int)a.sdy * ES;
            wg_u32x4* to = (wg_u32x4*)&va[i];
#pragma unroll
            for (int h = 0; h < ES / 2; ++h) to[h] = __builtin_amdgcn_raw_buffer_load_b128(rows, oa == WG_OUT ? WG_OUT : at + h * 16, 0, 0);
        } else {
            const int64_t row = n + ra + i * RA;
            va[i] = c8_take<E>(dy + row * a.sdy, o0 + ca * 8, a.O, row < n1);
        }
    };
    auto load_b = [&](int i, int64_t n) {
        const auto codes = wg_rows(a.codes + n * a.Fp, n1 - n, a.Fp);
        const wg_u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(codes, ob == WG_OUT ? WG_OUT : ob + i * RB * a.Fp, 0, 0);
        vb[i] = uint2{w[0], w[1]};
        if (i == NB - 1) vs = __builtin_amdgcn_raw_buffer_load_b8(wg_rows(a.scales + n * ng, n1 - n, ng), os, 0, 0);
    };
    auto put_a = [&](int i, char* buf) {
        char* at = buf + wg_at(ra + i * RA, ca, PA);
        if constexpr (NP == 1) {
            *(C8Eight<E>*)at = va[i];
        } else {
            float f[8];
#pragma unroll
            for (int e = 0; e < 8; ++e) f[e] = E::up(va[i].v[e]);
#pragma unroll
            for (int q = 0; q < NP; ++q) {
                unsigned int w[4];
#pragma unroll
                for (int e = 0; e < 8; e += 2) {  // cut, not rounded: a large finite number must not become infinite
                    w[e / 2] = __builtin_amdgcn_perm(__float_as_uint(f[e + 1]), __float_as_uint(f[e]), 0x07060302u);
                    f[e] = wg_rest(f[e], __uint_as_float(w[e / 2] << 16));
                    f[e + 1] = wg_rest(f[e + 1], __uint_as_float(w[e / 2] & 0xffff0000u));
                }
                *(uint4*)(at + q * SA) = uint4{w[0], w[1], w[2], w[3]};
            }
        }
    };
    auto put_b = [&](auto piece, char* buf) {
        constexpr int i = decltype(piece)::value;
        const int scale = __builtin_amdgcn_mov_dpp(vs, i * 0x55, 0xF, 0xF, true);  // quad_perm: lane i's to all four
        *(uint4*)(buf + NP * SA + wg_at(rb + i * RB, cb, PB)) = wg_decode<E>(vb[i], scale);
    };

    c8_f32x4 acc[MI][NI];
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) acc[i][j] = c8_f32x4{0.f, 0.f, 0.f, 0.f};

    // a lane's part of a transposing read: row (lane >> 4) * 8 + (lane >> 2 & 3), 4 columns
    const int row = (lane >> 4) * 8 + ((lane >> 2) & 3), sub = (lane & 3) * 8;
    auto frag = [&](const char* tile, int pitch, int chunk, int k) {
        const char* at = tile + (k + row) * pitch + ((chunk ^ wg_mix(row)) << 5) + sub;
        const wg_s16x4 lo = wg_turn(at), hi = wg_turn(at + 4 * pitch);
        return __builtin_shufflevector(lo, hi, 0, 1, 2, 3, 4, 5, 6, 7);
    };
    const int wm = (wid >> 2) * (BM / 2), wn = (wid & 3) * (BN / 4);
    // One step is a fragment of dy against all of x8's. Fragments are read two steps
    // before they are used. Between the steps the next tile is brought to LDS piece by
    // piece and the loads of the one after it go out, so that conversions, LDS writes
    // and loads run beside the matrix instructions. The order is held: left alone, the
    // compiler reads a fragment, waits for it, and the matrix unit waits too.
    auto tile = [&](const char* buf, char* next, int64_t n) {
        constexpr int S = MI * NP, ALL = 2 * S, PIECES = NA + NB;
        wg_s16x8 fa[3], fb[2][NI];
        auto read_a = [&](int s) { return frag(buf + (s % S / MI) * SA, PA, wm / 16 + s % MI, s / S * 32); };
        auto read_b = [&](int j, int k) { return frag(buf + NP * SA, PB, wn / 16 + j, k); };
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[0][j] = read_b(j, 0);
        fa[0] = read_a(0);
        fa[1] = read_a(1);
        c8_for<ALL>([&](auto step) {
            constexpr int s = decltype(step)::value;
            if (s + 2 < ALL) fa[(s + 2) % 3] = read_a(s + 2);
            if (s < NI) fb[1][s] = read_b(s, 32);
            __builtin_amdgcn_sched_barrier(0);
            constexpr int from = s * PIECES / ALL, upto = (s + 1) * PIECES / ALL;
            c8_for<upto - from>([&](auto k) {
                constexpr int piece = from + decltype(k)::value;
                if constexpr (piece < NA) {
                    put_a(piece, next);
                    load_a(piece, n + 2 * WG_K);
                } else {
                    put_b(std::integral_constant<int, piece - NA>{}, next);
                    load_b(piece - NA, n + 2 * WG_K);
                }
            });
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[s % MI][j] = wg_mfma<E>(fb[s / S][j], fa[s % 3], acc[s % MI][j]);
#pragma unroll
            for (int j = 0; j < NI; ++j) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);  // a matrix instruction,
                __builtin_amdgcn_sched_group_barrier(0x002, 8, 0);  // eight vector ones
            }
            __builtin_amdgcn_sched_barrier(0);
        });
    };
    // dy's column sums, from LDS: the blocks of one o take the tiles in turn, so that none
    // has more to do than the others. A thread has a column and a part of its rows.
    constexpr int RS = WG_K * BM / WG_THREADS;
    float sum = 0.f;
    auto add = [&](const char* buf) {
        const int c = tid % BM, r0 = tid / BM * RS;
#pragma unroll 8
        for (int r = r0; r < r0 + RS; ++r) {
            const char* at = buf + wg_at(r, c >> 3, PA) + (c & 7) * 2;
            float v = 0.f;
#pragma unroll
            for (int q = 0; q < NP; ++q) v += C::up(*(const unsigned short*)(at + q * SA));  // exact
            sum += v;
        }
    };

    // behind n1 there are zeros: the last tiles need no case of their own
#pragma unroll
    for (int i = 0; i < NA; ++i) load_a(i, n0);
#pragma unroll
    for (int i = 0; i < NB; ++i) load_b(i, n0);
#pragma unroll
    for (int i = 0; i < NA; ++i) {
        put_a(i, lds[0]);
        load_a(i, n0 + WG_K);
    }
    c8_for<NB>([&](auto i) {
        put_b(i, lds[0]);
        load_b(decltype(i)::value, n0 + WG_K);
    });
    __syncthreads();
    int buf = 0, turn = 0;
    for (int64_t n = n0; n < n1; n += WG_K) {
        if (a.db != nullptr && turn == tf) add(lds[buf]);
        turn = turn + 1 == a.tiles_f ? 0 : turn + 1;
        tile(lds[buf], lds[buf ^ 1], n);
        buf ^= 1;
        __syncthreads();
    }

    // a lane holds four f, at (lane >> 4) * 4, of one o, lane & 15
    const int Fq = (a.F + 3) & ~3;
    const int64_t slab = (int64_t)split * a.O * Fq;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int o = o0 + wm + i * 16 + (lane & 15), f = f0 + wn + j * 16 + (lane >> 4) * 4;
            if (o >= a.O || f >= a.F) continue;
            if (a.splits > 1) wg_store<C8Fp32>((float*)a.dw + slab + (int64_t)o * Fq + f, acc[i][j], f, Fq);
            else wg_store<G>((typename G::store*)a.dw + (int64_t)o * a.F + f, acc[i][j], f, a.F);
        }
    if (a.db != nullptr) {
        float* part = (float*)lds;  // [WG_THREADS / BM][BM]
        part[tid] = sum;
        __syncthreads();
        if (tid < BM && o0 + tid < a.O) {
            float v = 0.f;
#pragma unroll
            for (int r = 0; r < WG_THREADS / BM; ++r) v += part[r * BM + tid];
            if (a.splits * a.tiles_f > 1) ((float*)a.db)[((int64_t)split * a.tiles_f + tf) * ((a.O + 3) & ~3) + o0 + tid] = v;
            else ((typename G::store*)a.db)[o0 + tid] = G::down(v);
        }
    }
}

// Sums of parts in their order: [parts][rows][pitch] to [rows][F], four values a lane.
struct C8Join {
    const float* from;
    void* to;
    int64_t rows;
    int F, pitch, parts;
    unsigned int blocks;
};

// the weight's sums and the bias's in one launch
template <class G>
__global__ __launch_bounds__(256) void c8_join(C8Join w, C8Join b) {
    const bool bias = blockIdx.x >= w.blocks;
    const C8Join& j = bias ? b : w;
    const int64_t fours = j.pitch / 4, n = j.rows * fours;
    for (int64_t i = (int64_t)(blockIdx.x - (bias ? w.blocks : 0)) * 256 + threadIdx.x; i < n; i += (int64_t)j.blocks * 256) {
        const int64_t r = i / fours;
        const int f = (int)(i - r * fours) * 4;
        c8_f32x4 v = {0.f, 0.f, 0.f, 0.f};
#pragma unroll 4
        for (int s = 0; s < j.parts; ++s) v += *(const c8_f32x4*)(j.from + (int64_t)s * j.rows * j.pitch + i * 4);
        wg_store<G>((typename G::store*)j.to + r * j.F + f, v, f, j.F);
    }
}

template <class F>
void c8_type(at::ScalarType dt, const char* what, F&& f) {
    if (dt == at::kBFloat16) f(C8Bf16{});
    else if (dt == at::kHalf) f(C8Fp16{});
    else if (dt == at::kFloat) f(C8Fp32{});
    else TORCH_CHECK(false, what, " must be float32, bfloat16 or float16");
}

unsigned int c8_blocks(int64_t lanes) {
    int64_t n = (lanes + 255) / 256;
    return (unsigned int)(n < 1 ? 1 : (n > 65536 ? 65536 : n));
}

unsigned int c8_works(int64_t eights) {
    const int64_t n = (eights + 256 * C8_WORK - 1) / (256 * C8_WORK);
    TORCH_CHECK(n * 256 <= UINT32_MAX, "checkpoint8: too many values");  // a launch takes fewer than 2^32 threads
    return (unsigned int)n;
}

void c8_check(const torch::Tensor& codes, const torch::Tensor& scales, int64_t N, int64_t F) {
    const int64_t Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    TORCH_CHECK(F > 0 && F <= INT_MAX - C8_GROUP, "checkpoint8: row length out of range");
    TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device() && codes.scalar_type() == at::kChar &&
                    scales.scalar_type() == at::kByte && codes.is_contiguous() && scales.is_contiguous() &&
                    codes.numel() == N * Fp && scales.numel() == N * (Fp / C8_GROUP),
                "checkpoint8: codes and scales do not match ", N, " rows of ", F);
    TORCH_CHECK((uintptr_t)codes.data_ptr() % 16 == 0, "checkpoint8: codes must be 16-byte aligned");
}

// Side of the tiles, and parts that the rows are split into. The least of what was
// measured, in us: a step of 64 rows takes 2.5 in 256 x 256 tiles (one block a CU),
// 1.2 in 128 x 128 ones, 1.85 with two of those on a CU; beyond that blocks follow one
// another; parts are written and read again at 5 TB/s. E.g. 16384 rows, 4096 x 2048:
// 256 x 2 parts 330 + join, 128 x 1 part 457; 2048 rows, 2048 x 2048: 128 x 1 part 43,
// 256 x 4 parts 36 + join. 32-bit dy has three products a step, small tiles only
// (three pieces of dy in LDS) and one block a CU.
struct WgPlan {
    int side, splits;
    int64_t steps;
};

WgPlan wg_plan(int64_t N, int64_t O, int64_t F, bool pieces) {
    WgPlan best{128, 1, std::max<int64_t>(1, (N + WG_K - 1) / WG_K)};
    double least = 1e30;
    for (int side = pieces ? 128 : 256; side >= 128; side -= 128) {
        if (side == 256 && (O <= 128 || F <= 128)) continue;
        const int64_t tiles = ((O + side - 1) / side) * ((F + side - 1) / side);
        for (int s : {1, 2, 3, 4, 5, 6, 8, 10, 12, 16, 20, 24, 32, 48, 64}) {
            const int64_t steps = std::max<int64_t>(1, (N + (int64_t)s * WG_K - 1) / ((int64_t)s * WG_K));
            if (s > 1 && (s - 1) * steps * WG_K >= N) continue;  // an empty part
            const int64_t blocks = tiles * s;
            double t = 4;
            if (side == 256) t += (blocks + 255) / 256 * steps * 2.5;
            else if (pieces) t += (blocks + 255) / 256 * steps * 3.0;
            else t += (blocks / 512) * steps * 1.85 + (blocks % 512 == 0 ? 0 : blocks % 512 <= 256 ? steps * 1.2 : steps * 1.85);
            if (s > 1) t += 2 * s * (double)O * F * 4 / 5e6 + 4;
            if (t < least) {
                least = t;
                best = WgPlan{side, s, steps};
            }
        }
    }
    return best;
}

}  // namespace

std::tuple<torch::Tensor, torch::Tensor> save8_launch(torch::Tensor x) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1), "save8: x must be two-dimensional on the GPU, unit stride last");
    const int64_t N = x.size(0), F = x.size(1), Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    TORCH_CHECK(F > 0 && F <= INT_MAX - C8_GROUP, "save8: row length out of range");
    torch::Tensor codes = at::empty({N, Fp}, x.options().dtype(at::kChar));
    torch::Tensor scales = at::empty({N, Fp / C8_GROUP}, x.options().dtype(at::kByte));
    if (N == 0) return {codes, scales};
    const c10::DeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    c8_type(x.scalar_type(), "save8: x", [&](auto e) {
        typedef decltype(e) E;
        const bool vec = F % 8 == 0 && x.stride(0) * x.element_size() % 16 == 0 && (uintptr_t)x.data_ptr() % 16 == 0;
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(c8_works(N * (Fp / 8))), dim3(256), 0, stream, (const typename E::store*)x.data_ptr(),
                               x.stride(0), (signed char*)codes.data_ptr(), (unsigned char*)scales.data_ptr(), N, (int)F, (int)Fp);
        };
        if (vec) go(c8_save<E, true>);
        else go(c8_save<E, false>);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return {codes, scales};
}

torch::Tensor load8_launch(torch::Tensor codes, torch::Tensor scales, int64_t F, at::ScalarType dtype) {
    TORCH_CHECK(codes.dim() == 2 && F > 0, "load8: codes must be two-dimensional");
    const int64_t N = codes.size(0), Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    c8_check(codes, scales, N, F);
    torch::Tensor x = at::empty({N, F}, codes.options().dtype(dtype));
    if (N == 0) return x;
    const c10::DeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    c8_type(x.scalar_type(), "load8: x", [&](auto e) {
        typedef decltype(e) E;
        const auto go = [&](auto kernel) {
            hipLaunchKernelGGL(kernel, dim3(c8_works(N * (Fp / 8))), dim3(256), 0, stream, (const signed char*)codes.data_ptr(),
                               (const unsigned char*)scales.data_ptr(), (typename E::store*)x.data_ptr(), N, (int)F, (int)Fp);
        };
        if (F % 8 == 0 && (uintptr_t)x.data_ptr() % 16 == 0) go(c8_load<E, true>);
        else go(c8_load<E, false>);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
    return x;
}

void weight_grad8_launch(torch::Tensor dy, torch::Tensor codes, torch::Tensor scales, torch::Tensor dw,
                         c10::optional<torch::Tensor> db) {
    TORCH_CHECK(dy.is_cuda() && dy.dim() == 2 && (dy.size(1) == 1 || dy.stride(1) == 1), "weight_grad8: dy must be two-dimensional on the GPU, unit stride last");
    TORCH_CHECK(dw.device() == dy.device() && dw.dim() == 2 && dw.is_contiguous() && dw.size(0) == dy.size(1),
                "weight_grad8: dw must be contiguous [O, F] on the device of dy");
    const int64_t N = dy.size(0), O = dy.size(1), F = dw.size(1), Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    c8_check(codes, scales, N, F);
    TORCH_CHECK(codes.device() == dy.device(), "weight_grad8: dy and the codes are on different devices");
    TORCH_CHECK(O > 0 && O <= (1 << 24) && F <= (1 << 24), "weight_grad8: O or F out of range");
    if (db.has_value())
        TORCH_CHECK(db->device() == dy.device() && db->is_contiguous() && db->numel() == O && db->scalar_type() == dw.scalar_type(),
                    "weight_grad8: db must be contiguous [O] of the type of dw");
    const c10::DeviceGuard guard(dy.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    WgArgs a{};
    a.dy = dy.data_ptr();
    a.sdy = dy.stride(0);
    a.codes = (const signed char*)codes.data_ptr();
    a.scales = (const unsigned char*)scales.data_ptr();
    a.N = N;
    a.O = (int)O;
    a.F = (int)F;
    a.Fp = (int)Fp;
    const WgPlan plan = wg_plan(N, O, F, dy.scalar_type() == at::kFloat);
    const bool wide = plan.side == 256;
    a.tiles_f = (int)((F + plan.side - 1) / plan.side);
    a.tiles_o = (int)((O + plan.side - 1) / plan.side);
    const int64_t tiles = (int64_t)a.tiles_f * a.tiles_o, Fq = (F + 3) / 4 * 4, Oq = (O + 3) / 4 * 4;
    a.per = plan.steps * WG_K;
    a.splits = plan.splits;
    TORCH_CHECK(tiles * a.splits * WG_THREADS <= UINT32_MAX, "weight_grad8: sizes out of range");
    // whole 16-byte words, and a tile's rows within 31-bit offsets
    const bool aligned = O % 8 == 0 && a.sdy % 8 == 0 && a.sdy >= O && a.sdy <= (1 << 22) && (uintptr_t)a.dy % 16 == 0;
    torch::Tensor part, part_b;
    const bool join = a.splits > 1, join_b = db.has_value() && a.splits * a.tiles_f > 1;
    const auto f32 = dw.options().dtype(at::kFloat);
    a.dw = dw.data_ptr();
    a.db = db.has_value() ? db->data_ptr() : nullptr;
    if (join) {
        part = torch::empty({a.splits, O, Fq}, f32);
        a.dw = part.data_ptr();
    }
    if (join_b) {
        part_b = torch::empty({a.splits * a.tiles_f, Oq}, f32);
        a.db = part_b.data_ptr();
    }
    const dim3 grid((unsigned)(tiles * a.splits));
    c8_type(dy.scalar_type(), "weight_grad8: dy", [&](auto e) {
        c8_type(dw.scalar_type(), "weight_grad8: dw", [&](auto g) {
            typedef decltype(e) E;
            typedef decltype(g) G;
            if constexpr (WgPieces<E>::n == 1) {
                if (wide && aligned) hipLaunchKernelGGL((c8_weight_grad<E, G, 256, 256, true>), grid, dim3(WG_THREADS), 0, stream, a);
                else if (wide) hipLaunchKernelGGL((c8_weight_grad<E, G, 256, 256, false>), grid, dim3(WG_THREADS), 0, stream, a);
            }
            if (!wide && aligned) hipLaunchKernelGGL((c8_weight_grad<E, G, 128, 128, true>), grid, dim3(WG_THREADS), 0, stream, a);
            else if (!wide) hipLaunchKernelGGL((c8_weight_grad<E, G, 128, 128, false>), grid, dim3(WG_THREADS), 0, stream, a);
            if (join || join_b) {
                C8Join w{}, b{};
                if (join) w = {(const float*)part.data_ptr(), dw.data_ptr(), O, (int)F, (int)Fq, a.splits, c8_blocks(O * Fq / 4)};
                if (join_b) b = {(const float*)part_b.data_ptr(), db->data_ptr(), 1, (int)O, (int)Oq, a.splits * a.tiles_f, c8_blocks(Oq / 4)};
                hipLaunchKernelGGL((c8_join<G>), dim3(w.blocks + b.blocks), dim3(256), 0, stream, w, b);
            }
        });
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
}
