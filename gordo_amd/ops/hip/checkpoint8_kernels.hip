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
// save8: a group of 32 is two values in each of 16 lanes. load8: the reverse.
// ---------------------------------------------------------------------------
template <class E>
__global__ __launch_bounds__(256) void c8_save(const typename E::store* x, int64_t sx, signed char* codes,
                                               unsigned char* scales, int64_t N, int F, int Fp) {
    const int64_t ng = Fp / C8_GROUP, all = N * ng * 16;
    const int64_t step = (int64_t)gridDim.x * 256;
    // `all` is a multiple of 16: the lanes of a group stay together
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
        const int64_t row = i / (ng * 16);
        const int col = (int)(i - row * ng * 16) * 2;
        const float a = col < F ? E::up(x[row * sx + col]) : 0.f;
        const float b = col + 1 < F ? E::up(x[row * sx + col + 1]) : 0.f;
        const unsigned int s = c8_scale(c8_max16(max(c8_mag(a), c8_mag(b))));
        const float inv = c8_inv(s);
        *(unsigned short*)(codes + row * Fp + col) = (unsigned short)(c8_code_byte(a, inv) | (c8_code_byte(b, inv) << 8));
        if (col % C8_GROUP == 0) scales[row * ng + col / C8_GROUP] = (unsigned char)s;
    }
}

template <class E>
__global__ __launch_bounds__(256) void c8_load(const signed char* codes, const unsigned char* scales,
                                               typename E::store* x, int64_t N, int F, int Fp) {
    const int64_t ng = Fp / C8_GROUP, all = N * F;
    const int64_t step = (int64_t)gridDim.x * 256;
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < all; i += step) {
        const int64_t row = i / F;
        const int col = (int)(i - row * F);
        x[i] = E::down((float)codes[row * Fp + col] * c8_step(scales[row * ng + col / C8_GROUP]));
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
    void* dw;      // [O][F] in the output type, or fp32 [splits][O][F]
    void* db;      // [O], or fp32 [splits][O], or null
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

// eight neighbouring values of a row of dy
template <class E>
struct WgEight {
    typename E::store v[8];
};

// A buffer of the rows that are left, from this one on: what lies behind them reads as 0.
__device__ __forceinline__ __amdgpu_buffer_rsrc_t wg_rows(const void* at, int64_t left, int64_t row_bytes) {
    const int64_t bytes = left > 0 ? left * row_bytes : 0;
    return __builtin_amdgcn_make_buffer_rsrc((void*)at, 0, bytes < 0x7fffffff ? (int)bytes : 0x7fffffff, 0x00027000);
}

#define WG_OUT 0x7ffffff0  // an offset behind every buffer

typedef unsigned int wg_u32x4 __attribute__((ext_vector_type(4)));
typedef unsigned int wg_u32x2 __attribute__((ext_vector_type(2)));

// eight codes and their scale as 16-bit numbers
template <class E>
__device__ __forceinline__ uint4 wg_decode(uint2 codes, unsigned int scale) {
    const float s = c8_step(scale), off = -128.f * s;
    unsigned int out[4];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const unsigned int w = (h == 0 ? codes.x : codes.y) ^ 0x80808080u;  // code + 128, unsigned
        const float f0 = fmaf((float)(w & 0xff), s, off), f1 = fmaf((float)((w >> 8) & 0xff), s, off);
        const float f2 = fmaf((float)((w >> 16) & 0xff), s, off), f3 = fmaf((float)(w >> 24), s, off);
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
    const int ob = fb8 < a.Fp ? rb * a.Fp + fb8 : WG_OUT, os = fb8 < a.Fp ? rb * ng + fb8 / C8_GROUP : WG_OUT;
    WgEight<E> va[NA];
    uint2 vb[NB];
    unsigned int vs[NB];
    auto load = [&](int64_t n) {
        if constexpr (ALIGNED) {
            const auto rows = wg_rows(dy + n * a.sdy, n1 - n, a.sdy * ES);
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int at = oa + i * RA * (int)a.sdy * ES;
                wg_u32x4* to = (wg_u32x4*)&va[i];
#pragma unroll
                for (int h = 0; h < ES / 2; ++h) to[h] = __builtin_amdgcn_raw_buffer_load_b128(rows, oa == WG_OUT ? WG_OUT : at + h * 16, 0, 0);
            }
        } else {
#pragma unroll
            for (int i = 0; i < NA; ++i) {
                const int64_t row = n + ra + i * RA;
#pragma unroll
                for (int e = 0; e < 8; ++e) {
                    const int o = o0 + ca * 8 + e;
                    va[i].v[e] = row < n1 && o < a.O ? dy[row * a.sdy + o] : (typename E::store)0;
                }
            }
        }
        const auto codes = wg_rows(a.codes + n * a.Fp, n1 - n, a.Fp), scales = wg_rows(a.scales + n * ng, n1 - n, ng);
#pragma unroll
        for (int i = 0; i < NB; ++i) {
            const wg_u32x2 w = __builtin_amdgcn_raw_buffer_load_b64(codes, ob == WG_OUT ? WG_OUT : ob + i * RB * a.Fp, 0, 0);
            vb[i] = uint2{w[0], w[1]};
            vs[i] = __builtin_amdgcn_raw_buffer_load_b8(scales, os == WG_OUT ? WG_OUT : os + i * RB * ng, 0, 0);
        }
    };
    const bool sums = tf == 0 && a.db != nullptr;
    float sum[8] = {0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f, 0.f};
    auto put = [&](char* buf) {
#pragma unroll
        for (int i = 0; i < NA; ++i) {
            char* at = buf + wg_at(ra + i * RA, ca, PA);
            if constexpr (NP == 1) {
                *(WgEight<E>*)at = va[i];
            } else {
                float f[8];
#pragma unroll
                for (int e = 0; e < 8; ++e) f[e] = E::up(va[i].v[e]);
#pragma unroll
                for (int q = 0; q < NP; ++q) {
                    unsigned short h[8];
#pragma unroll
                    for (int e = 0; e < 8; ++e) {
                        h[e] = C8Bf16::down(f[e]);
                        f[e] -= C8Bf16::up(h[e]);
                    }
                    *(uint4*)(at + q * SA) = uint4{wg_pair(h[0], h[1]), wg_pair(h[2], h[3]), wg_pair(h[4], h[5]), wg_pair(h[6], h[7])};
                }
            }
            if (sums) {
#pragma unroll
                for (int e = 0; e < 8; ++e) sum[e] += E::up(va[i].v[e]);
            }
        }
#pragma unroll
        for (int i = 0; i < NB; ++i) *(uint4*)(buf + NP * SA + wg_at(rb + i * RB, cb, PB)) = wg_decode<E>(vb[i], vs[i]);
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
    // before they are used, and the order is held: left alone, the compiler reads one,
    // waits for it, and the matrix unit waits too.
    auto work = [&](const char* buf) {
        constexpr int S = MI * NP, ALL = 2 * S;
        wg_s16x8 fa[3], fb[2][NI];
        auto read_a = [&](int s) { return frag(buf + (s % S / MI) * SA, PA, wm / 16 + s % MI, s / S * 32); };
        auto read_b = [&](int j, int k) { return frag(buf + NP * SA, PB, wn / 16 + j, k); };
#pragma unroll
        for (int j = 0; j < NI; ++j) fb[0][j] = read_b(j, 0);
        fa[0] = read_a(0);
        fa[1] = read_a(1);
#pragma unroll
        for (int s = 0; s < ALL; ++s) {
            if (s + 2 < ALL) fa[(s + 2) % 3] = read_a(s + 2);
            if (s < NI) fb[1][s] = read_b(s, 32);
            __builtin_amdgcn_sched_barrier(0);
#pragma unroll
            for (int j = 0; j < NI; ++j) acc[s % MI][j] = wg_mfma<E>(fb[s / S][j], fa[s % 3], acc[s % MI][j]);
            __builtin_amdgcn_sched_barrier(0);
        }
    };

    // Two waves share a SIMD, wid and wid + 4. One decodes the next tile before its
    // products and the other after them, so that one's conversions and LDS writes run
    // beside the other's matrix instructions. Loads are a whole tile ahead either way.
    const bool early = wid < 4;
    int buf = 0;
    load(n0);
    put(lds[0]);
    load(n0 + WG_K);  // rows behind n1 are zeros
    __syncthreads();
    for (int64_t n = n0; n < n1; n += WG_K) {
        const bool more = n + WG_K < n1;
        if (early && more) {
            put(lds[buf ^ 1]);
            load(n + 2 * WG_K);
        }
        work(lds[buf]);
        buf ^= 1;
        if (!early && more) {
            put(lds[buf]);
            load(n + 2 * WG_K);
        }
        __syncthreads();
    }

    // a lane holds four f, at (lane >> 4) * 4, of one o, lane & 15
    const int64_t slab = (int64_t)split * a.O * a.F;
#pragma unroll
    for (int i = 0; i < MI; ++i)
#pragma unroll
        for (int j = 0; j < NI; ++j) {
            const int o = o0 + wm + i * 16 + (lane & 15), f = f0 + wn + j * 16 + (lane >> 4) * 4;
            if (o >= a.O || f >= a.F) continue;
            const int64_t at = (int64_t)o * a.F + f;
            if (a.splits > 1) wg_store<C8Fp32>((float*)a.dw + slab + at, acc[i][j], f, a.F);
            else wg_store<G>((typename G::store*)a.dw + at, acc[i][j], f, a.F);
        }
    if (sums) {
        float* part = (float*)lds;  // [RA][BM]
#pragma unroll
        for (int e = 0; e < 8; ++e) part[ra * BM + ca * 8 + e] = sum[e];
        __syncthreads();
        if (tid < BM && o0 + tid < a.O) {
            float v = 0.f;
            for (int r = 0; r < RA; ++r) v += part[r * BM + tid];
            if (a.splits > 1) ((float*)a.db)[(int64_t)split * a.O + o0 + tid] = v;
            else ((typename G::store*)a.db)[o0 + tid] = G::down(v);
        }
    }
}

// sums the splits in their order
template <class G>
__global__ __launch_bounds__(256) void c8_join(const float* part, typename G::store* out, int64_t n, int splits) {
    for (int64_t i = (int64_t)blockIdx.x * 256 + threadIdx.x; i < n; i += (int64_t)gridDim.x * 256) {
        float v = 0.f;
        for (int s = 0; s < splits; ++s) v += part[s * n + i];
        out[i] = G::down(v);
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

void c8_check(const torch::Tensor& codes, const torch::Tensor& scales, int64_t N, int64_t F) {
    const int64_t Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    TORCH_CHECK(F > 0 && F <= INT_MAX - C8_GROUP, "checkpoint8: row length out of range");
    TORCH_CHECK(codes.is_cuda() && scales.device() == codes.device() && codes.scalar_type() == at::kChar &&
                    scales.scalar_type() == at::kByte && codes.is_contiguous() && scales.is_contiguous() &&
                    codes.numel() == N * Fp && scales.numel() == N * (Fp / C8_GROUP),
                "checkpoint8: codes and scales do not match ", N, " rows of ", F);
    TORCH_CHECK((uintptr_t)codes.data_ptr() % 16 == 0, "checkpoint8: codes must be 16-byte aligned");
}

}  // namespace

void save8_launch(torch::Tensor x, torch::Tensor codes, torch::Tensor scales) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && (x.size(1) == 1 || x.stride(1) == 1), "save8: x must be two-dimensional on the GPU, unit stride last");
    const int64_t N = x.size(0), F = x.size(1), Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    c8_check(codes, scales, N, F);
    TORCH_CHECK(codes.device() == x.device(), "save8: x and its codes are on different devices");
    if (N == 0) return;
    const c10::DeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    c8_type(x.scalar_type(), "save8: x", [&](auto e) {
        typedef decltype(e) E;
        hipLaunchKernelGGL((c8_save<E>), dim3(c8_blocks(N * Fp / 2)), dim3(256), 0, stream, 
            (const typename E::store*)x.data_ptr(), x.stride(0), (signed char*)codes.data_ptr(),
            (unsigned char*)scales.data_ptr(), N, (int)F, (int)Fp);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
}

void load8_launch(torch::Tensor codes, torch::Tensor scales, torch::Tensor x) {
    TORCH_CHECK(x.is_cuda() && x.dim() == 2 && x.is_contiguous(), "load8: x must be two-dimensional and contiguous on the GPU");
    const int64_t N = x.size(0), F = x.size(1), Fp = (F + C8_GROUP - 1) / C8_GROUP * C8_GROUP;
    c8_check(codes, scales, N, F);
    TORCH_CHECK(codes.device() == x.device(), "load8: x and its codes are on different devices");
    if (N == 0) return;
    const c10::DeviceGuard guard(x.device());
    auto stream = at::hip::getCurrentHIPStream().stream();
    c8_type(x.scalar_type(), "load8: x", [&](auto e) {
        typedef decltype(e) E;
        hipLaunchKernelGGL((c8_load<E>), dim3(c8_blocks(N * F)), dim3(256), 0, stream, 
            (const signed char*)codes.data_ptr(), (const unsigned char*)scales.data_ptr(),
            (typename E::store*)x.data_ptr(), N, (int)F, (int)Fp);
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
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
    // Tiles of 256 x 256 read each operand least; 128 x 128 where those are too few, or
    // three pieces of dy would not fit LDS.
    const bool wide = dy.scalar_type() != at::kFloat && O > 128 && F > 128 && ((O + 255) / 256) * ((F + 255) / 256) * ((N + 511) / 512) >= 128;
    const int64_t side = wide ? 256 : 128;
    a.tiles_f = (int)((F + side - 1) / side);
    a.tiles_o = (int)((O + side - 1) / side);
    const int64_t tiles = (int64_t)a.tiles_f * a.tiles_o;
    // blocks for the chip (one a CU, or two of the small ones), but at least 256 rows a split
    int64_t splits = std::min<int64_t>((wide ? 256 : 512) / tiles, (N + 255) / 256);
    splits = std::max<int64_t>(1, splits);
    a.per = (((N + splits - 1) / splits) + WG_K - 1) / WG_K * WG_K;
    a.splits = (int)(a.per > 0 ? std::max<int64_t>(1, (N + a.per - 1) / a.per) : 1);
    TORCH_CHECK(tiles * a.splits <= INT_MAX, "weight_grad8: sizes out of range");
    // whole 16-byte words, and a tile's rows within 31-bit offsets
    const bool aligned = O % 8 == 0 && a.sdy % 8 == 0 && a.sdy >= O && a.sdy <= (1 << 22) && (uintptr_t)a.dy % 16 == 0;
    torch::Tensor part, part_b;
    const bool join = a.splits > 1;
    if (join) {
        auto opt = dw.options().dtype(at::kFloat);
        part = torch::empty({a.splits, O, F}, opt);
        a.dw = part.data_ptr();
        if (db.has_value()) {
            part_b = torch::empty({a.splits, O}, opt);
            a.db = part_b.data_ptr();
        }
    } else {
        a.dw = dw.data_ptr();
        a.db = db.has_value() ? db->data_ptr() : nullptr;
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
            if (join) {
                hipLaunchKernelGGL((c8_join<G>), dim3(c8_blocks(O * F)), dim3(256), 0, stream, (const float*)part.data_ptr(), (typename G::store*)dw.data_ptr(), O * F, a.splits);
                if (db.has_value())
                    hipLaunchKernelGGL((c8_join<G>), dim3(c8_blocks(O)), dim3(256), 0, stream, (const float*)part_b.data_ptr(), (typename G::store*)db->data_ptr(), O, a.splits);
            }
        });
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
}
