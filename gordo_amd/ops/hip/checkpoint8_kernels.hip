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
typedef unsigned short c8_u16x8 __attribute__((ext_vector_type(8)));

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
// Both operands have the summed axis outermost, so tiles go to LDS transposed.
// 32-bit dy is taken as a sum of three bf16 numbers (8 + 8 + 8 bits: all of its
// 24), one product each; x8 is exact in bf16 and in fp16.
// ---------------------------------------------------------------------------
#define WG_M 128
#define WG_N 128
#define WG_K 32
#define WG_PITCH 40  // 16-bit elements of a tile row: 32 and a pad, rows stay 16-byte aligned

struct WgArgs {
    const void* dy;  // [N][O], rows at sdy
    int64_t sdy;
    const signed char* codes;
    const unsigned char* scales;
    void* dw;      // [O][F] in the output type, or fp32 [splits][O][F]
    void* db;      // [O], or fp32 [splits][O], or null
    int64_t N, per;  // rows, and rows of one split
    int O, F, Fp;
    int splits;
};

// pieces of one dy value as 16-bit patterns
__device__ __forceinline__ void wg_pieces(C8Bf16, unsigned short u, unsigned short* o) { o[0] = u; }
__device__ __forceinline__ void wg_pieces(C8Fp16, unsigned short u, unsigned short* o) { o[0] = u; }
__device__ __forceinline__ void wg_pieces(C8Fp32, float f, unsigned short* o) {
#pragma unroll
    for (int j = 0; j < 3; ++j) {
        o[j] = C8Bf16::down(f);
        f -= C8Bf16::up(o[j]);
    }
}

template <class E>
struct WgPieces { static const int n = 1; };
template <>
struct WgPieces<C8Fp32> { static const int n = 3; };

template <class E>
__device__ __forceinline__ c8_f32x4 wg_mfma(c8_u16x8 a, c8_u16x8 b, c8_f32x4 c) {
    union { c8_u16x8 u; c8_bf16x8 h; c8_f16x8 f; } x, y;
    x.u = a;
    y.u = b;
    if constexpr (std::is_same<E, C8Fp16>::value) return __builtin_amdgcn_mfma_f32_16x16x32_f16(x.f, y.f, c, 0, 0, 0);
    else return __builtin_amdgcn_mfma_f32_16x16x32_bf16(x.h, y.h, c, 0, 0, 0);
}

// E: type of dy; G: type of the gradient; C: type that x8 is multiplied in
template <class E, class G>
__global__ __launch_bounds__(256) void c8_weight_grad(WgArgs a) {
    typedef typename std::conditional<std::is_same<E, C8Fp16>::value, C8Fp16, C8Bf16>::type C;
    const int NP = WgPieces<E>::n;
    __shared__ __attribute__((aligned(16))) unsigned short A[WgPieces<E>::n][WG_M][WG_PITCH];
    __shared__ __attribute__((aligned(16))) unsigned short B[WG_N][WG_PITCH];
    const int tid = threadIdx.x, lane = tid & 63, wid = tid >> 6;
    const int f0 = blockIdx.x * WG_N, o0 = blockIdx.y * WG_M;
    const int64_t n0 = blockIdx.z * a.per, n1 = min(a.N, n0 + a.per);
    const typename E::store* dy = (const typename E::store*)a.dy;
    const int ng = a.Fp / C8_GROUP;
    const int wm = (wid >> 1) * 64, wn = (wid & 1) * 64;

    c8_f32x4 acc[4][4];
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j) acc[i][j] = c8_f32x4{0.f, 0.f, 0.f, 0.f};
    float sum = 0.f;  // of dy's column o0 + tid

    for (int64_t n = n0; n < n1; n += WG_K) {
        __syncthreads();
        for (int e = tid; e < WG_K * WG_M; e += 256) {
            const int r = e / WG_M, c = e % WG_M;
            unsigned short o[3] = {0, 0, 0};
            if (n + r < n1 && o0 + c < a.O) wg_pieces(E{}, dy[(n + r) * a.sdy + o0 + c], o);
#pragma unroll
            for (int j = 0; j < NP; ++j) A[j][c][r] = o[j];
        }
        for (int e = tid; e < WG_K * WG_N; e += 256) {
            const int r = e / WG_N, c = e % WG_N;
            float v = 0.f;
            if (n + r < n1 && f0 + c < a.F)
                v = (float)a.codes[(n + r) * a.Fp + f0 + c] * c8_step(a.scales[(n + r) * ng + (f0 + c) / C8_GROUP]);
            B[c][r] = C::down(v);
        }
        __syncthreads();
        if (blockIdx.x == 0 && a.db != nullptr && tid < WG_M) {
            for (int r = 0; r < WG_K; ++r) {
                float v = 0.f;
#pragma unroll
                for (int j = 0; j < NP; ++j) v += C::up(A[j][tid][r]);
                sum += v;
            }
        }
        c8_u16x8 fb[4];
#pragma unroll
        for (int j = 0; j < 4; ++j) fb[j] = *(const c8_u16x8*)&B[wn + j * 16 + (lane & 15)][(lane >> 4) * 8];
#pragma unroll
        for (int q = 0; q < NP; ++q) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const c8_u16x8 fa = *(const c8_u16x8*)&A[q][wm + i * 16 + (lane & 15)][(lane >> 4) * 8];
#pragma unroll
                for (int j = 0; j < 4; ++j) acc[i][j] = wg_mfma<E>(fa, fb[j], acc[i][j]);
            }
        }
    }
    // a lane holds rows (lane >> 4) * 4 + r of column lane & 15
    const int64_t slab = (int64_t)blockIdx.z * a.O * a.F;
#pragma unroll
    for (int i = 0; i < 4; ++i)
#pragma unroll
        for (int j = 0; j < 4; ++j)
#pragma unroll
            for (int r = 0; r < 4; ++r) {
                const int o = o0 + wm + i * 16 + (lane >> 4) * 4 + r, f = f0 + wn + j * 16 + (lane & 15);
                if (o < a.O && f < a.F) {
                    const int64_t at = (int64_t)o * a.F + f;
                    if (a.splits > 1) ((float*)a.dw)[slab + at] = acc[i][j][r];
                    else ((typename G::store*)a.dw)[at] = G::down(acc[i][j][r]);
                }
            }
    if (blockIdx.x == 0 && a.db != nullptr && tid < WG_M && o0 + tid < a.O) {
        if (a.splits > 1) ((float*)a.db)[(int64_t)blockIdx.z * a.O + o0 + tid] = sum;
        else ((typename G::store*)a.db)[o0 + tid] = G::down(sum);
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
    TORCH_CHECK(O > 0 && O <= INT_MAX - WG_M, "weight_grad8: O out of range");
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
    const int64_t tf = (F + WG_N - 1) / WG_N, to = (O + WG_M - 1) / WG_M;
    TORCH_CHECK(to <= 65535, "weight_grad8: O out of range");
    // enough blocks for the chip, but at least 256 rows a split
    int64_t splits = std::min<int64_t>(512 / (tf * to), (N + 255) / 256);
    splits = std::max<int64_t>(1, splits);
    a.per = (((N + splits - 1) / splits) + WG_K - 1) / WG_K * WG_K;
    a.splits = (int)(a.per > 0 ? std::max<int64_t>(1, (N + a.per - 1) / a.per) : 1);
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
    const dim3 grid((unsigned)tf, (unsigned)to, (unsigned)a.splits);
    c8_type(dy.scalar_type(), "weight_grad8: dy", [&](auto e) {
        c8_type(dw.scalar_type(), "weight_grad8: dw", [&](auto g) {
            typedef decltype(e) E;
            typedef decltype(g) G;
            hipLaunchKernelGGL((c8_weight_grad<E, G>), dim3(grid), dim3(256), 0, stream, a);
            if (join) {
                hipLaunchKernelGGL((c8_join<G>), dim3(c8_blocks(O * F)), dim3(256), 0, stream, (const float*)part.data_ptr(), (typename G::store*)dw.data_ptr(), O * F, a.splits);
                if (db.has_value())
                    hipLaunchKernelGGL((c8_join<G>), dim3(c8_blocks(O)), dim3(256), 0, stream, (const float*)part_b.data_ptr(), (typename G::store*)db->data_ptr(), O, a.splits);
            }
        });
    });
    C10_HIP_KERNEL_LAUNCH_CHECK();
}
