// Gated linear recurrence over a batch of sequences, its gradient, and its
// one-token form.
//
//   p = [x | r | z] along the last axis (z optional), k = sigmoid(-r)
//   h_t = h_{t-1} + k_t (x_t - h_{t-1})        ( = (1-k) h + k x )
//   y_t = h_t * z_t * sigmoid(z_t)             (y_t = h_t without z)
//
// The update is written with k and not with 1 - k: a long memory has k near 0,
// where 1 - k in 32 bits has lost k's digits. Every state is held in 32 bits;
// only y and dp are rounded, once, to the type of p.
//
// A wave owns 64 * V channels (V neighbours a lane) and takes GS_R tokens at a
// time: all their loads are issued before the first is used, so that enough
// bytes are in flight, and the recurrence then runs in registers.
#include <ATen/hip/HIPContext.h>
#include <c10/core/DeviceGuard.h>

#include "checkpoint8.h"
#include "launchers.h"

#define GS_R 16  // tokens of a tile, and between two kept states

namespace {

__device__ __forceinline__ float gs_rcp(float x) { return __builtin_amdgcn_rcpf(x); }
// exp overflows to +inf for x far below 0, whose reciprocal is the right 0
__device__ __forceinline__ float gs_sigmoid(float x) { return gs_rcp(1.f + __expf(-x)); }

// V neighbouring elements of type E
template <class E, int V>
struct alignas(sizeof(typename E::store) * V) GsVec {
    typename E::store v[V];
};

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
    unsigned char* scales;  // [B][T][P][Dp / 32]
    // backward
    const void* dy;         // [B][T][D], rows at dsb, dst
    int64_t dsb, dst;
    const float* dh_last;   // [B][D] or null
    void* dp;               // [B][T][P*D]
    float* dh0;             // [B][D] or null
    int B, T, D, Dp;
    int tps;                // lanes of one sequence
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
};

template <int V>
__device__ __forceinline__ GsLane gs_lane(const GsArgs& a, int64_t id) {
    GsLane l;
    int64_t b = id / a.tps;
    l.d = (int)(id - b * a.tps) * V;
    l.live = b < a.B && l.d < a.D;
    l.b = b < a.B ? (int)b : a.B - 1;   // lanes without a channel read one that exists
    l.d = l.d < a.D ? l.d : a.D - V;
    l.len = l.live ? gs_len(a, l.b) : 0;
    return l;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
template <class E, int V, int P, bool KEEP>
__global__ __launch_bounds__(64) void gs_fwd(GsArgs a) {
    typedef GsVec<E, V> vec;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 64 + lane;
    const GsLane l = gs_lane<V>(a, id);
    const int nT = (a.T + GS_R - 1) / GS_R;
    const typename E::store* p = (const typename E::store*)a.p + l.b * a.sb + l.d;
    typename E::store* y = (typename E::store*)a.y + (int64_t)l.b * a.T * a.D + l.d;

    float h[V];
#pragma unroll
    for (int v = 0; v < V; ++v) h[v] = a.h0 != nullptr ? a.h0[(int64_t)l.b * a.D + l.d + v] : 0.f;

    for (int tile = 0; tile < nT; ++tile) {
        const int t0 = tile * GS_R;
        if (a.states != nullptr && l.live) {
#pragma unroll
            for (int v = 0; v < V; ++v) a.states[((int64_t)l.b * nT + tile) * a.D + l.d + v] = h[v];
        }
        vec raw[P][GS_R];
#pragma unroll
        for (int i = 0; i < GS_R; ++i) {
            const int t = min(t0 + i, a.T - 1);
#pragma unroll
            for (int q = 0; q < P; ++q) raw[q][i] = *(const vec*)(p + (int64_t)t * a.st + q * a.D);
        }
        if constexpr (KEEP) {
            const int64_t ng = a.Dp / C8_GROUP;
            const bool mine = id < (int64_t)a.B * a.tps;
            const int dd = (int)(id % a.tps) * V;  // channel, padding included
#pragma unroll
            for (int q = 0; q < P; ++q) {
#pragma unroll
                for (int i = 0; i < GS_R; ++i) {
                    float f[V];
                    unsigned int top = 0;
#pragma unroll
                    for (int v = 0; v < V; ++v) {
                        f[v] = l.live ? E::up(raw[q][i].v[v]) : 0.f;
                        top = max(top, c8_mag(f[v]));
                    }
                    top = c8_max16(top);
                    if constexpr (V == 1) top = max(top, (unsigned int)__shfl_xor((int)top, 16, 64));
                    const unsigned int s = c8_scale(top);
                    const float inv = c8_inv(s);
                    if (mine && t0 + i < a.T) {
                        const int64_t row = ((int64_t)l.b * a.T + t0 + i) * P + q;
                        signed char* c = a.codes + row * a.Dp + dd;
                        if constexpr (V == 2) {
                            *(short*)c = (short)((c8_code(f[0], inv) & 0xff) | (c8_code(f[1], inv) << 8));
                        } else {
                            c[0] = (signed char)c8_code(f[0], inv);
                        }
                        if ((dd & (C8_GROUP - 1)) == 0) a.scales[row * ng + dd / C8_GROUP] = (unsigned char)s;
                    }
                }
            }
        }
#pragma unroll
        for (int i = 0; i < GS_R; ++i) {
            const bool in = t0 + i < l.len;
            vec out;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float k = gs_sigmoid(-E::up(raw[1][i].v[v])), x = E::up(raw[0][i].v[v]);
                // selected, not multiplied by 0: padding may hold anything
                h[v] = in ? fmaf(k, x - h[v], h[v]) : h[v];
                float o = h[v];
                if constexpr (P == 3) {
                    const float z = E::up(raw[2][i].v[v]);
                    o *= z * gs_sigmoid(z);
                }
                out.v[v] = E::down(in ? o : 0.f);
            }
            if (l.live && t0 + i < a.T) *(vec*)(y + (int64_t)(t0 + i) * a.D) = out;
        }
    }
    if (l.live) {
#pragma unroll
        for (int v = 0; v < V; ++v) a.h_last[(int64_t)l.b * a.D + l.d + v] = h[v];
    }
}

// ---------------------------------------------------------------------------
// backward: tiles from the last to the first. The states of a tile are computed
// again from the one kept before it, then
//   g_t = dy_t silu(z_t) + c,  c = (1-k_t) g_t for the token before
//   dx = g k, dr = g (h_{t-1} - x) k (1-k), dz = dy h silu'(z)
// ---------------------------------------------------------------------------
template <class E, int V, int P, bool KEEP>
__global__ __launch_bounds__(64) void gs_bwd(GsArgs a) {
    typedef GsVec<E, V> vec;
    const int lane = threadIdx.x & 63;
    const int64_t id = (int64_t)blockIdx.x * 64 + lane;
    const GsLane l = gs_lane<V>(a, id);
    const int nT = (a.T + GS_R - 1) / GS_R;
    const int64_t row0 = (int64_t)l.b * a.T;
    const typename E::store* p = (const typename E::store*)a.p + l.b * a.sb + l.d;
    const typename E::store* dy = (const typename E::store*)a.dy + l.b * a.dsb + l.d;
    typename E::store* dp = (typename E::store*)a.dp + row0 * P * a.D + l.d;

    float c[V];
#pragma unroll
    for (int v = 0; v < V; ++v) c[v] = a.dh_last != nullptr ? a.dh_last[(int64_t)l.b * a.D + l.d + v] : 0.f;

    for (int tile = nT - 1; tile >= 0; --tile) {
        const int t0 = tile * GS_R;
        float val[P][GS_R][V];
        vec raw_dy[GS_R];
#pragma unroll
        for (int i = 0; i < GS_R; ++i) {
            const int t = min(t0 + i, a.T - 1);
            raw_dy[i] = *(const vec*)(dy + (int64_t)t * a.dst);
#pragma unroll
            for (int q = 0; q < P; ++q) {
                if constexpr (KEEP) {
                    const int64_t row = (row0 + t) * P + q;
                    const float step = c8_step(a.scales[row * (a.Dp / C8_GROUP) + l.d / C8_GROUP]);
#pragma unroll
                    for (int v = 0; v < V; ++v) val[q][i][v] = (float)a.codes[row * a.Dp + l.d + v] * step;
                } else {
                    const vec w = *(const vec*)(p + (int64_t)t * a.st + q * a.D);
#pragma unroll
                    for (int v = 0; v < V; ++v) val[q][i][v] = E::up(w.v[v]);
                }
            }
        }
        float h[V], before[GS_R][V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = a.states[((int64_t)l.b * nT + tile) * a.D + l.d + v];
#pragma unroll
        for (int i = 0; i < GS_R; ++i) {
            const bool in = t0 + i < l.len;
#pragma unroll
            for (int v = 0; v < V; ++v) {
                before[i][v] = h[v];
                val[1][i][v] = gs_sigmoid(-val[1][i][v]);  // from here on k
                h[v] = in ? fmaf(val[1][i][v], val[0][i][v] - h[v], h[v]) : h[v];
            }
        }
#pragma unroll
        for (int i = GS_R - 1; i >= 0; --i) {
            const bool in = t0 + i < l.len;
            vec out[P];
#pragma unroll
            for (int v = 0; v < V; ++v) {
                const float x = val[0][i][v], k = val[1][i][v], hp = before[i][v];
                float g = E::up(raw_dy[i].v[v]);
                if constexpr (P == 3) {
                    const float z = val[2][i][v];
                    const float s = gs_sigmoid(z), zs = z * s;
                    const float hn = fmaf(k, x - hp, hp);
                    out[2].v[v] = E::down(in ? g * hn * fmaf(zs, 1.f - s, s) : 0.f);
                    g *= zs;
                }
                g += c[v];
                const float gk = g * k;
                c[v] = in ? g - gk : c[v];
                out[0].v[v] = E::down(in ? gk : 0.f);
                out[1].v[v] = E::down(in ? (hp - x) * fmaf(-k, gk, gk) : 0.f);
            }
            if (l.live && t0 + i < a.T) {
#pragma unroll
                for (int q = 0; q < P; ++q) *(vec*)(dp + ((int64_t)(t0 + i) * P + q) * a.D) = out[q];
            }
        }
    }
    if (l.live && a.dh0 != nullptr) {
#pragma unroll
        for (int v = 0; v < V; ++v) a.dh0[(int64_t)l.b * a.D + l.d + v] = c[v];
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
    typedef GsVec<E, V> vec;
    const int row = blockIdx.x;
    const int64_t slot = a.slots != nullptr ? gs_slot(a, row) : row;
    typename E::store* y = (typename E::store*)a.y;
    if (slot < 0 || slot >= a.S) {  // no state: a row of padding
        vec zero;
#pragma unroll
        for (int v = 0; v < V; ++v) zero.v[v] = E::down(0.f);
        for (int d = threadIdx.x * V; d < a.D; d += blockDim.x * V) *(vec*)(y + (int64_t)row * a.D + d) = zero;
        return;
    }
    int later = 0;
    if (a.slots != nullptr) {
        int earlier = 0;
        for (int b = threadIdx.x; b < a.B; b += blockDim.x) {
            if (b != row && gs_slot(a, b) == slot) {
                earlier |= b < row;
                later |= b > row;
            }
        }
        if (__syncthreads_or(earlier)) return;
        later = __syncthreads_or(later);
    }
    for (int d = threadIdx.x * V; d < a.D; d += blockDim.x * V) {
        float h[V];
#pragma unroll
        for (int v = 0; v < V; ++v) h[v] = a.state[slot * a.D + d + v];
        for (int b = row; b < a.B; ++b) {
            if (b != row && gs_slot(a, b) != slot) continue;
            const typename E::store* p = (const typename E::store*)a.p + b * a.sb + d;
            vec raw[P], out;
#pragma unroll
            for (int q = 0; q < P; ++q) raw[q] = *(const vec*)(p + (int64_t)q * a.D);
#pragma unroll
            for (int v = 0; v < V; ++v) {
                h[v] = fmaf(gs_sigmoid(-E::up(raw[1].v[v])), E::up(raw[0].v[v]) - h[v], h[v]);
                float o = h[v];
                if constexpr (P == 3) {
                    const float z = E::up(raw[2].v[v]);
                    o *= z * gs_sigmoid(z);
                }
                out.v[v] = E::down(o);
            }
            *(vec*)(y + (int64_t)b * a.D + d) = out;
            if (!later) break;
        }
#pragma unroll
        for (int v = 0; v < V; ++v) a.out[slot * a.D + d + v] = h[v];
    }
}

bool gs_pairs(const torch::Tensor& t) {
    return ((uintptr_t)t.data_ptr() % (2 * t.element_size())) == 0;
}

// calls f.template operator()<E, V, P>()
template <class F>
void gs_types(at::ScalarType dt, bool pair, int64_t parts, F&& f) {
    auto with = [&](auto e) {
        typedef decltype(e) E;
        if (pair) {
            if (parts == 3) f.template operator()<E, 2, 3>();
            else f.template operator()<E, 2, 2>();
        } else {
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

struct GsFwdCall {
    const GsArgs& a;
    int64_t blocks;
    hipStream_t stream;
    bool keep;
    template <class E, int V, int P>
    void operator()() {
        if (keep) hipLaunchKernelGGL((gs_fwd<E, V, P, true>), dim3((unsigned)blocks), dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((gs_fwd<E, V, P, false>), dim3((unsigned)blocks), dim3(64), 0, stream, a);
    }
};

struct GsBwdCall {
    const GsArgs& a;
    int64_t blocks;
    hipStream_t stream;
    bool keep;
    template <class E, int V, int P>
    void operator()() {
        if (keep) hipLaunchKernelGGL((gs_bwd<E, V, P, true>), dim3((unsigned)blocks), dim3(64), 0, stream, a);
        else hipLaunchKernelGGL((gs_bwd<E, V, P, false>), dim3((unsigned)blocks), dim3(64), 0, stream, a);
    }
};

struct GsStepCall {
    const GsStepArgs& a;
    int threads;
    hipStream_t stream;
    template <class E, int V, int P>
    void operator()() {
        hipLaunchKernelGGL((gs_step<E, V, P>), dim3(a.B), dim3(threads), 0, stream, a);
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
    const int64_t rows = p.size(0) * p.size(1) * parts;
    TORCH_CHECK(scales.has_value() && codes->device() == p.device() && scales->device() == p.device() &&
                    codes->scalar_type() == at::kChar && scales->scalar_type() == at::kByte &&
                    codes->is_contiguous() && scales->is_contiguous() &&
                    codes->numel() == rows * a.Dp && scales->numel() == rows * (a.Dp / C8_GROUP),
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
    const int64_t blocks = ((int64_t)a.B * a.tps + 63) / 64;
    TORCH_CHECK(blocks <= INT_MAX, "gated_scan: too many channels");
    GsFwdCall call{a, blocks, at::hip::getCurrentHIPStream().stream(), a.codes != nullptr};
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
    a.tps = a.D / (pair ? 2 : 1);
    const c10::DeviceGuard guard(p.device());
    const int64_t blocks = ((int64_t)a.B * a.tps + 63) / 64;
    TORCH_CHECK(blocks <= INT_MAX, "gated_scan: too many channels");
    GsBwdCall call{a, blocks, at::hip::getCurrentHIPStream().stream(), a.codes != nullptr};
    gs_types(p.scalar_type(), pair, parts, call);
    C10_HIP_KERNEL_LAUNCH_CHECK();
}

void gated_step_launch(torch::Tensor p, int64_t dim, torch::Tensor state, c10::optional<torch::Tensor> slots,
                       torch::Tensor out, torch::Tensor y) {
    TORCH_CHECK(p.is_cuda() && p.dim() == 2 && p.stride(1) == 1 && dim > 0 &&
                    (p.size(1) == 2 * dim || p.size(1) == 3 * dim) && p.size(0) > 0 && p.size(0) <= INT_MAX && p.size(1) <= INT_MAX,
                "gated_step: p must be [B, 2 or 3 times dim] on the GPU, unit stride last");
    GsStepArgs a{};
    a.B = (int)p.size(0);
    a.D = (int)dim;
    TORCH_CHECK(state.dim() == 2 && state.size(1) == dim, "gated_step: state must be [slots, dim]");
    a.S = state.size(0);
    gs_f32(state, a.S * dim, p, "state");
    gs_f32(out, a.S * dim, p, "out");
    TORCH_CHECK(y.device() == p.device() && y.scalar_type() == p.scalar_type() && y.is_contiguous() &&
                    y.numel() == (int64_t)a.B * dim, "gated_step: y does not match p");
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
}
