// rope.cu -- rotary positions of packed (ragged) token rows, with the q/k RMSNorm that precedes them in the hybrid
// model, forward and adjoint, and the tables they read (reference src/adjoint/host/qk.cpp and rope.cpp, there over
// one sequence's positions).
//
//   y = R(pos) n,   n = x rstd w (or x),   rstd = (mean x^2 + eps)^-1/2
//   R rotates pair i < rot / 2 of the head, (i, i + rot / 2) or (2 i, 2 i + 1), by pos * inv_i
//   adjoint: d = R(-pos) dy (the tables' amplitude included), dx = rstd w d - x rstd^3 mean(w d x)
//
// Bound by HBM: each row is read once and written once (the adjoint reads x and dy). A lane holds 16 values of a row as
// two 16-byte chunks that rotate with one another -- in the half layout chunk k and the one rot / 2 after it -- so the
// rotation needs no exchange between lanes and D / 16 lanes sum the norm. A warp takes kWarpRows rows a lane of one token,
// queries and keys alike, with the token's cos and sin in registers; what hides the loads is the number of warps, so the
// gain is read again (from L1) for every row rather than held.
#include "sm100.cuh"
#include "r97b_internal.h"
#include "fastmath.cuh"

#include <cuda_bf16.h>
#include <math.h>

namespace r97b {

R97B_ERROR_READER(rope_error_word)

namespace {

constexpr int kBlockThreads = 128;
// Rows a lane takes in turn, and the blocks an SM holds (what their registers, 70 and 80 a thread, then may be): measured at
// 8192 tokens of 16 + 4 heads of 256 (forward / adjoint) and the adjoint of 32749 tokens, 16 + 4 heads of 128, rotated
// whole: 5 rows at 7 / 6 blocks 39.7 / 54.8 / 101 us; 10 rows at 8 / 6 41.8 / 56.8 / 102; 4 rows at 8 / 6 44.4 / 60.4 / 121;
// 10 / 8 blocks (spills) 70 / 82 / 141. The copy-rate times of the same bytes are 25.9 / 38.7 / 79.6 us.
// 5 divides those 20 heads evenly; a head count that it does not leaves a token's last warp short. Other heads, forward /
// adjoint, at 5 rows, 4 and 10: 12 + 4 of 256, 8192 tokens 37.6 / 50.0, 35.6 / 48.0, 33.6 / 48.3 us (copy rate 20.7 / 31);
// 24 + 8 of 128 interleaved, rotated whole, 16384 tokens 70.5 / 91.0, 66.5 / 85.2, 64.3 / 81.3; 32 + 8 of 256, 4096 tokens
// 41.7 / 56.3, 42.2 / 56.3, 40.0 / 58.4.
constexpr int kWarpRows = 5;
constexpr int kFwdBlocks = 7, kBwdBlocks = 6;

struct RopeArgs {
    R97bRopePart part[2];
    const float* cos_tab;
    const float* sin_tab;
    const int32_t* pos;
    int64_t units, n_pos;
    int32_t heads, chunks, rot;
    float eps;
};

struct Row16 {  // a lane's two chunks of a row
    uint4 a, b;
};
__device__ __forceinline__ Row16 ld_row(const R97bHeadRows& r, int64_t t, int h, int ea, int eb) {
    const __nv_bfloat16* p = reinterpret_cast<const __nv_bfloat16*>(r.ptr) + t * r.tok + h * r.head;
    return Row16{*reinterpret_cast<const uint4*>(p + ea), *reinterpret_cast<const uint4*>(p + eb)};
}
__device__ __forceinline__ void unpack8(const uint4& u, float2* v) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) v[i] = __bfloat1622float2(p[i]);
}
__device__ __forceinline__ uint4 pack8(const float2* v) {
    uint4 u;
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(v[i].x, v[i].y);
    return u;
}
__device__ __forceinline__ void ld8f(const float* p, float2* v) {
    const float4 a = *reinterpret_cast<const float4*>(p), b = *reinterpret_cast<const float4*>(p + 4);
    v[0] = make_float2(a.x, a.y), v[1] = make_float2(a.z, a.w), v[2] = make_float2(b.x, b.y), v[3] = make_float2(b.z, b.w);
}

template <int D, bool INTER, bool BACK>
__global__ void __launch_bounds__(kBlockThreads, BACK ? kBwdBlocks : kFwdBlocks) qk_rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kLanes = D / 16;         // lanes of one row
    constexpr int kRows = 32 / kLanes;     // rows a warp covers at once
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (unit >= a.units) return;
    const int64_t t = a.chunks == 1 ? unit : unit / a.chunks;
    const int lane = threadIdx.x & 31, l = lane & (kLanes - 1);
    const int heads0 = (int)a.part[0].heads;
    int hh = (int)(unit - t * a.chunks) * (kWarpRows * kRows) + lane / kLanes;
    const int32_t pos = a.pos[t];

    // the lane's chunks: the l-th pair of the rotated part, or two neighbours of the rest
    const int half = a.rot / 2, pairs = half / 8;
    const bool in_rot = l < pairs;
    const int ea = in_rot ? (INTER ? 16 * l : 8 * l) : a.rot + 16 * (l - pairs);
    const int eb = in_rot && !INTER ? ea + half : ea + 8;

    const bool known = pos >= 0 && pos < a.n_pos;
    if (!known && lane == 0) atomicOr(&g_device_error, kErrArgs);
    float2 cs[4], sn[4];  // the chunks' 8 pairs
#pragma unroll
    for (int i = 0; i < 4; ++i) cs[i] = both(1.0f), sn[i] = both(0.0f);
    if (in_rot && known) {
        ld8f(a.cos_tab + (int64_t)pos * half + 8 * l, cs);
        ld8f(a.sin_tab + (int64_t)pos * half + 8 * l, sn);
        if (BACK) {
#pragma unroll
            for (int i = 0; i < 4; ++i) sn[i] = make_float2(-sn[i].x, -sn[i].y);
        }
    }

#pragma unroll 1
    for (int n = 0; n < kWarpRows; ++n, hh += kRows) {
        const bool live = hh < a.heads;
        if (!__any_sync(0xFFFFFFFFu, live)) break;
        const int i = live && hh >= heads0, h = i ? hh - heads0 : hh;
        const R97bRopePart& p = a.part[i];
        const bool norm = p.w != nullptr;
        float2 x[8], v[8];  // (lanes past the last row compute on zeros and store nothing)
        Row16 rx{}, rd{};
        if (live && (!BACK || norm)) rx = ld_row(p.x, t, h, ea, eb);
        if (BACK && live) rd = ld_row(p.y, t, h, ea, eb);
        float2 w[8];
        if (norm) {
            ld8f(p.w + ea, w);
            ld8f(p.w + eb, w + 4);
        }
        unpack8(rx.a, x);
        unpack8(rx.b, x + 4);
        float2 ss = both(0.0f), dot = both(0.0f);
#pragma unroll
        for (int k = 0; k < 8; ++k) ss = fma2(x[k], x[k], ss);
        float s = ss.x + ss.y, r = 1.0f;
        if (BACK) {
            unpack8(rd.a, v);
            unpack8(rd.b, v + 4);
        } else {
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
            if (norm) r = rsqrtf(s / (float)D + a.eps);
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = norm ? mul2(x[k], mul2(w[k], both(r))) : x[k];
        }
        if (INTER) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float c = k & 1 ? cs[k / 2].y : cs[k / 2].x, z = k & 1 ? sn[k / 2].y : sn[k / 2].x;
                v[k] = fma2(make_float2(v[k].y, v[k].x), make_float2(-z, z), mul2(v[k], both(c)));
            }
        } else {
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                const float2 c0 = v[k], c1 = v[k + 4];
                v[k] = fma2(c1, make_float2(-sn[k].x, -sn[k].y), mul2(c0, cs[k]));
                v[k + 4] = fma2(c0, sn[k], mul2(c1, cs[k]));
            }
        }
        if (BACK && norm) {
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                v[k] = mul2(v[k], w[k]);
                dot = fma2(v[k], x[k], dot);
            }
        }
        if (BACK) {
            float d = dot.x + dot.y;
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) {
                s += __shfl_xor_sync(0xFFFFFFFFu, s, o);
                d += __shfl_xor_sync(0xFFFFFFFFu, d, o);
            }
            if (norm) {
                r = rsqrtf(s / (float)D + a.eps);
                const float k3 = -r * r * r * (d / (float)D);
#pragma unroll
                for (int k = 0; k < 8; ++k) v[k] = fma2(x[k], both(k3), mul2(v[k], both(r)));
            }
        }
        if (!known) {
#pragma unroll
            for (int k = 0; k < 8; ++k) v[k] = both(0.0f);
        }
        if (live) {
            const R97bHeadRows& o = BACK ? p.dx : p.y;
            __nv_bfloat16* q = reinterpret_cast<__nv_bfloat16*>(o.ptr) + t * o.tok + h * o.head;
            *reinterpret_cast<uint4*>(q + ea) = pack8(v);
            *reinterpret_cast<uint4*>(q + eb) = pack8(v + 4);
        }
    }
}

struct TableArgs {
    float* cos_tab;
    float* sin_tab;
    int64_t n;
    int32_t half;
    double theta, factor, low, width, amp;
    int32_t scaling;
};

// One table entry a thread, the angle and its functions in f64: at position 10^6 an f32 angle would be off by 0.03.
__global__ void __launch_bounds__(256) rope_table_kernel(const TableArgs a) {
    const int64_t at = (int64_t)blockIdx.x * blockDim.x + threadIdx.x;
    if (at >= a.n) return;
    const int64_t pos = at / a.half;
    const int i = (int)(at - pos * a.half);
    double inv = pow(a.theta, -(double)i / (double)a.half);
    if (a.scaling == R97B_ROPE_LINEAR) inv /= a.factor;
    if (a.scaling == R97B_ROPE_YARN) {
        const double ramp = fmin(fmax(((double)i - a.low) / a.width, 0.0), 1.0);
        inv = inv * (1.0 - ramp) + inv / a.factor * ramp;
    }
    double s, c;
    sincos((double)pos * inv, &s, &c);
    a.cos_tab[at] = (float)(c * a.amp);
    a.sin_tab[at] = (float)(s * a.amp);
}

bool f32_ok(const void* p) { return p && (reinterpret_cast<uintptr_t>(p) & 15) == 0; }

bool rope_ok(const R97bRope& a, bool back) {
    if ((a.D != 64 && a.D != 128 && a.D != 256) || a.rot <= 0 || a.rot > a.D || a.rot % 16) return false;
    if (a.n_parts < 1 || a.n_parts > 2 || a.T < 0 || a.T > 0x7FFFFFFF || a.n_pos < 1 || a.n_pos > 0x7FFFFFFF) return false;
    if (!f32_ok(a.cos_tab) || !f32_ok(a.sin_tab) || !a.pos || (reinterpret_cast<uintptr_t>(a.pos) & 3)) return false;
    for (int i = 0; i < a.n_parts; ++i) {
        const R97bRopePart& p = a.part[i];
        if (p.w && !f32_ok(p.w)) return false;
        if ((!back || p.w) && !head_rows_ok(p.x, p.heads, a.D)) return false;
        if (!head_rows_ok(p.y, p.heads, a.D)) return false;
        if (back && !head_rows_ok(p.dx, p.heads, a.D)) return false;
    }
    return true;
}

template <bool BACK>
int rope_run(const R97bRope* a, void* stream) {
    if (!a || !rope_ok(*a, BACK)) return R97B_EINVAL;
    if (a->T == 0) return R97B_OK;
    RopeArgs r{};
    r.heads = 0;
    for (int i = 0; i < a->n_parts; ++i) {
        r.part[i] = a->part[i];
        r.heads += (int32_t)a->part[i].heads;
    }
    r.cos_tab = a->cos_tab;
    r.sin_tab = a->sin_tab;
    r.pos = a->pos;
    r.n_pos = a->n_pos;
    r.rot = a->rot;
    r.eps = a->eps;
    const int per = kWarpRows * (512 / a->D);  // rows a warp takes
    r.chunks = (r.heads + per - 1) / per;
    r.units = a->T * r.chunks;
    const int64_t grid = (r.units + kBlockThreads / 32 - 1) / (kBlockThreads / 32);
    if (grid > 0x7FFFFFFF) return R97B_EINVAL;
    cudaStream_t st = as_stream(stream);
    const bool inter = a->interleaved != 0;
#define R97B_ROPE_D(DD)                                                                    \
    if (a->D == DD) {                                                                      \
        if (inter)                                                                         \
            qk_rope_kernel<DD, true, BACK><<<(unsigned)grid, kBlockThreads, 0, st>>>(r);             \
        else                                                                               \
            qk_rope_kernel<DD, false, BACK><<<(unsigned)grid, kBlockThreads, 0, st>>>(r);            \
    }
    R97B_ROPE_D(64)
    R97B_ROPE_D(128)
    R97B_ROPE_D(256)
#undef R97B_ROPE_D
    return launch_status();
}

}  // namespace
}  // namespace r97b

extern "C" int r97b_qk_rope_fwd(const R97bRope* a, void* stream) { return r97b::rope_run<false>(a, stream); }

extern "C" int r97b_qk_rope_bwd(const R97bRope* a, void* stream) { return r97b::rope_run<true>(a, stream); }

extern "C" int r97b_rope_tables(float* cos_tab, float* sin_tab, int64_t n_pos, int32_t rot, double theta, int32_t scaling,
                                double factor, double original, double beta_fast, double beta_slow, void* stream) {
    using namespace r97b;
    if (!cos_tab || !sin_tab || n_pos < 1 || n_pos > 0x7FFFFFFF || rot <= 0 || rot % 2 || rot > 4096 || !(theta > 1.0) ||
        !isfinite(theta))
        return R97B_EINVAL;
    if (scaling < R97B_ROPE_NONE || scaling > R97B_ROPE_YARN) return R97B_EINVAL;
    if (scaling != R97B_ROPE_NONE && !(factor >= 1.0 && isfinite(factor))) return R97B_EINVAL;
    if (scaling == R97B_ROPE_YARN &&
        !(original > 0.0 && beta_slow > 0.0 && beta_fast > beta_slow && isfinite(original) && isfinite(beta_fast)))
        return R97B_EINVAL;
    TableArgs t{cos_tab, sin_tab, n_pos * (rot / 2), rot / 2, theta, factor, 0.0, 1.0, 1.0, scaling};
    if (scaling == R97B_ROPE_YARN) {
        // pair i's wavelength is 2 pi theta^(2 i / rot): it turns `beta` times over `original` positions at
        // i = rot ln(original / (2 pi beta)) / (2 ln theta)
        auto pair_of = [&](double beta) {
            return rot * log(original / (2.0 * 3.14159265358979323846 * beta)) / (2.0 * log(theta));
        };
        // the slow end may lie past the last pair, whose ramp then stays short of 1; it is held to the rotated width's dims
        const double low = fmax(floor(pair_of(beta_fast)), 0.0), high = fmin(ceil(pair_of(beta_slow)), rot - 1.0);
        t.low = low;
        t.width = fmax(high - low, 1e-3);  // a step where both ends fall on one pair
        t.amp = 0.1 * log(factor) + 1.0;
    }
    const int64_t grid = (t.n + 255) / 256;
    if (grid > 0x7FFFFFFF) return R97B_EINVAL;
    rope_table_kernel<<<(unsigned)grid, 256, 0, as_stream(stream)>>>(t);
    return launch_status();
}
