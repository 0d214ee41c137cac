// rope.cu -- rotary positions of packed (ragged) token rows, with the q/k RMSNorm that precedes them in the hybrid
// model, forward and adjoint, and the tables they read (reference src/adjoint/host/qk.cpp and rope.cpp, there over
// one sequence's positions).
//
//   y = R(pos) n,   n = x rstd w (or x),   rstd = (mean x^2 + eps)^-1/2
//   R rotates pair i < rot / 2 of the head, (i, i + rot / 2) or (2 i, 2 i + 1), by pos * inv_i
//   adjoint: d = R(-pos) dy (the tables' amplitude included), dx = rstd w d - x rstd^3 mean(w d x)
//
// Bound by HBM: each row is read once and written once (the adjoint reads x and dy). A warp owns one token and
// up to kBatch head rows of it at a time, 16 bytes a lane, so the token's cos and sin values are fetched once per
// batch into registers and all the batch's row loads are in flight together; queries and keys share one launch.
#include "sm100.cuh"
#include "r97b_internal.h"

#include <cuda_bf16.h>
#include <math.h>

namespace r97b {

R97B_ERROR_READER(rope_error_word)

namespace {

constexpr int kBatch = 4;  // row loads a lane has in flight (two a row in the adjoint)

struct RopeArgs {
    R97bRopePart part[2];
    const float* cos_tab;
    const float* sin_tab;
    const int32_t* pos;
    int64_t units, n_pos;
    int32_t heads, chunks, rot;
    float eps;
};

__device__ __forceinline__ uint4 ld_row(const R97bHeadRows& r, int64_t t, int h, int e) {
    return *reinterpret_cast<const uint4*>(reinterpret_cast<const __nv_bfloat16*>(r.ptr) + t * r.tok + h * r.head + e);
}
__device__ __forceinline__ void unpack8(const uint4& u, float (&v)[8]) {
    const __nv_bfloat162* p = reinterpret_cast<const __nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        const float2 f = __bfloat1622float2(p[i]);
        v[2 * i] = f.x;
        v[2 * i + 1] = f.y;
    }
}
__device__ __forceinline__ void st_row(const R97bHeadRows& r, int64_t t, int h, int e, const float (&v)[8]) {
    uint4 u;
    __nv_bfloat162* p = reinterpret_cast<__nv_bfloat162*>(&u);
#pragma unroll
    for (int i = 0; i < 4; ++i) p[i] = __floats2bfloat162_rn(v[2 * i], v[2 * i + 1]);
    *reinterpret_cast<uint4*>(reinterpret_cast<__nv_bfloat16*>(r.ptr) + t * r.tok + h * r.head + e) = u;
}

// Rotates the lane's 8 values by the pairs' (cos, sin); sign -1 is the inverse rotation. `src` is the lane that
// holds the partners of a half-layout lane, `lead` whether this lane holds the pairs' first members.
template <bool INTER>
__device__ __forceinline__ void rotate8(float (&v)[8], const float (&cs)[8], const float (&sn)[8], bool in_rot, bool lead,
                                        int src, float sign) {
    if (INTER) {
        if (in_rot) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const float a = v[2 * i], b = v[2 * i + 1], s = sign * sn[i];
                v[2 * i] = a * cs[i] - b * s;
                v[2 * i + 1] = b * cs[i] + a * s;
            }
        }
    } else {
        const float sg = lead ? -sign : sign;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const float o = __shfl_sync(0xFFFFFFFFu, v[i], src);  // every lane joins
            if (in_rot) v[i] = v[i] * cs[i] + sg * o * sn[i];
        }
    }
}

template <int D, bool INTER, bool BACK>
__global__ void __launch_bounds__(256) qk_rope_kernel(const __grid_constant__ RopeArgs a) {
    constexpr int kLanes = D / 8;          // lanes of one row
    constexpr int kRows = 32 / kLanes;     // rows a warp covers at once
    const int64_t unit = ((int64_t)blockIdx.x * blockDim.x + threadIdx.x) >> 5;
    if (unit >= a.units) return;
    const int64_t t = a.chunks == 1 ? unit : unit / a.chunks;
    const int h0 = (int)(unit - t * a.chunks) * (kBatch * kRows);
    const int lane = threadIdx.x & 31, l = lane & (kLanes - 1), e = 8 * l;
    const int heads0 = (int)a.part[0].heads;

    int head[kBatch];
    bool live[kBatch], second[kBatch];
    uint4 rx[kBatch], rd[kBatch];
#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
        const int hh = h0 + b * kRows + lane / kLanes;
        live[b] = hh < a.heads;
        second[b] = hh >= heads0;
        head[b] = second[b] ? hh - heads0 : hh;
        rx[b] = rd[b] = make_uint4(0, 0, 0, 0);
        if (live[b]) {
            const R97bRopePart& p = a.part[second[b]];
            if (!BACK || p.w) rx[b] = ld_row(p.x, t, head[b], e);
            if (BACK) rd[b] = ld_row(p.y, t, head[b], e);
        }
    }

    // this lane's rotary values: 8 pairs of one member each (half layout) or 4 whole pairs
    const int half = a.rot / 2;
    const bool in_rot = e < a.rot, lead = e < half;
    const int src = in_rot ? (lane & ~(kLanes - 1)) + (lead ? l + half / 8 : l - half / 8) : lane;
    const int32_t pos = a.pos[t];
    const bool known = pos >= 0 && pos < a.n_pos;
    if (!known && lane == 0) atomicOr(&g_device_error, kErrArgs);
    float cs[8], sn[8];
#pragma unroll
    for (int i = 0; i < 8; ++i) cs[i] = sn[i] = 0.0f;
    if (in_rot && known) {
        const int64_t at = (int64_t)pos * half + (INTER ? e / 2 : (lead ? e : e - half));
#pragma unroll
        for (int i = 0; i < (INTER ? 1 : 2); ++i) {
            const float4 c = *reinterpret_cast<const float4*>(a.cos_tab + at + 4 * i);
            const float4 s = *reinterpret_cast<const float4*>(a.sin_tab + at + 4 * i);
            cs[4 * i] = c.x, cs[4 * i + 1] = c.y, cs[4 * i + 2] = c.z, cs[4 * i + 3] = c.w;
            sn[4 * i] = s.x, sn[4 * i + 1] = s.y, sn[4 * i + 2] = s.z, sn[4 * i + 3] = s.w;
        }
    }

#pragma unroll
    for (int b = 0; b < kBatch; ++b) {
        const R97bRopePart& p = a.part[second[b] && live[b]];
        const bool norm = p.w != nullptr;
        float x[8], d[8], w[8];
        unpack8(rx[b], x);
        if (BACK) unpack8(rd[b], d);
        if (norm) {
            const float4 w0 = *reinterpret_cast<const float4*>(p.w + e), w1 = *reinterpret_cast<const float4*>(p.w + e + 4);
            w[0] = w0.x, w[1] = w0.y, w[2] = w0.z, w[3] = w0.w, w[4] = w1.x, w[5] = w1.y, w[6] = w1.z, w[7] = w1.w;
        }
        if (BACK) {
            rotate8<INTER>(d, cs, sn, in_rot, lead, src, -1.0f);
            float ss = 0.0f, dot = 0.0f;
            if (norm) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    d[i] *= w[i];
                    ss = fmaf(x[i], x[i], ss);
                    dot = fmaf(d[i], x[i], dot);
                }
            }
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) {
                ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
                dot += __shfl_xor_sync(0xFFFFFFFFu, dot, o);
            }
            if (norm) {
                const float r = rsqrtf(ss / (float)D + a.eps);
                const float k = r * r * r * (dot / (float)D);
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = r * d[i] - k * x[i];
            }
            if (!known) {
#pragma unroll
                for (int i = 0; i < 8; ++i) d[i] = 0.0f;
            }
            if (live[b]) st_row(p.dx, t, head[b], e, d);
        } else {
            float ss = 0.0f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = fmaf(x[i], x[i], ss);
#pragma unroll
            for (int o = kLanes / 2; o > 0; o >>= 1) ss += __shfl_xor_sync(0xFFFFFFFFu, ss, o);
            if (norm) {
                const float r = rsqrtf(ss / (float)D + a.eps);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] *= r * w[i];
            }
            rotate8<INTER>(x, cs, sn, in_rot, lead, src, 1.0f);
            if (!known) {
#pragma unroll
                for (int i = 0; i < 8; ++i) x[i] = 0.0f;
            }
            if (live[b]) st_row(p.y, t, head[b], e, x);
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
    const int per = kBatch * 256 / a->D;  // head rows a warp takes: kBatch x (32 lanes x 8 / D)
    r.chunks = (r.heads + per - 1) / per;
    r.units = a->T * r.chunks;
    const int64_t grid = (r.units + 7) / 8;
    if (grid > 0x7FFFFFFF) return R97B_EINVAL;
    cudaStream_t st = as_stream(stream);
    const bool inter = a->interleaved != 0;
#define R97B_ROPE_D(DD)                                                                    \
    if (a->D == DD) {                                                                      \
        if (inter)                                                                         \
            qk_rope_kernel<DD, true, BACK><<<(unsigned)grid, 256, 0, st>>>(r);             \
        else                                                                               \
            qk_rope_kernel<DD, false, BACK><<<(unsigned)grid, 256, 0, st>>>(r);            \
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
        const double low = fmax(floor(pair_of(beta_fast)), 0.0), high = fmin(ceil(pair_of(beta_slow)), rot / 2 - 1.0);
        t.low = low;
        t.width = fmax(high - low, 1e-3);  // a step where both ends fall on one pair
        t.amp = 0.1 * log(factor) + 1.0;
    }
    const int64_t grid = (t.n + 255) / 256;
    if (grid > 0x7FFFFFFF) return R97B_EINVAL;
    rope_table_kernel<<<(unsigned)grid, 256, 0, as_stream(stream)>>>(t);
    return launch_status();
}
