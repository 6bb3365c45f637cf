// The norms of a decoder block's query and key heads and their rotary
// positions, in one pass over the q|k|v rows of the projection.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          per head, where a norm is given
//   (a, b) -> (a c - b s, b c + a s)            per pair, (c, s) = table[position][i]
//
// Pairs are (i, i + rot/2) or (2i, 2i + 1) of the head's first rot elements;
// the others, and v, pass. fp32 throughout, one rounding when stored.
//
// Bound by memory: every element is read once and written once. d/8 lanes
// (rounded up to a power of two) own one head of one token, eight elements
// each, so a wave reads and writes whole lines; the partners of the half
// layout meet in LDS, each lane group's own part of it, which needs no
// barrier beyond the wave's.
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

template <int IN, int OUT>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeArgs a, int lanes) {
    using I = Val<IN>;
    using O = Val<OUT>;
    __shared__ float stage[256 * 8];
    const int heads = (int)(a.q_heads + (a.v ? 2 : 1) * a.kv_heads);
    const int sub = threadIdx.x & (lanes - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / lanes) + threadIdx.x / lanes;
    if (unit >= a.tokens * heads) return;              // whole lane groups leave; nothing below waits for them
    const int64_t t = unit / heads;
    const int h = (int)(unit - t * heads);
    const bool is_q = h < a.q_heads, is_k = !is_q && h < a.q_heads + a.kv_heads;
    const int d = (int)a.head_dim, rot = (int)a.rot, e0 = sub * 8;
    const bool on = e0 < d;
    float x[8] = {0, 0, 0, 0, 0, 0, 0, 0};
    if (on) I::load8(static_cast<const typename I::Elem*>(a.x) + t * a.ld_x + (int64_t)h * d + e0, x);
    typename O::Elem* dst = static_cast<typename O::Elem*>(is_q ? a.q : is_k ? a.k : a.v) +
                            t * (is_q ? a.ld_q : is_k ? a.ld_k : a.ld_v) +
                            (int64_t)(is_q ? h : is_k ? h - a.q_heads : h - a.q_heads - a.kv_heads) * d + e0;
    if (!is_q && !is_k) {
        if (on) O::store8(dst, x);
        return;
    }
    const float* w = is_q ? a.q_norm : a.k_norm;
    if (w) {
        float ss = 0.f;
#pragma unroll
        for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[i], x[i], ss);
        for (int m = lanes >> 1; m; m >>= 1) ss += __shfl_xor(ss, m);
        const float r = 1.0f / sqrtf(ss / (float)d + a.eps);
        if (on) {
            float wv[8];
            Val<kTypeF32>::load8(w + e0, wv);
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = x[i] * r * wv[i];
        }
    }
    const int64_t pos = rot ? a.positions[t] : 0;
    const bool known = rot == 0 || (pos >= 0 && pos < a.n_pos);      // else the row is NaN
    const float2* row = reinterpret_cast<const float2*>(a.table) + (known ? pos : 0) * (rot / 2);
    if (a.interleaved) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if (e0 + 2 * i < rot) {
                const float2 cs = row[e0 / 2 + i];
                const float p = x[2 * i], q = x[2 * i + 1];
                x[2 * i] = __builtin_fmaf(p, cs.x, -(q * cs.y));
                x[2 * i + 1] = __builtin_fmaf(q, cs.x, p * cs.y);
            }
        }
    } else {
        float* mine = stage + (threadIdx.x - sub) * 8;
#pragma unroll
        for (int i = 0; i < 8; ++i) mine[e0 + i] = x[i];
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
        const int half = rot / 2;
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const int e = e0 + i;
            if (e < rot) {
                const bool low = e < half;
                const float2 cs = row[low ? e : e - half];
                const float other = mine[low ? e + half : e - half];
                x[i] = __builtin_fmaf(x[i], cs.x, low ? -(other * cs.y) : other * cs.y);
            }
        }
    }
    if (!known) {
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = __builtin_nanf("");
    }
    if (on) O::store8(dst, x);
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeArgs& a, hipStream_t stream) {
    int lanes = 1;
    while (lanes * 8 < a.head_dim) lanes *= 2;
    const int64_t units = a.tokens * (a.q_heads + (a.v ? 2 : 1) * a.kv_heads);
    const int64_t grid = (units + 256 / lanes - 1) / (256 / lanes);
    return with_type(a.x_type, [&](auto in) {
        return with_type(a.out_type, [&](auto out) {
            qk_norm_rope_kernel<decltype(in)::value, decltype(out)::value><<<(unsigned)grid, 256, 0, stream>>>(a, lanes);
            return hipGetLastError();
        });
    });
}

}  // namespace frq
