// The norms of a decoder block's query and key heads and their rotary
// positions, in one pass over the q|k|v rows of the projection.
//
//   y = x * rsqrt(mean(x^2) + eps) * w          per head, where a norm is given
//   (a, b) -> (a c - b s, b c + a s)            per pair, (c, s) = table[position][i]
//
// Pairs are (i, i + rot/2) or (2i, 2i + 1) of the head's first rot elements;
// the others, and v, pass. fp32 throughout, one rounding when stored.
//
// Bound by memory: every element is read once and written once. A lane holds
// eight elements of each half of a head, so that the partners of a full half
// layout, and of any interleaved one, are its own; its cosines and sines serve
// all heads of the token. The other half layouts, and head sizes that are not a
// power of two, take a second kernel, whose partners meet in LDS.
//
// 8192 tokens of 48 heads of 128, normed, fp32 to bf16: 51 us, 6.0 TB/s, what a
// large copy reaches. 1001 tokens of 16 heads of 256, a quarter turned, bf16:
// 5.0 us, 3.3 TB/s (the start and end of so short a kernel); one token: 2.0 us.
// The second kernel, which waits for LDS and reads a head's cosines again for
// each: 8192 tokens of 48 heads of 128, half of each turned, fp32 to bf16: 67 us
// (47 with whole heads turned, both without norms), 80-wide heads 57 us, 3.4 TB/s.
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

template <int IN, int OUT, int LANES, bool INTER>
__global__ void __launch_bounds__(256) rope_rows_kernel(RopeArgs a) {
    using I = Val<IN>;
    using O = Val<OUT>;
    constexpr int D = 16 * LANES, kHeads = 256 / LANES;
    const int sub = threadIdx.x % LANES;
    const int heads = (int)(a.q_heads + (a.v ? 2 : 1) * a.kv_heads), turned = (int)(a.q_heads + a.kv_heads);
    const int64_t t = blockIdx.x;
    const int rot = (int)a.rot;
    const int64_t pos = rot ? a.positions[t] : 0;
    const bool known = rot == 0 || (pos >= 0 && pos < a.n_pos);      // else the row is NaN
    const float* row = a.table + (known ? pos : 0) * rot;
    // eight elements at e0 = 8 sub and at D/2 + 8 sub
    float cs[2][8];
#pragma unroll
    for (int h = 0; h < 2; ++h) {
        const int at = INTER ? h * (D / 2) + 8 * sub : 16 * sub + 8 * h;     // of the table's row
#pragma unroll
        for (int i = 0; i < 8; i += 4) {
            float4 v = make_float4(1.f, 0.f, 1.f, 0.f);
            if (at + i < rot) v = *reinterpret_cast<const float4*>(row + at + i);    // rot is a multiple of 4
            cs[h][i] = v.x;
            cs[h][i + 1] = v.y;
            cs[h][i + 2] = v.z;
            cs[h][i + 3] = v.w;
        }
    }
    const typename I::Elem* xrow = static_cast<const typename I::Elem*>(a.x) + t * a.ld_x + 8 * sub;
    for (int h = (int)blockIdx.y * kHeads + (int)threadIdx.x / LANES; h < heads; h += (int)gridDim.y * kHeads) {
        float x[2][8];
        I::load8(xrow + h * D, x[0]);
        I::load8(xrow + h * D + D / 2, x[1]);
        const bool is_q = h < a.q_heads, is_v = h >= turned;
        const float* w = is_q ? a.q_norm : is_v ? nullptr : a.k_norm;
        if (w) {
            float ss = 0.f;
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fmaf(x[0][i], x[0][i], __builtin_fmaf(x[1][i], x[1][i], ss));
#pragma unroll
            for (int m = LANES >> 1; m; m >>= 1) ss += __shfl_xor(ss, m);
            const float r = 1.0f / sqrtf(ss / (float)D + a.eps);
#pragma unroll
            for (int k = 0; k < 2; ++k) {
                float wv[8];
                Val<kTypeF32>::load8(w + k * (D / 2) + 8 * sub, wv);
#pragma unroll
                for (int i = 0; i < 8; ++i) x[k][i] = x[k][i] * r * wv[i];
            }
        }
        if (!is_v) {
            if constexpr (INTER) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 8; i += 2) {
                        const float p = x[k][i], q = x[k][i + 1], c = cs[k][i], s = cs[k][i + 1];
                        const bool turn = k * (D / 2) + 8 * sub + i < rot;    // else they pass: 0 times an inf is a NaN
                        x[k][i] = turn ? __builtin_fmaf(p, c, -(q * s)) : p;
                        x[k][i + 1] = turn ? __builtin_fmaf(q, c, p * s) : q;
                    }
            } else if (rot) {
#pragma unroll
                for (int i = 0; i < 8; ++i) {
                    const float p = x[0][i], q = x[1][i], c = cs[i >> 2][(2 * i) & 7], s = cs[i >> 2][((2 * i) & 7) + 1];
                    x[0][i] = __builtin_fmaf(p, c, -(q * s));
                    x[1][i] = __builtin_fmaf(q, c, p * s);
                }
            }
            if (!known) {
#pragma unroll
                for (int k = 0; k < 2; ++k)
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[k][i] = __builtin_nanf("");
            }
        }
        typename O::Elem* dst =
            is_q ? static_cast<typename O::Elem*>(a.q) + t * a.ld_q + h * D
                 : is_v ? static_cast<typename O::Elem*>(a.v) + t * a.ld_v + (h - turned) * D
                        : static_cast<typename O::Elem*>(a.k) + t * a.ld_k + (h - (int)a.q_heads) * D;
        O::store8(dst + 8 * sub, x[0]);
        O::store8(dst + D / 2 + 8 * sub, x[1]);
    }
}

template <int IN, int OUT>
__global__ void __launch_bounds__(256) qk_norm_rope_kernel(RopeArgs a, int lanes) {
    using I = Val<IN>;
    using O = Val<OUT>;
    __shared__ float stage[256 * 8];
    const int heads = (int)(a.q_heads + (a.v ? 2 : 1) * a.kv_heads);
    const int sub = threadIdx.x & (lanes - 1);
    const int64_t t = blockIdx.x;
    const int h = (int)blockIdx.y * (256 / lanes) + threadIdx.x / lanes;
    if (h >= heads) return;                            // whole lane groups leave; nothing below waits for them
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

hipError_t launch_tokens(const RopeArgs& a, hipStream_t stream) {
    int lanes = 1;
    while (lanes * 8 < a.head_dim) lanes *= 2;
    const unsigned heads = (unsigned)(a.q_heads + (a.v ? 2 : 1) * a.kv_heads), tokens = (unsigned)a.tokens;
    const bool rows = lanes * 8 == a.head_dim && a.head_dim >= 64 && (a.interleaved || a.rot == a.head_dim || a.rot == 0) &&
                      (reinterpret_cast<uintptr_t>(a.table) & 15) == 0 && (a.rot % 4 == 0);
    return with_type(a.x_type, [&](auto in) {
        return with_type(a.out_type, [&](auto out) {
            constexpr int kIn = decltype(in)::value, kOut = decltype(out)::value;
            if (rows) {
                const auto run = [&](auto l) {
                    constexpr int kL = decltype(l)::value;
                    // all heads of a token in one workgroup, which loads its cosines
                    // once, unless that leaves the GPU empty
                    const unsigned parts = (heads + 256 / kL - 1) / (256 / kL);
                    const dim3 grid(tokens, tokens < 1024 ? parts : 1);
                    if (a.interleaved)
                        rope_rows_kernel<kIn, kOut, kL, true><<<grid, 256, 0, stream>>>(a);
                    else
                        rope_rows_kernel<kIn, kOut, kL, false><<<grid, 256, 0, stream>>>(a);
                    return hipGetLastError();
                };
                return a.head_dim == 64 ? run(Int<4>{}) : a.head_dim == 128 ? run(Int<8>{}) : run(Int<16>{});
            }
            const unsigned per = 256 / (unsigned)lanes;
            qk_norm_rope_kernel<kIn, kOut><<<dim3(tokens, (heads + per - 1) / per), 256, 0, stream>>>(a, lanes);
            return hipGetLastError();
        });
    });
}

}  // namespace

hipError_t launch_qk_norm_rope(const RopeArgs& all, hipStream_t stream) {
    constexpr int64_t kMost = (int64_t)1 << 23;        // tokens of 256 threads: a launch has fewer than 2^32
    RopeArgs a = all;
    const int64_t xs = a.x_type == kTypeF32 ? 4 : 2, os = a.out_type == kTypeF32 ? 4 : 2;
    for (int64_t at = 0; at < all.tokens; at += kMost) {
        a.tokens = all.tokens - at < kMost ? all.tokens - at : kMost;
        a.x = static_cast<const char*>(all.x) + at * a.ld_x * xs;
        a.q = static_cast<char*>(all.q) + at * a.ld_q * os;
        a.k = static_cast<char*>(all.k) + at * a.ld_k * os;
        if (all.v) a.v = static_cast<char*>(all.v) + at * a.ld_v * os;
        if (all.positions) a.positions = all.positions + at;
        if (const hipError_t e = launch_tokens(a, stream); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace frq
