// Attention over packed sequences of different lengths:
//   S[i, j] = scale q_i . k_j,  out_i = sum_j softmax(S)[i, j] v_j
// for the queries and keys of each sequence, j <= i + (keys - queries) where
// causal, query heads grouped over key heads. A query that no key is left for
// gives zeros.
//
// Bound by the matrix cores on long prompts: v_mfma_f32_32x32x16 in bf16 or
// fp16 with fp32 sums; scores, running maximum and sum in fp32; the softmax
// weights are rounded to the inputs' type for the second product, as their
// values are (the error that leaves is below the inputs' own rounding).
//
// A workgroup takes 128 queries of one head, a wave 32, and walks keys 64 at a
// time through LDS. The products are S^T = K Q^T and O^T = V^T P^T: a lane then
// holds one query's scores in both, the maximum and sum need one exchange
// between the wave's halves, and P^T is in the registers the second product
// reads, with the keys in the order in which S^T left them; V^T comes from the
// row-major tile by transposing LDS reads.
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr int kWaves = 4, kKeys = 64, kRows = 32 * kWaves;

template <int TYPE>
__device__ __forceinline__ f32x16 mfma(uint4 a, uint4 b, f32x16 c) {
    if constexpr (TYPE == kTypeBF16)
        return __builtin_amdgcn_mfma_f32_32x32x16_bf16(__builtin_bit_cast(bf16x8, a), __builtin_bit_cast(bf16x8, b), c, 0,
                                                       0, 0);
    else
        return __builtin_amdgcn_mfma_f32_32x32x16_f16(__builtin_bit_cast(f16x8, a), __builtin_bit_cast(f16x8, b), c, 0, 0,
                                                      0);
}

template <int TYPE>
__device__ __forceinline__ uint32_t pack2(float a, float b) {
    return (uint32_t)Val<TYPE>::one(a) | ((uint32_t)Val<TYPE>::one(b) << 16);
}

// Whether one of eight 16-bit values is an inf or a NaN.
template <int TYPE>
__device__ __forceinline__ bool any_special(uint4 v) {
    constexpr uint32_t e = TYPE == kTypeBF16 ? 0x7F80u : 0x7C00u;
    const uint32_t w[4] = {v.x, v.y, v.z, v.w};
    bool r = false;
#pragma unroll
    for (int i = 0; i < 4; ++i) r |= (w[i] & e) == e || ((w[i] >> 16) & e) == e;
    return r;
}

template <int TYPE>
__device__ __forceinline__ float widen(uint16_t b) {
    if constexpr (TYPE == kTypeBF16) return __builtin_bit_cast(float, (uint32_t)b << 16);
    return f16_bits_to_f32(b);
}

// Four keys of one column: the 16 lanes of a block point at the 16 groups of
// four columns of four rows (lane 4r + c: row r, columns 4c .. 4c + 3), lane i
// gets column i.
__device__ __forceinline__ uint2 read_column4(const uint16_t* p) {
    const s16x4 v =
        __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)const_cast<uint16_t*>(p));
    return __builtin_bit_cast(uint2, v);
}

template <int TYPE, int OUT, int D>
__global__ void __launch_bounds__(64 * kWaves) attn_prefill_kernel(PrefillArgs a) {
    constexpr int NK = D / 16, ND = D / 32, CH = D / 8;          // k-steps, column tiles, 16-byte pieces of a row
    __shared__ __attribute__((aligned(16))) uint16_t sk[kKeys * D], sv[kKeys * D];
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int ln = lane & 31, h = lane >> 5;
    int64_t id = blockIdx.x;
    const int head = (int)(id % a.q_heads);
    id /= a.q_heads;
    const int seq = (int)(id % a.seqs);
    const int64_t qb = a.q_blocks - 1 - id / a.seqs;             // the longest rows first
    const int64_t q0 = a.cu_q[seq], k0 = a.cu_k[seq];
    const int64_t nq = a.cu_q[seq + 1] - q0, nk = a.cu_k[seq + 1] - k0;
    if (q0 < 0 || k0 < 0 || nk < 0 || q0 + nq > a.tokens_q || k0 + nk > a.tokens_k || qb * kRows >= nq) return;
    const int64_t past = nk - nq;
    const int64_t i0 = qb * kRows + 32 * wave;                   // the wave's first query
    const int64_t qi = i0 + ln;                                  // the lane's
    int64_t end = nk;                                            // keys that the workgroup needs
    if (a.causal) {
        const int64_t e = (qb + 1) * kRows + past;
        end = e < nk ? e : nk;
    }
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (q0 + (qi < nq ? qi : nq - 1)) * a.ld_q + head * a.hs_q;
    const int64_t kvh = head / (a.q_heads / a.kv_heads);
    const uint16_t* kp = static_cast<const uint16_t*>(a.k) + k0 * a.ld_k + kvh * a.hs_k;
    const uint16_t* vp = static_cast<const uint16_t*>(a.v) + k0 * a.ld_v + kvh * a.hs_v;

    uint4 qf[NK];
#pragma unroll
    for (int s = 0; s < NK; ++s) qf[s] = *reinterpret_cast<const uint4*>(q + 16 * s + 8 * h);
    f32x16 o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -__builtin_inff(), l = 0.f;
    const float c = a.scale * 1.4426950408889634f;

    for (int64_t kt = 0; kt < end; kt += kKeys) {
        __syncthreads();
        for (int at = threadIdx.x; at < kKeys * CH; at += 64 * kWaves) {
            const int r = at / CH, p = at % CH;
            const bool on = kt + r < nk;                         // rows past the sequence are zeros
            const uint4 z = make_uint4(0, 0, 0, 0);
            const int to = r * D + 8 * (p ^ (r & (CH - 1)));
            *reinterpret_cast<uint4*>(sk + to) = on ? *reinterpret_cast<const uint4*>(kp + (kt + r) * a.ld_k + 8 * p) : z;
            *reinterpret_cast<uint4*>(sv + to) = on ? *reinterpret_cast<const uint4*>(vp + (kt + r) * a.ld_v + 8 * p) : z;
        }
        __syncthreads();
        const int64_t limit = a.causal ? qi + past : nk - 1;     // the lane's last key
        const int64_t lim = limit < nk - 1 ? limit : nk - 1;
        if (a.causal && kt > i0 + 31 + past) continue;           // nothing here for the wave
        const bool masked = kt + kKeys > nk || (a.causal && kt + kKeys - 1 > i0 + past);
        f32x16 st[2];
#pragma unroll
        for (int t = 0; t < 2; ++t) {
#pragma unroll
            for (int i = 0; i < 16; ++i) st[t][i] = 0.f;
#pragma unroll
            for (int s = 0; s < NK; ++s) {
                const int r = 32 * t + ln;
                const uint4 kf = *reinterpret_cast<const uint4*>(sk + r * D + 8 * ((2 * s + h) ^ (r & (CH - 1))));
                st[t] = mfma<TYPE>(kf, qf[s], st[t]);
            }
        }
        if (masked) {
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (kt + 32 * t + 8 * (i >> 2) + 4 * h + (i & 3) > lim) st[t][i] = -__builtin_inff();
        }
        float top = st[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, st[t][i]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        const float mn = __builtin_fmaxf(m, top * c);
        const float ref = mn == -__builtin_inff() ? 0.f : mn;
        const float keep = __builtin_amdgcn_exp2f(m - ref);
        m = mn;
        l *= keep;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; ++i) o[d][i] *= keep;
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                st[t][i] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[t][i], c, -ref));
                l += st[t][i];
            }
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            const f32x16& p = st[s >> 1];
            const int b = 8 * (s & 1);
            uint4 pf;
            pf.x = pack2<TYPE>(p[b + 0], p[b + 1]);
            pf.y = pack2<TYPE>(p[b + 2], p[b + 3]);
            pf.z = pack2<TYPE>(p[b + 4], p[b + 5]);
            pf.w = pack2<TYPE>(p[b + 6], p[b + 7]);
            const int key = 16 * s + 4 * h + ((lane & 15) >> 2);
#pragma unroll
            for (int d = 0; d < ND; ++d) {
                const int col = 32 * d + (lane & 16) + 4 * (lane & 3);
                const uint2 lo = read_column4(sv + key * D + 8 * ((col / 8) ^ (key & (CH - 1))) + (col & 7));
                const uint2 hi = read_column4(sv + (key + 8) * D + 8 * ((col / 8) ^ ((key + 8) & (CH - 1))) + (col & 7));
                const uint4 vf = make_uint4(lo.x, lo.y, hi.x, hi.y);
                if (masked && __builtin_amdgcn_ballot_w64(any_special<TYPE>(vf))) {
                    // an inf or NaN among these values: keys that the mask takes must not meet it
#pragma unroll
                    for (int e = 0; e < 16; ++e) {
                        // key 16 s + e is element e of the step: held by the half (e >> 2) & 1
                        const float mine = p[b + (e & 3) + 4 * (e >> 3)];
                        const float other = __shfl_xor(mine, 32);
                        const float w = ((e >> 2) & 1) == h ? mine : other;
                        const int kr = 16 * s + e;
                        if (kt + kr <= lim) {
#pragma unroll
                            for (int i = 0; i < 16; ++i) {
                                const int cc = 32 * d + 8 * (i >> 2) + 4 * h + (i & 3);
                                const uint16_t vb = sv[kr * D + 8 * ((cc / 8) ^ (kr & (CH - 1))) + (cc & 7)];
                                o[d][i] = __builtin_fmaf(w, widen<TYPE>(vb), o[d][i]);
                            }
                        }
                    }
                } else {
                    o[d] = mfma<TYPE>(vf, pf, o[d]);
                }
            }
        }
    }
    l += __shfl_xor(l, 32);
    if (qi >= nq) return;
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    using O = Val<OUT>;
    typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (q0 + qi) * a.ld_out + head * a.hs_out;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) out[32 * d + 8 * (i >> 2) + 4 * h + (i & 3)] = O::one(l == 0.f ? 0.f : o[d][i] * inv);
}

template <int TYPE, int OUT>
hipError_t launch_typed(const PrefillArgs& a, unsigned grid, hipStream_t stream) {
    switch (a.head_dim) {
        case 64: attn_prefill_kernel<TYPE, OUT, 64><<<grid, 64 * kWaves, 0, stream>>>(a); break;
        case 128: attn_prefill_kernel<TYPE, OUT, 128><<<grid, 64 * kWaves, 0, stream>>>(a); break;
        case 256: attn_prefill_kernel<TYPE, OUT, 256><<<grid, 64 * kWaves, 0, stream>>>(a); break;
        default: return hipErrorInvalidValue;
    }
    return hipGetLastError();
}

}  // namespace

hipError_t launch_attn_prefill(PrefillArgs a, hipStream_t stream) {
    a.q_blocks = (a.max_q + kRows - 1) / kRows;
    const unsigned grid = (unsigned)(a.q_blocks * a.seqs * a.q_heads);
    if (a.type == kTypeBF16)
        return a.out_type == kTypeF32 ? launch_typed<kTypeBF16, kTypeF32>(a, grid, stream)
                                      : launch_typed<kTypeBF16, kTypeBF16>(a, grid, stream);
    return a.out_type == kTypeF32 ? launch_typed<kTypeF16, kTypeF32>(a, grid, stream)
                                  : launch_typed<kTypeF16, kTypeF16>(a, grid, stream);
}

}  // namespace frq
