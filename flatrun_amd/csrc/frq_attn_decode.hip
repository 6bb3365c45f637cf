// Attention of one query token per sequence against the 4-bit paged cache
// (frq_kv4.h):
//   S[h, t] = scale q_h . k_t,  t < len;   out_h = sum_t softmax(S)[h, t] v_t.
//
// The cache is read as it is held, once for up to eight query heads that share
// a key head. Both products run on v_mfma_f32_16x16x32_f16 with fp32 precision:
// the codes c - 8 are exact fp16 integers, and q and the softmax weights go in
// as two fp16 numbers each, rows h and h + 8 of the product (hi and the rest,
// 22 bits together). q is put under a power of two per head that brings its
// largest element to [2^13, 2^14), so that the rest stays a normal number. A
// block of K has its scale on the product of one instruction; the scale of V
// goes into the weights, under 2^(6 - E) with E the exponent of the largest
// |scale| seen, so that tiny and huge values keep their bits.
//
// S^T = K q^T leaves the tokens in the registers in which P V wants them, so
// nothing passes through LDS. Running maximum and sum per head in fp32. Each
// wave walks its own tiles; the waves of a workgroup meet in LDS at the end,
// and a sequence split over workgroups in a second, small kernel.
#include "frq_kernels.h"
#include "frq_kv4.h"

namespace frq {
namespace {

using half2v = _Float16 __attribute__((ext_vector_type(2)));
using half8v = _Float16 __attribute__((ext_vector_type(8)));
using float4v = float __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;

// Eight codes of a word as fp16 integers c - 8, pairs (nibble r, nibble r + 4).
// 0x6400 | n is 1024 + n; under the mask 0xF0 it is 1024 + 16 n.
__device__ __forceinline__ half2v low_pair(uint32_t w) {
    const half2v x = __builtin_bit_cast(half2v, (w & 0x000F000Fu) | 0x64006400u);
    return x - (half2v){1032, 1032};
}
__device__ __forceinline__ half2v high_pair(uint32_t w) {
    const half2v x = __builtin_bit_cast(half2v, (w & 0x00F000F0u) | 0x64006400u);
    return __builtin_elementwise_fma(x, (half2v){0.0625f16, 0.0625f16}, (half2v){-72, -72});
}
__device__ __forceinline__ half8v join(half2v a, half2v b, half2v c, half2v d) {
    return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ float half_of(uint32_t w, int hi) { return f16_bits_to_f32(hi ? w >> 16 : w); }

// 2^e as a float, e in the normal range.
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }

template <int TYPE, int NG>
__global__ void __launch_bounds__(64 * kWaves) attn_decode_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    constexpr int D = 32 * NG, kTile = kv_tile_bytes(NG);
    constexpr int kSW = 2 * NG;               // 32-bit words of the scales of four tokens
    __shared__ float sh_o[kWaves][8][D];
    __shared__ float sh_m[kWaves][8], sh_l[kWaves][8];

    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int n = lane & 15, j = lane >> 4;
    const int group = (int)(a.q_heads / a.kv_heads), chunks = (group + 7) / 8;
    int64_t id = blockIdx.x;
    const int split = (int)(id % a.splits);
    id /= a.splits;
    const int hc = (int)(id % chunks);
    id /= chunks;
    const int kvh = (int)(id % a.kv_heads);
    const int64_t b = id / a.kv_heads;

    const int64_t want = a.lens[b];
    bool bad = want > a.max_len;              // longer than the caller said: NaN
    const int64_t len = want < 0 ? 0 : bad ? 0 : want;
    const int tiles = (int)((len + kKvTile - 1) / kKvTile);
    const int first = split * a.chunk_tiles;
    const int last = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    const int rows = group - 8 * hc < 8 ? group - 8 * hc : 8;     // query heads here

    // q: row n & 7, hi or (n >= 8) the rest
    const int row = n & 7;
    half8v qf[NG];
    float rs = 0.f;
    {
        float x[NG][8], top = 0.f;
        bool odd = false;
        const typename T::Elem* qp = static_cast<const typename T::Elem*>(a.q) + b * a.ld_q +
                                     ((int64_t)kvh * group + 8 * hc + (row < rows ? row : 0)) * D;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            T::load8(qp + 32 * g + 8 * j, x[g]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float m = __builtin_fabsf(x[g][c]);
                odd |= !(m < __builtin_inff());
                top = __builtin_fmaxf(top, m);
            }
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        odd |= __shfl_xor((int)odd, 16) != 0;
        odd |= __shfl_xor((int)odd, 32) != 0;
        int e = 0;
        if (top > 0.f && !odd) (void)frexpf(top, &e);             // top in [2^(e-1), 2^e)
        const int up = 14 - e;                                    // -114 .. 163
        const int u1 = up / 2, u2 = up - u1;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float v = x[g][c] * pow2(u1) * pow2(u2);
                const _Float16 hi = (_Float16)v;
                qf[g][c] = n < 8 ? hi : (_Float16)(v - (float)hi);
            }
        }
        rs = odd ? __builtin_nanf("") : a.scale * kLog2e * pow2(-u1) * pow2(-u2);
    }

    float4v o[2 * NG];
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) o[i] = float4v{0, 0, 0, 0};
    float m = -__builtin_inff(), l = 0.f;
    int ev = -24;                              // exponent under which V's scales enter

    const int64_t page_tiles = a.page_tokens / kKvTile;
    for (int tile = first + wave; tile < last; tile += kWaves) {
        const int64_t pg = tile / page_tiles;
        const int64_t page = a.table[b * a.ld_table + pg];
        if (page < 0 || page >= a.pages) {
            bad = true;
            break;
        }
        const uint8_t* tp = static_cast<const uint8_t*>(a.cache) +
                            ((page * a.kv_heads + kvh) * page_tiles + (tile - pg * page_tiles)) * (int64_t)kTile;
        uint32_t kw[2 * NG], vw[2 * NG], ks[2][kSW], vs[2][kSW];
#pragma unroll
        for (int p = 0; p < 2 * NG; p += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(tp + kv_word(p, lane));
            const uint4 y = *reinterpret_cast<const uint4*>(tp + kv_vc_off(NG) + kv_word(p, lane));
            kw[p] = x.x; kw[p + 1] = x.y; kw[p + 2] = x.z; kw[p + 3] = x.w;
            vw[p] = y.x; vw[p + 1] = y.y; vw[p + 2] = y.z; vw[p + 3] = y.w;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int p = 0; p < kSW; p += 4) {
                const int at = (16 * u + 4 * j) * NG * 2 + 4 * p;
                const uint4 x = *reinterpret_cast<const uint4*>(tp + kv_ks_off(NG) + at);
                const uint4 y = *reinterpret_cast<const uint4*>(tp + kv_vs_off(NG) + at);
                ks[u][p] = x.x; ks[u][p + 1] = x.y; ks[u][p + 2] = x.z; ks[u][p + 3] = x.w;
                vs[u][p] = y.x; vs[u][p + 1] = y.y; vs[u][p + 2] = y.z; vs[u][p + 3] = y.w;
            }
        }
        // S^T: tokens 16u + 4j + i of head row n
        float s[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = 0.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t w = kw[u * NG + g];
                const half8v kf = join(low_pair(w), high_pair(w), low_pair(w >> 8), high_pair(w >> 8));
                const float4v c = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, qf[g], float4v{0, 0, 0, 0}, 0, 0, 0);
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    const int at = i * NG + g;
                    s[u][i] = __builtin_fmaf(c[i], half_of(ks[u][at / 2], at & 1), s[u][i]);
                }
            }
#pragma unroll
            for (int i = 0; i < 4; ++i) s[u][i] = (s[u][i] + __shfl_xor(s[u][i], 8)) * rs;
        }
        const int left = (int)(len - (int64_t)tile * kKvTile);     // valid tokens from here
        if (left < kKvTile) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
#pragma unroll
                for (int i = 0; i < 4; ++i) {
                    if (16 * u + 4 * j + i >= left) {
                        s[u][i] = -__builtin_inff();
#pragma unroll
                        for (int p = 0; p < NG / 2; ++p) vs[u][i * NG / 2 + p] = 0;
                    }
                }
            }
        }
        float top = s[0][0];
#pragma unroll
        for (int i = 1; i < 8; ++i) top = __builtin_fmaxf(top, s[i >> 2][i & 3]);
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        float big = 0.f;
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 2 * kSW; ++i) big = __builtin_fmaxf(big, __builtin_fabsf(half_of(vs[u][i / 2], i & 1)));
        }
        big = __builtin_fmaxf(big, __shfl_xor(big, 16));
        big = __builtin_fmaxf(big, __shfl_xor(big, 32));
        int eb = -24;
        if (big > 0.f) {
            (void)frexpf(big, &eb);
            --eb;
        }
        eb = eb > ev ? eb : ev;
        const float mn = __builtin_fmaxf(m, top);
        const float ref = mn == -__builtin_inff() ? 0.f : mn;
        const float keep = __builtin_amdgcn_exp2f(m - ref);
        const float down = pow2(ev - eb);
        l *= keep;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float k = __shfl(keep, 4 * j + i) * down;
#pragma unroll
            for (int c = 0; c < 2 * NG; ++c) o[c][i] *= k;
        }
        m = mn;
        ev = eb;
        const float lift = pow2(6 - ev);
        float p[2][4];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                p[u][i] = __builtin_amdgcn_exp2f(s[u][i] - ref);
                l += p[u][i];
                p[u][i] *= lift;
            }
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            half8v pf;
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const int at = (e & 3) * NG + g;
                const float v = p[e >> 2][e & 3] * half_of(vs[e >> 2][at / 2], at & 1);
                const _Float16 hi = (_Float16)v;
                pf[e] = n < 8 ? hi : (_Float16)(v - (float)hi);
            }
            const uint32_t w0 = vw[2 * g], w1 = vw[2 * g + 1];
            const half8v va = join(low_pair(w0), low_pair(w0 >> 8), low_pair(w1), low_pair(w1 >> 8));
            const half8v vb = join(high_pair(w0), high_pair(w0 >> 8), high_pair(w1), high_pair(w1 >> 8));
            o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, va, o[2 * g], 0, 0, 0);
            o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, vb, o[2 * g + 1], 0, 0, 0);
        }
    }
    // join: hi and rest, lane groups, waves
    l += __shfl_xor(l, 16);
    l += __shfl_xor(l, 32);
    if (bad) l = __builtin_nanf("");
    const float back = pow2(ev - 6);
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const float v = (o[c][i] + __shfl_xor(o[c][i], 32)) * back;
            if (j < 2) sh_o[wave][4 * j + i][16 * c + n] = v;
        }
    }
    if (lane < 8) {
        sh_m[wave][lane] = m;
        sh_l[wave][lane] = l;
    }
    __syncthreads();
    for (int at = threadIdx.x; at < rows * D; at += 64 * kWaves) {
        const int r = at / D, c = at - r * D;
        float mm = sh_m[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mm = __builtin_fmaxf(mm, sh_m[w][r]);
        const float ref = mm == -__builtin_inff() ? 0.f : mm;
        float sum = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sh_m[w][r] - ref);
            sum += f * sh_l[w][r];
            val += f * sh_o[w][r][c];
        }
        const int64_t h = (int64_t)kvh * group + 8 * hc + r;
        if (a.splits == 1) {
            static_cast<typename T::Elem*>(a.out)[b * a.ld_out + h * D + c] = T::one(sum == 0.f ? 0.f : val / sum);
        } else {
            const int64_t part = (b * a.q_heads + h) * a.splits + split;
            a.part_o[part * D + c] = val;
            if (c == 0) {
                a.part_ml[2 * part] = mm;
                a.part_ml[2 * part + 1] = sum;
            }
        }
    }
}

// out = the splits of a row joined in their order.
template <int TYPE>
__global__ void __launch_bounds__(256) attn_join_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    const int64_t r = blockIdx.x;
    const int D = (int)a.head_dim, c = threadIdx.x;
    const float* ml = a.part_ml + 2 * r * a.splits;
    float mm = -__builtin_inff();
    for (int s = 0; s < a.splits; ++s) mm = __builtin_fmaxf(mm, ml[2 * s]);
    const float ref = mm == -__builtin_inff() ? 0.f : mm;
    float sum = 0.f, val = 0.f;
    for (int s = 0; s < a.splits; ++s) {
        const float f = __builtin_amdgcn_exp2f(ml[2 * s] - ref);
        sum += f * ml[2 * s + 1];
        if (c < D) val += f * a.part_o[(r * a.splits + s) * D + c];
    }
    const int64_t b = r / a.q_heads, h = r - b * a.q_heads;
    if (c < D) static_cast<typename T::Elem*>(a.out)[b * a.ld_out + h * D + c] = T::one(sum == 0.f ? 0.f : val / sum);
}

}  // namespace

void plan_attn_decode(DecodeArgs* a) {
    const int64_t tiles = (a->max_len + kKvTile - 1) / kKvTile;
    const int64_t group = a->q_heads / a->kv_heads, base = a->batch * a->kv_heads * ((group + 7) / 8);
    int64_t splits = (1024 + base - 1) / base;
    const int64_t most = (tiles + kWaves - 1) / kWaves;
    splits = splits > most ? most : splits;
    splits = splits < 1 ? 1 : splits;
    a->chunk_tiles = (int)((tiles + splits - 1) / splits);
    a->splits = (int)(tiles ? (tiles + a->chunk_tiles - 1) / a->chunk_tiles : 1);
}

size_t attn_decode_scratch(const DecodeArgs& a) {
    return a.splits == 1 ? 0 : sizeof(float) * (size_t)(a.batch * a.q_heads * a.splits) * (size_t)(a.head_dim + 2);
}

hipError_t launch_attn_decode(DecodeArgs a, float* scratch, hipStream_t stream) {
    const int64_t group = a.q_heads / a.kv_heads;
    const int64_t grid = a.batch * a.kv_heads * ((group + 7) / 8) * a.splits;
    a.part_o = scratch;
    a.part_ml = scratch ? scratch + a.batch * a.q_heads * a.splits * a.head_dim : nullptr;
    return with_type(a.type, [&](auto ty) {
        constexpr int kT = decltype(ty)::value;
        switch (a.head_dim) {
            case 64: attn_decode_kernel<kT, 2><<<(unsigned)grid, 64 * kWaves, 0, stream>>>(a); break;
            case 128: attn_decode_kernel<kT, 4><<<(unsigned)grid, 64 * kWaves, 0, stream>>>(a); break;
            case 256: attn_decode_kernel<kT, 8><<<(unsigned)grid, 64 * kWaves, 0, stream>>>(a); break;
            default: return hipErrorInvalidValue;
        }
        if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) return e;
        attn_join_kernel<kT><<<(unsigned)(a.batch * a.q_heads), 256, 0, stream>>>(a);
        return hipGetLastError();
    });
}

}  // namespace frq
