// Attention of one query token per sequence against the 4-bit paged cache
// (frq_kv4.h):
//   S[h, t] = scale q_h . k_t,  t < len;   out_h = sum_t softmax(S)[h, t] v_t.
//
// The cache is read as it is held, once for up to eight query heads that share
// a key head. Both products run on v_mfma_f32_16x16x32_f16 with fp32 precision:
// the codes c - 8 are exact fp16 integers, and q and the softmax weights go in
// as two fp16 numbers each, rows 2h and 2h + 1 of the product (the value and
// the rest, 22 bits together). q is put under a power of two per head that
// brings its largest element to [2^13, 2^14), so that the rest stays a normal
// number. A block of K has its scale on the product of one instruction; the
// scale of V goes into the weights, which stand under 2^(6 - E) with E the
// exponent of the largest |scale| seen, so that tiny and huge values keep
// their bits: out = sum / sum, the power cancels.
//
// A wave takes 32 tokens a step. S = q K^T gives a lane one token of each half
// and both numbers of two heads, so scores, weights and their scales need no
// other lane; the weights pass through LDS, a wave's own part of it, to stand
// as the second product's operand (transposing reads). The reference that the
// exponentials are taken from follows the running maximum only when that is
// 2^8 ahead, so sums are rarely rescaled and the maximum over lanes is rarely
// taken. The next step's tile is loaded while this one is worked on.
//
// Each wave walks its own tiles; the waves of a workgroup meet in LDS at the
// end, and a sequence split over workgroups in a second, small kernel.
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
    const half2v x = __builtin_bit_cast(half2v, vand_or(w, 0x000F000Fu, 0x64006400u));
    return x - (half2v){1032, 1032};
}
__device__ __forceinline__ half2v high_pair(uint32_t w) {
    const half2v x = __builtin_bit_cast(half2v, vand_or(w, 0x00F000F0u, 0x64006400u));
    return __builtin_elementwise_fma(x, (half2v){0.0625f16, 0.0625f16}, (half2v){-72, -72});
}
__device__ __forceinline__ half2v pair_of(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ half8v join(half2v a, half2v b, half2v c, half2v d) {
    return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ _Float16 half_of(uint32_t w, int hi) {
    return __builtin_bit_cast(_Float16, (uint16_t)(hi ? w >> 16 : w));
}

// 2^e as a float, e in the normal range.
__device__ __forceinline__ float pow2(int e) { return __builtin_bit_cast(float, (uint32_t)(127 + e) << 23); }

// The largest of x over the 16 lanes of a row.
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
    for (int i = 1; i <= 8; i <<= 1) x = __builtin_fmaxf(x, __shfl_xor(x, i));
    return x;
}

// A tile as a lane holds it.
template <int NG>
struct Tile {
    uint32_t kw[2 * NG], vw[2 * NG], ks[NG], vs[NG];     // ks, vs: words u NG/2 + g/2
    __device__ __forceinline__ void load(const uint8_t* t, int lane) {
#pragma unroll
        for (int p = 0; p < 2 * NG; p += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(t + kv_word(p, lane));
            const uint4 y = *reinterpret_cast<const uint4*>(t + kv_vc_off(NG) + kv_word(p, lane));
            kw[p] = x.x; kw[p + 1] = x.y; kw[p + 2] = x.z; kw[p + 3] = x.w;
            vw[p] = y.x; vw[p + 1] = y.y; vw[p + 2] = y.z; vw[p + 3] = y.w;
        }
        const uint8_t* k = t + kv_ks_off(NG) + kv_scale(lane & 15, 0, NG);
        const uint8_t* v = t + kv_vs_off(NG) + kv_scale(lane & 15, 0, NG);
#pragma unroll
        for (int p = 0; p < NG; p += 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(k + 4 * p), y = *reinterpret_cast<const uint2*>(v + 4 * p);
            ks[p] = x.x; ks[p + 1] = x.y;
            vs[p] = y.x; vs[p + 1] = y.y;
        }
    }
};

using lds_bytes = __attribute__((address_space(3))) char*;
using short4v = short __attribute__((ext_vector_type(4)));
using uint2v = uint32_t __attribute__((ext_vector_type(2)));

template <int TYPE, int NG>
__global__ void __launch_bounds__(64 * kWaves, NG == 8 ? 1 : 2) attn_decode_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    constexpr int D = 32 * NG, kTile = kv_tile_bytes(NG);
    // the waves' weights [group][token][row] while tiles last, then their results
    constexpr int kOut = kWaves * 8 * D * 4, kP = kWaves * NG * 1024;
    __shared__ __attribute__((aligned(16))) char sh[kOut > kP ? kOut : kP];
    __shared__ float sh_m[kWaves][8], sh_l[kWaves][8];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    const uint32_t chunks = (uint32_t)(group + 7) / 8;
    uint32_t id = blockIdx.x;
    const int split = (int)(id % (uint32_t)a.splits);
    id /= (uint32_t)a.splits;
    const int hc = chunks == 1 ? 0 : (int)(id % chunks);
    id /= chunks;
    const int kvh = (int)(id % (uint32_t)a.kv_heads);
    const int64_t b = id / (uint32_t)a.kv_heads;

    const int64_t want = a.lens[b];
    bool bad = want > a.max_len || (want > 0 && a.pages == 0);       // not what the caller said: NaN
    const int len = want < 0 || bad ? 0 : (int)want;
    const int tiles = (len + kKvTile - 1) / kKvTile;
    const int first = split * a.chunk_tiles;
    const int last = first + a.chunk_tiles < tiles ? first + a.chunk_tiles : tiles;
    const int rows = group - 8 * hc < 8 ? group - 8 * hc : 8;        // query heads here
    if (first >= last && split > 0) {                                // nothing of the sequence: the join skips it
        return;
    }

    // this wave's tiles, their pages one ahead
    const uint32_t page_tiles = (uint32_t)a.page_tokens / kKvTile;
    const int32_t* table = a.table + b * a.ld_table;
    const uint8_t* heads = static_cast<const uint8_t*>(a.cache) + (int64_t)kvh * page_tiles * kTile;
    const int64_t page_bytes = a.kv_heads * (int64_t)page_tiles * kTile;
    auto tile_at = [&](int tile) {
        const uint32_t pg = (uint32_t)tile / page_tiles, in = (uint32_t)tile - pg * page_tiles;
        int64_t page = table[pg];
        if (page < 0 || page >= a.pages) {
            bad = true;
            page = 0;
        }
        return heads + page * page_bytes + (int64_t)in * kTile;
    };
    int tile = first + wave;
    Tile<NG> even, odd;
    if (tile < last) even.load(tile_at(tile), lane);

    // q: row n holds head n / 2, the value or (n odd) the rest
    half8v qf[NG];
    float rs;
    {
        const int row = n >> 1;
        float x[NG][8], top = 0.f;
        bool special = false;
        const typename T::Elem* qp = static_cast<const typename T::Elem*>(a.q) + b * a.ld_q +
                                     ((int64_t)kvh * group + 8 * hc + (row < rows ? row : 0)) * D;
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            T::load8(qp + 32 * g + 8 * j, x[g]);
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float m = __builtin_fabsf(x[g][c]);
                special |= !(m < __builtin_inff());
                top = __builtin_fmaxf(top, m);
            }
        }
        top = __builtin_fmaxf(top, __shfl_xor(top, 16));
        top = __builtin_fmaxf(top, __shfl_xor(top, 32));
        special |= __shfl_xor((int)special, 16) != 0;
        special |= __shfl_xor((int)special, 32) != 0;
        int e = 0;
        if (top > 0.f && !special) (void)frexpf(top, &e);            // top in [2^(e-1), 2^e)
        const int up = 14 - e, u1 = up / 2, u2 = up - u1;            // up is -114 .. 162
#pragma unroll
        for (int g = 0; g < NG; ++g) {
#pragma unroll
            for (int c = 0; c < 8; ++c) {
                const float v = x[g][c] * pow2(u1) * pow2(u2);
                const _Float16 hi = (_Float16)v;
                qf[g][c] = n & 1 ? (_Float16)(v - (float)hi) : hi;
            }
        }
        rs = special ? __builtin_nanf("") : a.scale * kLog2e * pow2(-u1) * pow2(-u2);
    }
    // of the lane's two heads 2j and 2j + 1: rows 4j .. 4j + 3 of both products
    const float rs2[2] = {__shfl(rs, 4 * j), __shfl(rs, 4 * j + 2)};
    float ref[2] = {-__builtin_inff(), -__builtin_inff()}, l[2] = {0.f, 0.f};
    int ev = -24;                                                    // E
    float4v o[2 * NG];
#pragma unroll
    for (int i = 0; i < 2 * NG; ++i) o[i] = float4v{0, 0, 0, 0};

    const lds_bytes sp = (lds_bytes)sh + wave * (NG * 1024);
    const lds_bytes sp_to = sp + n * 32 + j * 8, sp_from = sp + lane * 8;

    auto step = [&](Tile<NG>& t, int tile) __attribute__((always_inline)) {
        // scores of tokens n and 16 + n for heads 2j, 2j + 1
        float s[2][2];
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const uint32_t w = t.kw[u * NG + g];
                const half8v kf = join(low_pair(w), high_pair(w), low_pair(w >> 8), high_pair(w >> 8));
                const float4v c = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[g], kf, float4v{0, 0, 0, 0}, 0, 0, 0);
                const int at = u * NG + g;
                const float d = (float)half_of(t.ks[at / 2], at & 1);
#pragma unroll
                for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(c[i], d, acc[i]);
            }
            s[u][0] = (acc[0] + acc[1]) * rs2[0];
            s[u][1] = (acc[2] + acc[3]) * rs2[1];
        }
        const int left = len - tile * kKvTile;                       // valid tokens from here
        if (left < kKvTile) {
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                if (16 * u + n >= left) {
                    s[u][0] = s[u][1] = -__builtin_inff();
#pragma unroll
                    for (int p = 0; p < NG / 2; ++p) t.vs[u * (NG / 2) + p] = 0;
                }
            }
        }
        // a score 2^8 past its reference's maximum, or a scale past E?
        uint32_t big = 0;
#pragma unroll
        for (int p = 0; p < NG; ++p) {
            const uint32_t w = t.vs[p] & 0x7FFF7FFFu;
            using us2 = unsigned short __attribute__((ext_vector_type(2)));
            big = __builtin_bit_cast(uint32_t, __builtin_elementwise_max(__builtin_bit_cast(us2, big), __builtin_bit_cast(us2, w)));
        }
        const float cap = pow2(ev + 1);
        const float b0 = (float)half_of(big, 0), b1 = (float)half_of(big, 1);
        const float t0 = __builtin_fmaxf(s[0][0], s[1][0]), t1 = __builtin_fmaxf(s[0][1], s[1][1]);
        const float room = (float)(14 - ev);                         // ref = maximum - 6 + E
        if (__builtin_amdgcn_ballot_w64(t0 > ref[0] + room || t1 > ref[1] + room || !(b0 < cap) || !(b1 < cap))) {
            float top = 0.f;                                         // of the scales that are numbers
#pragma unroll
            for (int p = 0; p < 2 * NG; ++p) {
                const float v = __builtin_fabsf((float)half_of(t.vs[p / 2], p & 1));
                top = v < __builtin_inff() ? __builtin_fmaxf(top, v) : top;
            }
            top = row_max(top);
            int e = ev;
            if (top >= cap) {
                (void)frexpf(top, &e);
                --e;
            }
            const float up = (float)(e - ev);
#pragma unroll
            for (int i = 0; i < 2; ++i) {
                const float now = row_max(i ? t1 : t0) - 6.f + (float)e;
                const float r = __builtin_fmaxf(ref[i] + up, now);
                const float keep = r == ref[i] ? 1.f : __builtin_amdgcn_exp2f(ref[i] - r);
                ref[i] = r;
                l[i] *= keep;
#pragma unroll
                for (int c = 0; c < 2 * NG; ++c) {
                    o[c][2 * i] *= keep;
                    o[c][2 * i + 1] *= keep;
                }
            }
            ev = e;
        }
#pragma unroll
        for (int u = 0; u < 2; ++u) {
            const float p0 = __builtin_amdgcn_exp2f(s[u][0] - ref[0]), p1 = __builtin_amdgcn_exp2f(s[u][1] - ref[1]);
            l[0] += p0;
            l[1] += p1;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
                const int at = u * NG + g;
                const float d = (float)half_of(t.vs[at / 2], at & 1);
                const _Float16 h0 = (_Float16)__builtin_fmaf(p0, d, 0.f), h1 = (_Float16)__builtin_fmaf(p1, d, 0.f);
                const _Float16 r0 = (_Float16)__builtin_fmaf(p0, d, -(float)h0), r1 = (_Float16)__builtin_fmaf(p1, d, -(float)h1);
                const half2v x = {h0, r0}, y = {h1, r1};
                *(__attribute__((address_space(3))) uint2v*)(sp_to + g * 1024 + u * 512) =
                    uint2v{__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
            }
        }
        __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
        __builtin_amdgcn_wave_barrier();
        __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            using tr = __attribute__((address_space(3))) short4v*;
            const uint2v x = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(sp_from + g * 1024)));
            const uint2v y = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(sp_from + g * 1024 + 512)));
            const half8v pf = join(pair_of(x[0]), pair_of(x[1]), pair_of(y[0]), pair_of(y[1]));
            const uint32_t w0 = t.vw[2 * g], w1 = t.vw[2 * g + 1];
            const half8v va = join(low_pair(w0), low_pair(w0 >> 8), low_pair(w1), low_pair(w1 >> 8));
            const half8v vb = join(high_pair(w0), high_pair(w0 >> 8), high_pair(w1), high_pair(w1 >> 8));
            o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, va, o[2 * g], 0, 0, 0);
            o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, vb, o[2 * g + 1], 0, 0, 0);
        }
        __builtin_amdgcn_wave_barrier();
    };
    while (tile < last) {
        if (tile + kWaves < last) odd.load(tile_at(tile + kWaves), lane);
        step(even, tile);
        tile += kWaves;
        if (tile >= last) break;
        if (tile + kWaves < last) even.load(tile_at(tile + kWaves), lane);
        step(odd, tile);
        tile += kWaves;
    }
    // join the lanes' sums, then the waves
    if (__builtin_amdgcn_ballot_w64(bad)) l[0] = l[1] = __builtin_nanf("");
#pragma unroll
    for (int i = 0; i < 2; ++i) {
#pragma unroll
        for (int k = 1; k <= 8; k <<= 1) l[i] += __shfl_xor(l[i], k);
        if (n == 0) {
            sh_m[wave][2 * j + i] = ref[i];
            sh_l[wave][2 * j + i] = l[i];
        }
    }
    __syncthreads();
    float* sh_o = reinterpret_cast<float*>(sh);
#pragma unroll
    for (int c = 0; c < 2 * NG; ++c) {
        sh_o[(wave * 8 + 2 * j) * D + 16 * c + n] = o[c][0] + o[c][1];
        sh_o[(wave * 8 + 2 * j + 1) * D + 16 * c + n] = o[c][2] + o[c][3];
    }
    __syncthreads();
    const bool whole = a.splits == 1;
    for (int at = threadIdx.x; at < rows * D; at += 64 * kWaves) {
        const int r = at / D, c = at - r * D;
        float mm = sh_m[0][r];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mm = __builtin_fmaxf(mm, sh_m[w][r]);
        const float base = mm == -__builtin_inff() ? 0.f : mm;
        float sum = 0.f, val = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) {
            const float f = __builtin_amdgcn_exp2f(sh_m[w][r] - base);
            sum += f * sh_l[w][r];
            val += f * sh_o[(w * 8 + r) * D + c];
        }
        const int64_t h = (int64_t)kvh * group + 8 * hc + r;
        if (whole) {
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

// out = the splits of a row, joined in their order: 256 / (D / 4) splits at a
// time, four columns a thread, then over those.
template <int TYPE, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    constexpr int kCols = D / 4, kAt = 256 / kCols;
    __shared__ float part[kAt][D], sums[kAt];
    const int64_t r = blockIdx.x;
    const int64_t b = (uint32_t)r / (uint32_t)a.q_heads, h = r - b * a.q_heads;
    const int64_t want = a.lens[b];
    const int tiles = want > a.max_len || want < 0 || a.pages == 0 ? 0 : (int)((want + kKvTile - 1) / kKvTile);
    int used = (tiles + a.chunk_tiles - 1) / a.chunk_tiles;
    used = used < 1 ? 1 : used;                                      // split 0 speaks for an empty row
    const float* ml = a.part_ml + 2 * r * a.splits;
    float mm = -__builtin_inff();
    for (int s = threadIdx.x & 63; s < used; s += 64) mm = __builtin_fmaxf(mm, ml[2 * s]);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) mm = __builtin_fmaxf(mm, __shfl_xor(mm, i));
    const float base = mm == -__builtin_inff() ? 0.f : mm;
    const int c = threadIdx.x % kCols, at = threadIdx.x / kCols;
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int s = at; s < used; s += kAt) {
        const float4 o = *reinterpret_cast<const float4*>(a.part_o + (r * a.splits + s) * D + 4 * c);
        const float f = __builtin_amdgcn_exp2f(ml[2 * s] - base);
        sum = __builtin_fmaf(f, ml[2 * s + 1], sum);
        val.x = __builtin_fmaf(f, o.x, val.x);
        val.y = __builtin_fmaf(f, o.y, val.y);
        val.z = __builtin_fmaf(f, o.z, val.z);
        val.w = __builtin_fmaf(f, o.w, val.w);
    }
    *reinterpret_cast<float4*>(&part[at][4 * c]) = val;
    if (c == 0) sums[at] = sum;
    __syncthreads();
    if (threadIdx.x < D) {
        float v = 0.f, t = 0.f;
#pragma unroll
        for (int i = 0; i < kAt; ++i) {
            v += part[i][threadIdx.x];
            t += sums[i];
        }
        static_cast<typename T::Elem*>(a.out)[b * a.ld_out + h * D + threadIdx.x] = T::one(t == 0.f ? 0.f : v / t);
    }
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
        const auto run = [&](auto ng) {
            constexpr int kN = decltype(ng)::value;
            attn_decode_kernel<kT, kN><<<(unsigned)grid, 64 * kWaves, 0, stream>>>(a);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) return e;
            attn_join_kernel<kT, 32 * kN><<<(unsigned)(a.batch * a.q_heads), 256, 0, stream>>>(a);
            return hipGetLastError();
        };
        switch (a.head_dim) {
            case 64: return run(Int<2>{});
            case 128: return run(Int<4>{});
            case 256: return run(Int<8>{});
            default: return hipErrorInvalidValue;
        }
    });
}

}  // namespace frq
