// Keys and values quantised to 4 bits as they enter the paged cache, and the
// values they stand for read back (block and tile layout: frq_kv4.h).
//
// Bound by memory. d/8 lanes own one head of one token, eight channels each;
// four lanes share a block and find its largest element with two exchanges.
// Quotients are correctly rounded, so a code is the one that exact arithmetic
// gives: x / d is a quotient of a 24-bit and an 11-bit number, which never
// rounds onto a tie it is not on.
//
// A token's V codes are single bytes 8 or more apart (a byte is two channels of
// one token). A few tokens are written and read so; many, as a prompt brings
// them, 32 at a time by one workgroup per head, which, where the 32 are one
// tile, puts the tile together in LDS and moves it in 16-byte pieces.
//
// 8192 tokens of 8 heads of 128 in bf16, 43 MB each way: written in 12.7 us, 3.4
// TB/s, beside some 20 instructions an element for the block's largest, the
// quotient and the code; read in 9.7 us, 4.4 TB/s. 64 tokens in fp32: 3.2 and
// 3.4 us, the start of a kernel and three dependent accesses.
//
// Packed prompts whose 32 are seldom one tile: 24 of 17 to 1500 tokens, each from
// its page's start, 18950 together: written in 24.8 us, read in 26.1, where the
// bytes take 18.2 at copy rate; 8192 tokens from place 13 of a page 13.2 and 13.6
// (10.8 and 9.1 from its start, called again and again).
#include "frq_kernels.h"
#include "frq_kv4.h"

namespace frq {
namespace {

struct KvAt {
    uint8_t* tile;    // the tile of the token's head
    int t;            // token within the tile
};

__device__ __forceinline__ KvAt kv_at(const KvArgs& a, int64_t slot, int head, int ng) {
    const uint32_t tile = (uint32_t)(slot / kKvTile), tiles = (uint32_t)a.page_tokens / kKvTile;   // fewer than 2^32
    const uint32_t page = tile / tiles;
    uint8_t* p = static_cast<uint8_t*>(a.cache) +
                 (((int64_t)page * a.kv_heads + head) * tiles + (tile - page * tiles)) * (int64_t)kv_tile_bytes(ng);
    return {p, (int)(slot % kKvTile)};
}

// x of the lane one (0xB1) or two (0x4E) away in a quad.
template <int CTRL>
__device__ __forceinline__ float quad(float x) {
    return __builtin_bit_cast(float, __builtin_amdgcn_mov_dpp(__builtin_bit_cast(int, x), CTRL, 0xF, 0xF, true));
}
template <int CTRL>
__device__ __forceinline__ uint32_t quad(uint32_t x) {
    return (uint32_t)__builtin_amdgcn_mov_dpp((int)x, CTRL, 0xF, 0xF, true);
}

// Codes of eight channels 8 sub .. 8 sub + 7 of a block, channel i's in nibble
// i/2 + 4 (i%2), and the block's scale, from its four lanes.
__device__ __forceinline__ uint32_t quantise8(const float (&x)[8], int sub, uint32_t& scale) {
    float hi = x[0], lo = x[0], odd = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        hi = __builtin_fmaxf(hi, x[i]);
        lo = __builtin_fminf(lo, x[i]);
        odd = __builtin_fmaf(x[i], 0.f, odd);              // NaN once there is an inf or a NaN
    }
    hi = __builtin_fmaxf(hi, quad<0xB1>(hi));
    lo = __builtin_fminf(lo, quad<0xB1>(lo));
    odd += quad<0xB1>(odd);
    hi = __builtin_fmaxf(hi, quad<0x4E>(hi));
    lo = __builtin_fminf(lo, quad<0x4E>(lo));
    odd += quad<0x4E>(odd);
    const bool bad = !(odd == 0.f);
    float ext = hi >= -lo ? hi : lo;
    if (__builtin_amdgcn_ballot_w64(hi == -lo && hi > 0.f)) {
        // both signs reach the largest magnitude: the first channel's
        uint32_t first = 64;
#pragma unroll
        for (int i = 7; i >= 0; --i) first = __builtin_fabsf(x[i]) == hi ? 2 * (8 * (sub & 3) + i) + (x[i] < 0.f) : first;
        uint32_t other = quad<0xB1>(first);
        first = first < other ? first : other;
        other = quad<0x4E>(first);
        first = first < other ? first : other;
        if (hi == -lo) ext = first & 1 ? lo : hi;
    }
    const float held = __builtin_fminf(__builtin_fmaxf(ext * -0.125f, -65504.f), 65504.f);
    const uint16_t bits = f32_to_f16_bits(held);
    const float d = f16_bits_to_f32(bits), r = 1.0f / d;
    const bool none = bad || d == 0.f;
    scale = bad ? 0x7E00u : d == 0.f ? 0u : bits;
    uint32_t word = 0, over = 0;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        // x / d, correctly rounded: r is, and one correction of x r leaves the
        // nearest quotient (Markstein's theorem)
        const float q = x[i] * r, y = __builtin_fmaf(__builtin_fmaf(-q, d, x[i]), r, q);
        // 1.5 2^23 + 8 puts the code, rounded to even, into the lowest bits
        const float c = __builtin_amdgcn_fmed3f(y, -8.f, 7.f) + 12582920.f;
        const int at = 4 * (i / 2 + 4 * (i % 2));
        word += __builtin_bit_cast(uint32_t, c) << at;
        over += 0x4B400000u << at;
    }
    word -= over;
    return none ? 0x88888888u : word;
}

// Writes lane `sub`'s eight channels of token t into a tile (in memory or LDS).
template <int NG>
__device__ __forceinline__ void put(uint8_t* tile, int t, int sub, bool is_v, const float (&x)[8]) {
    uint32_t scale;
    const uint32_t c = quantise8(x, sub, scale);
    const int g = sub >> 2, j = sub & 3, u = t >> 4;
    if (j == 0)
        *reinterpret_cast<uint16_t*>(tile + (is_v ? kv_vs_off(NG) : kv_ks_off(NG)) + kv_scale(t, g, NG)) = (uint16_t)scale;
    if (!is_v) {
        *reinterpret_cast<uint32_t*>(tile + kv_word(u * NG + g, 16 * j + (t & 15))) = c;
    } else {
        // channels 8j + i of the block: n = 8 (j % 2) + i, the upper half (j >= 2) in the high nibbles
        const int tj = (t & 15) >> 2, byte = (t & 1) * 2 + ((t & 3) >> 1);
        const uint32_t up = quad<0x4E>(c);
        const uint32_t even = (c & 0x0F0F0F0Fu) | (up << 4 & 0xF0F0F0F0u);         // channels 0 4 1 5
        const uint32_t odd = (c >> 4 & 0x0F0F0F0Fu) | (up & 0xF0F0F0F0u);          // channels 2 6 3 7
        if (j < 2) {
#pragma unroll
            for (int i = 0; i < 8; ++i)
                tile[kv_vc_off(NG) + kv_word(2 * g + u, 16 * tj + 8 * j + i) + byte] =
                    (uint8_t)((i & 2 ? odd : even) >> (8 * ((i >> 2) + 2 * (i & 1))));
        }
    }
}
// Their values.
template <int NG>
__device__ __forceinline__ void get(const uint8_t* tile, int t, int sub, bool is_v, float (&x)[8]) {
    const int g = sub >> 2, j = sub & 3, u = t >> 4;
    const float d = f16_bits_to_f32(
        *reinterpret_cast<const uint16_t*>(tile + (is_v ? kv_vs_off(NG) : kv_ks_off(NG)) + kv_scale(t, g, NG)));
    if (!is_v) {
        const uint32_t w = *reinterpret_cast<const uint32_t*>(tile + kv_word(u * NG + g, 16 * j + (t & 15)));
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = d * ((float)((w >> (4 * (i / 2 + 4 * (i % 2)))) & 15u) - 8.f);
    } else {
        const int tj = (t & 15) >> 2, byte = (t & 1) * 2 + ((t & 3) >> 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t b = tile[kv_vc_off(NG) + kv_word(2 * g + u, 16 * tj + 8 * (j & 1) + i) + byte];
            x[i] = d * ((float)(j >= 2 ? b >> 4 : b & 15u) - 8.f);
        }
    }
}

// One head of one token to d/8 lanes.
template <int TYPE, int NG, bool WRITE>
__global__ void __launch_bounds__(256) kv_token_kernel(KvArgs a) {
    using T = Val<TYPE>;
    constexpr int kLanes = 4 * NG;
    const int sub = threadIdx.x & (kLanes - 1);
    const uint32_t heads = (uint32_t)a.kv_heads;
    const uint32_t unit = blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const uint32_t tok = unit / (2 * heads), r = unit - tok * 2 * heads;
    if (tok >= a.tokens) return;
    const bool is_v = r >= heads;
    const uint32_t h = is_v ? r - heads : r;
    const int64_t slot = a.slots[tok];
    typename T::Elem* row = static_cast<typename T::Elem*>(is_v ? a.v : a.k) + tok * (is_v ? a.ld_v : a.ld_k) +
                            (int64_t)h * NG * 32 + sub * 8;
    const bool there = slot >= 0 && slot < a.pages * a.page_tokens;
    float x[8];
    if constexpr (WRITE) {
        if (!there) return;
        T::load8(row, x);
        const KvAt at = kv_at(a, slot, (int)h, NG);
        put<NG>(at.tile, at.t, sub, is_v, x);
    } else {
        if (there) {
            const KvAt at = kv_at(a, slot, (int)h, NG);
            get<NG>(at.tile, at.t, sub, is_v, x);
        } else {
            const float fill = slot < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = fill;
        }
        T::store8(row, x);
    }
}

// One head of 32 tokens of the call to a workgroup.
template <int TYPE, int NG, bool WRITE>
__global__ void __launch_bounds__(256) kv_tile_kernel(KvArgs a) {
    using T = Val<TYPE>;
    constexpr int kLanes = 4 * NG, kPer = 256 / kLanes;              // tokens of K, or of V, at a time
    __shared__ __attribute__((aligned(16))) uint8_t image[kv_tile_bytes(NG)];
    const uint32_t heads = (uint32_t)a.kv_heads, chunk = blockIdx.x / heads;
    const int h = (int)(blockIdx.x - chunk * heads), sub = threadIdx.x & (kLanes - 1);
    const int64_t first = (int64_t)chunk * kKvTile, slots = a.pages * a.page_tokens;
    const int count = a.tokens - first < kKvTile ? (int)(a.tokens - first) : kKvTile;
    const int lane = threadIdx.x & 63, mine = lane & 31;
    // is it one tile, in its order?
    const int64_t s0 = a.slots[first], own = mine < count ? a.slots[first + mine] : -1;
    const bool whole = s0 >= 0 && s0 + kKvTile <= slots && s0 % kKvTile == 0 &&
                       __builtin_amdgcn_ballot_w64(own != s0 + mine) == 0;
    uint4* tile = whole ? reinterpret_cast<uint4*>(kv_at(a, s0, h, NG).tile) : nullptr;
    const int64_t at0 = (int64_t)h * NG * 32 + sub * 8;
    typename T::Elem* rows[2] = {static_cast<typename T::Elem*>(a.k) + at0, static_cast<typename T::Elem*>(a.v) + at0};
    const int64_t ld[2] = {a.ld_k, a.ld_v};
    const int t0 = (int)threadIdx.x / kLanes;
    if (whole) {
        if constexpr (WRITE) {
            float x[2][kKvTile / kPer][8];                           // all loads under way before the first is waited for
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                for (int i = 0; i < kKvTile / kPer; ++i) T::load8(rows[kv] + (first + t0 + i * kPer) * ld[kv], x[kv][i]);
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                for (int i = 0; i < kKvTile / kPer; ++i) put<NG>(image, t0 + i * kPer, sub, kv == 1, x[kv][i]);
            __syncthreads();
            for (int i = threadIdx.x; i < kv_tile_bytes(NG) / 16; i += 256) tile[i] = reinterpret_cast<const uint4*>(image)[i];
        } else {
            for (int i = threadIdx.x; i < kv_tile_bytes(NG) / 16; i += 256) reinterpret_cast<uint4*>(image)[i] = tile[i];
            __syncthreads();
#pragma unroll
            for (int kv = 0; kv < 2; ++kv)
#pragma unroll
                for (int i = 0; i < kKvTile / kPer; ++i) {
                    float x[8];
                    get<NG>(image, t0 + i * kPer, sub, kv == 1, x);
                    T::store8(rows[kv] + (first + t0 + i * kPer) * ld[kv], x);
                }
        }
        return;
    }
    for (int t = t0; t < count; t += kPer) {
        const int64_t slot = a.slots[first + t];
        const bool there = slot >= 0 && slot < slots;
        const KvAt place = kv_at(a, there ? slot : 0, h, NG);
#pragma unroll
        for (int kv = 0; kv < 2; ++kv) {
            typename T::Elem* row = rows[kv] + (first + t) * ld[kv];
            float x[8];
            if constexpr (WRITE) {
                if (!there) continue;
                T::load8(row, x);
                put<NG>(place.tile, place.t, sub, kv == 1, x);
            } else {
                if (there) {
                    get<NG>(place.tile, place.t, sub, kv == 1, x);
                } else {
                    const float fill = slot < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
                    for (int i = 0; i < 8; ++i) x[i] = fill;
                }
                T::store8(row, x);
            }
        }
    }
}

template <typename F>
hipError_t with_groups(int64_t head_dim, F&& f) {
    switch (head_dim) {
        case 64: return f(Int<2>{});
        case 128: return f(Int<4>{});
        case 256: return f(Int<8>{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

namespace {

constexpr int64_t kTileTokens = 256;       // from here on 32 tokens to a workgroup

template <bool WRITE>
hipError_t launch_kv(const KvArgs& a, hipStream_t stream) {
    return with_type(a.type, [&](auto ty) {
        return with_groups(a.head_dim, [&](auto ng) {
            constexpr int kT = decltype(ty)::value, kN = decltype(ng)::value, kUnits = 256 / (4 * kN);
            if (a.tokens >= kTileTokens) {
                const int64_t grid = (a.tokens + kKvTile - 1) / kKvTile * a.kv_heads;
                kv_tile_kernel<kT, kN, WRITE><<<(unsigned)grid, 256, 0, stream>>>(a);
            } else {
                const int64_t grid = (a.tokens * a.kv_heads * 2 + kUnits - 1) / kUnits;
                kv_token_kernel<kT, kN, WRITE><<<(unsigned)grid, 256, 0, stream>>>(a);
            }
            return hipGetLastError();
        });
    });
}

}  // namespace

hipError_t launch_kv_write(const KvArgs& a, hipStream_t stream) { return launch_kv<true>(a, stream); }
hipError_t launch_kv_read(const KvArgs& a, hipStream_t stream) { return launch_kv<false>(a, stream); }

}  // namespace frq
