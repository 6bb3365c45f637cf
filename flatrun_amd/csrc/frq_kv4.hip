// Keys and values quantised to 4 bits as they enter the paged cache, and the
// values they stand for read back (block and tile layout: frq_kv4.h).
//
// Bound by memory. d/8 lanes own one head of one token, eight channels each;
// four lanes share a block and find its largest element with two exchanges.
// The scale's division and every code's are IEEE divisions, so a code is the
// one that exact arithmetic gives: x / d is a quotient of a 24-bit and an
// 11-bit number, which never rounds onto a tie it is not on.
#include "frq_kernels.h"
#include "frq_kv4.h"

namespace frq {
namespace {

struct KvAt {
    uint8_t* tile;    // the tile of the token's head
    int t;            // token within the tile
};

__device__ __forceinline__ KvAt kv_at(const KvArgs& a, int64_t slot, int head, int ng) {
    const int64_t page = slot / a.page_tokens, in = slot - page * a.page_tokens;
    const int64_t tiles = a.page_tokens / kKvTile;
    uint8_t* p = static_cast<uint8_t*>(a.cache) +
                 ((page * a.kv_heads + head) * tiles + in / kKvTile) * (int64_t)kv_tile_bytes(ng);
    return {p, (int)(in % kKvTile)};
}

// Codes of eight channels 8 sub .. 8 sub + 7 of a block, and its scale, from
// the four lanes of the block.
__device__ __forceinline__ void quantise8(const float (&x)[8], int sub, uint32_t (&code)[8], uint32_t& scale) {
    float top = -1.f, ext = 0.f;
    bool bad = false;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float m = __builtin_fabsf(x[i]);
        bad |= !(m < __builtin_inff());
        if (m > top) {
            top = m;
            ext = x[i];
        }
    }
#pragma unroll
    for (int m = 1; m <= 2; m <<= 1) {
        const float ot = __shfl_xor(top, m), oe = __shfl_xor(ext, m);
        const bool lower = (sub & m) != 0;             // the other lane's channels come first
        if (lower ? ot >= top : ot > top) {
            top = ot;
            ext = oe;
        }
        bad |= __shfl_xor((int)bad, m) != 0;
    }
    const float want = ext * -0.125f;
    const float held = __builtin_fminf(__builtin_fmaxf(want, -65504.f), 65504.f);
    const uint16_t bits = f32_to_f16_bits(held);
    const float d = f16_bits_to_f32(bits);
    scale = bad ? 0x7E00u : d == 0.f ? 0u : bits;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float c = __builtin_fminf(__builtin_fmaxf(rintf(x[i] / d) + 8.f, 0.f), 15.f);
        code[i] = bad || d == 0.f ? 8u : (uint32_t)c;
    }
}

template <int TYPE, int NG>
__global__ void __launch_bounds__(256) kv_write_kernel(KvArgs a) {
    using T = Val<TYPE>;
    constexpr int kLanes = 4 * NG;
    const int sub = threadIdx.x & (kLanes - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const int heads = (int)a.kv_heads;
    if (unit >= a.tokens * heads * 2) return;
    const int64_t tok = unit / (2 * heads);
    const int r = (int)(unit - tok * 2 * heads);
    const bool is_v = r >= heads;
    const int h = is_v ? r - heads : r;
    const int64_t slot = a.slots[tok];
    if (slot < 0 || slot >= a.pages * a.page_tokens) return;
    float x[8];
    T::load8(static_cast<const typename T::Elem*>(is_v ? a.v : a.k) + tok * (is_v ? a.ld_v : a.ld_k) +
                 (int64_t)h * NG * 32 + sub * 8, x);
    uint32_t c[8], scale;
    quantise8(x, sub, c, scale);
    const KvAt at = kv_at(a, slot, h, NG);
    const int g = sub >> 2, j = sub & 3;
    if ((sub & 3) == 0)
        *reinterpret_cast<uint16_t*>(at.tile + (is_v ? kv_vs_off(NG) : kv_ks_off(NG)) + kv_scale(at.t, g, NG)) =
            (uint16_t)scale;
    if (!is_v) {
        uint32_t w = 0;
#pragma unroll
        for (int i = 0; i < 8; ++i) w |= c[i] << (4 * (i / 2 + 4 * (i % 2)));
        const int u = at.t >> 4, lane = 16 * j + (at.t & 15);
        *reinterpret_cast<uint32_t*>(at.tile + kv_word(u * NG + g, lane)) = w;
    } else {
        // channels 8j + i of the block: n = 8 (j % 2) + i, the upper half (j >= 2) in the high nibbles
        const int u = at.t >> 4, tj = (at.t & 15) >> 2, i4 = at.t & 3;
        const int byte = (i4 & 1) * 2 + (i4 >> 1);
#pragma unroll
        for (int i = 0; i < 8; ++i) {
            const uint32_t up = __shfl_down(c[i], 2);
            if (j < 2) {
                const int n = 8 * j + i;
                at.tile[kv_vc_off(NG) + kv_word(2 * g + u, 16 * tj + n) + byte] = (uint8_t)(c[i] | (up << 4));
            }
        }
    }
}

template <int TYPE, int NG>
__global__ void __launch_bounds__(256) kv_read_kernel(KvArgs a) {
    using T = Val<TYPE>;
    constexpr int kLanes = 4 * NG;
    const int sub = threadIdx.x & (kLanes - 1);
    const int64_t unit = (int64_t)blockIdx.x * (256 / kLanes) + threadIdx.x / kLanes;
    const int heads = (int)a.kv_heads;
    if (unit >= a.tokens * heads * 2) return;
    const int64_t tok = unit / (2 * heads);
    const int r = (int)(unit - tok * 2 * heads);
    const bool is_v = r >= heads;
    const int h = is_v ? r - heads : r;
    const int64_t slot = a.slots[tok];
    float x[8];
    if (slot < 0 || slot >= a.pages * a.page_tokens) {
        const float fill = slot < 0 ? 0.f : __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 8; ++i) x[i] = fill;
    } else {
        const KvAt at = kv_at(a, slot, h, NG);
        const int g = sub >> 2, j = sub & 3, u = at.t >> 4;
        const float d = f16_bits_to_f32(*reinterpret_cast<const uint16_t*>(
            at.tile + (is_v ? kv_vs_off(NG) : kv_ks_off(NG)) + kv_scale(at.t, g, NG)));
        if (!is_v) {
            const uint32_t w = *reinterpret_cast<const uint32_t*>(at.tile + kv_word(u * NG + g, 16 * j + (at.t & 15)));
#pragma unroll
            for (int i = 0; i < 8; ++i) x[i] = d * ((float)((w >> (4 * (i / 2 + 4 * (i % 2)))) & 15u) - 8.f);
        } else {
            const int tj = (at.t & 15) >> 2, i4 = at.t & 3, byte = (i4 & 1) * 2 + (i4 >> 1);
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t b = at.tile[kv_vc_off(NG) + kv_word(2 * g + u, 16 * tj + 8 * (j & 1) + i) + byte];
                x[i] = d * ((float)(j >= 2 ? b >> 4 : b & 15u) - 8.f);
            }
        }
    }
    T::store8(static_cast<typename T::Elem*>(is_v ? a.v : a.k) + tok * (is_v ? a.ld_v : a.ld_k) +
                  (int64_t)h * NG * 32 + sub * 8, x);
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

hipError_t launch_kv_write(const KvArgs& a, hipStream_t stream) {
    return with_type(a.type, [&](auto ty) {
        return with_groups(a.head_dim, [&](auto ng) {
            constexpr int kUnits = 256 / (4 * decltype(ng)::value);
            const int64_t grid = (a.tokens * a.kv_heads * 2 + kUnits - 1) / kUnits;
            kv_write_kernel<decltype(ty)::value, decltype(ng)::value><<<(unsigned)grid, 256, 0, stream>>>(a);
            return hipGetLastError();
        });
    });
}

hipError_t launch_kv_read(const KvArgs& a, hipStream_t stream) {
    return with_type(a.type, [&](auto ty) {
        return with_groups(a.head_dim, [&](auto ng) {
            constexpr int kUnits = 256 / (4 * decltype(ng)::value);
            const int64_t grid = (a.tokens * a.kv_heads * 2 + kUnits - 1) / kUnits;
            kv_read_kernel<decltype(ty)::value, decltype(ng)::value><<<(unsigned)grid, 256, 0, stream>>>(a);
            return hipGetLastError();
        });
    });
}

}  // namespace frq
