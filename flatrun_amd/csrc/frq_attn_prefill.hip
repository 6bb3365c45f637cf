// Attention over packed sequences of different lengths:
//   S[i, j] = scale q_i . k_j,  out_i = sum_j softmax(S)[i, j] v_j
// for the queries and keys of each sequence, j <= i + (keys - queries) where
// causal, query heads grouped over key heads. A query that no key is left for
// gives zeros.
//
// Bound by the matrix cores on long prompts: v_mfma_f32_32x32x16 in bf16 or
// fp16 with fp32 sums; scores, running maximum and sum in fp32; the softmax
// weights are rounded to the inputs' type for the second product, as their
// values are, and summed as they are rounded. In bf16 the error against 64 bits,
// of the output's norm, is 0.0019 (333 tokens), 0.0022 (24 packed sequences) and
// 0.0021 (16384 tokens), where the output's own rounding leaves 0.0016; weights
// in two parts would take half as many products again.
//
// A wave takes 32 queries of one head; the waves of a workgroup (4 or 8) the
// heads that share a key head, then the next 32 queries, so that short
// sequences waste little and one copy of a key tile serves all. Where there are
// few queries two waves share them, each with every other tile, and join at the
// end. Keys are walked 64 (then 128) at a time through LDS, the next copy in
// flight. The products are
// S^T = K Q^T and O^T = V^T P^T: a lane then holds one query's scores in both,
// the maximum and sum need one exchange between the wave's halves, and P^T is
// in the registers the second product reads, with the keys in the order in
// which S^T left them; V^T comes from the row-major tile by transposing LDS
// reads.
//
// 16384 tokens of 32 heads of 128 over 8, causal, bf16: 1.9 to 2.0 ms, 1.1 to
// 1.16 PFLOP/s, where a large plain product reaches 1.35: the matrix cores are
// busy 58 % of the time and vector instructions 38 %, at the 1.86 GHz that the
// power leaves; the LDS 29 %, without conflicts. 24 sequences of 17 to 1500
// tokens after up to 1200: 444 us, 845 TFLOP/s, matrix cores 41 %, 2.07 GHz: a
// workgroup's start and end, its two tiles cut by the mask and what its 18 tiles
// round up to. Workgroups that stay and take the next block of queries from a
// queue, its tile loaded ahead, gave 435 there, nothing on the long prompt and
// 13.7 against 12.7 us on a short one.
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

using bf16x8 = __bf16 __attribute__((ext_vector_type(8)));
using f16x8 = _Float16 __attribute__((ext_vector_type(8)));
using bf16x2 = __bf16 __attribute__((ext_vector_type(2)));
using f16x2 = _Float16 __attribute__((ext_vector_type(2)));
using s16x4 = short __attribute__((ext_vector_type(4)));
using u32x4 = uint32_t __attribute__((ext_vector_type(4)));
using u32x2 = uint32_t __attribute__((ext_vector_type(2)));
using f32x16 = float __attribute__((ext_vector_type(16)));

constexpr int kKeys = 64;             // keys of a step

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
    if constexpr (TYPE == kTypeBF16) {
        const bf16x2 v = {(__bf16)a, (__bf16)b};
        return __builtin_bit_cast(uint32_t, v);
    } else {
        const f16x2 v = {(_Float16)a, (_Float16)b};
        return __builtin_bit_cast(uint32_t, v);
    }
}

// The larger of a lane's value and that of the lane 32 away.
__device__ __forceinline__ float half_max(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x);
    const auto r = __builtin_amdgcn_permlane32_swap(b, b, false, false);
    const uint32_t low = r[0], high = r[1];
    return __builtin_fmaxf(__builtin_bit_cast(float, low), __builtin_bit_cast(float, high));
}

// acc + both halves of a pair of weights, as they are rounded.
template <int TYPE>
__device__ __forceinline__ float add_pair(uint32_t w, float acc) {
    if constexpr (TYPE == kTypeBF16) {
        return __builtin_amdgcn_fdot2_f32_bf16(__builtin_bit_cast(bf16x2, w), (bf16x2){(__bf16)1.f, (__bf16)1.f}, acc, false);
    } else {
        return __builtin_amdgcn_fdot2(__builtin_bit_cast(f16x2, w), (f16x2){(_Float16)1.f, (_Float16)1.f}, acc, false);
    }
}

// The halves of w that are an inf or a NaN, as a mask of ones.
template <int TYPE>
__device__ __forceinline__ uint32_t specials(uint32_t w) {
    constexpr uint32_t e = TYPE == kTypeBF16 ? 0x7F80u : 0x7C00u;
    return ((w & e) == e ? 0xFFFFu : 0u) | (((w >> 16) & e) == e ? 0xFFFF0000u : 0u);
}

template <int TYPE>
__device__ __forceinline__ float widen(uint16_t b) {
    if constexpr (TYPE == kTypeBF16) return __builtin_bit_cast(float, (uint32_t)b << 16);
    return f16_bits_to_f32(b);
}

// Where 16-byte piece p of row r lies in a tile of rows of CH pieces. A wave
// reads K as 16 rows of one piece at a time and V as 4 rows of 4 pieces; with
// the row's low bits on the piece's high ones both touch every bank once.
template <int CH>
__device__ __forceinline__ int swizzle(int r) {
    if constexpr (CH == 8) return (((r >> 1) & 1) << 2) | ((r >> 2) & 3);
    return ((r & 3) << 2) | ((r >> 2) & 3);
}

// Four keys of one column: the 16 lanes of a block point at the 16 groups of
// four columns of four rows (lane 4r + c: row r, columns 4c .. 4c + 3), lane i
// gets column i.
using lds_bytes = __attribute__((address_space(3))) const char*;
__device__ __forceinline__ uint2 read_column4(lds_bytes p) {
    const s16x4 v = __builtin_amdgcn_ds_read_tr16_b64_v4i16((__attribute__((address_space(3))) s16x4*)p);
    return __builtin_bit_cast(uint2, v);
}
__device__ __forceinline__ uint4 read_row8(lds_bytes p) {
    const u32x4 v = *(__attribute__((address_space(3))) const u32x4*)p;
    return make_uint4(v[0], v[1], v[2], v[3]);
}

// Asynchronous copy of a tile of kKeys rows (`rows` of them present, the others
// become zeros) to LDS, 16 bytes a lane and step, swizzled on the way. The host
// keeps a tile's bytes, kKeys rows of ld, below 2^31.
template <int D, int WAVES>
__device__ __forceinline__ void stage(const uint16_t* src, int64_t ld, int rows, uint16_t* tile) {
    constexpr int CH = D / 8, kSteps = kKeys * CH / (64 * WAVES);
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const uint32_t bytes = rows > 0 ? (uint32_t)(((int64_t)(rows - 1) * ld + D) * 2) : 0u;
    const __amdgpu_buffer_rsrc_t r = buffer_rsrc(src, bytes);
#pragma unroll
    for (int i = 0; i < kSteps; ++i) {
        const int first = (i * WAVES + wave) * 64;
        const int at = first + lane, row = at / CH, piece = (at % CH) ^ swizzle<CH>(row);
        __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(tile + first * 8), 16,
                                                 (int)(row * (uint32_t)(ld * 2) + piece * 16), 0, 0, 0);
    }
}

// Waves to a SIMD: 64-wide heads in workgroups of eight fit two of those on a CU
// with 128 registers a lane, which the compiler passes if it is not told.
template <int TYPE, int OUT, int D, int WAVES, int SPLIT>
__global__ void __launch_bounds__(64 * WAVES, D == 256 ? 1 : D == 64 && WAVES == 8 ? 4 : 2) attn_prefill_kernel(PrefillArgs a) {
    constexpr int kUnits = WAVES / SPLIT;                        // of 32 queries of a head
    // Operands read four products ahead of their use in the order of the source:
    // heads of 256, which the compiler's order serves one by one (4096 tokens, 8
    // heads: 141 us against 183), and whole tiles of 64 (14 heads, 8192 tokens: 152
    // against 165; 24 packed sequences: 125 against 120). For the others its own
    // order is as good or 2 to 3 % better.
    constexpr bool kAhead = D == 256 || (D == 64 && SPLIT == 1);
    constexpr int NK = D / 16, ND = D / 32, CH = D / 8;          // k-steps, column tiles, 16-byte pieces of a row
    // Two buffers of a K and a V tile, used in turn. Objects of their own and a
    // step's code for each, so that the compiler sees that a read of one need
    // not wait for the copies into the other.
    constexpr int kTile = kKeys * D;
    __shared__ int special_at;
    __shared__ __attribute__((aligned(16))) uint16_t lk0[SPLIT * kTile], lv0[SPLIT * kTile];
    __shared__ __attribute__((aligned(16))) uint16_t lk1[SPLIT * kTile], lv1[SPLIT * kTile];
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ln = lane & 31, h = lane >> 5;
    // neighbouring workgroups go to different XCDs: give each its own key head
    uint32_t id = blockIdx.x;
    const int kvh = (int)(id % (uint32_t)a.kv_heads);
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    id /= (uint32_t)a.kv_heads;
    const uint32_t most = (uint32_t)a.blocks, seqs = (uint32_t)a.seqs;
    const int seq = (int)(a.together ? id % seqs : id / most);
    const int block = (int)(most - 1 - (a.together ? id / seqs : id % most));    // the longest rows first
    const int64_t q0 = a.cu_q[seq], k0 = a.cu_k[seq];
    const int64_t nq = a.cu_q[seq + 1] - q0, nk = a.cu_k[seq + 1] - k0;
    const int first = (int)((uint32_t)(block * kUnits) / (uint32_t)group) * 32;   // the workgroup's first query
    if (q0 < 0 || k0 < 0 || nk < 0 || q0 + nq > a.tokens_q || k0 + nk > a.tokens_k) return;
    if (nq > a.max_q) {                                          // more queries than the grid is made for: NaN
        using O = Val<OUT>;
        for (int64_t i = block; i < nq; i += most) {
            typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (q0 + i) * a.ld_out + (int64_t)kvh * group * a.hs_out;
            for (int e = threadIdx.x; e < group * D; e += 64 * WAVES) out[e / D * a.hs_out + e % D] = O::one(__builtin_nanf(""));
        }
        return;
    }
    if (first >= nq) return;
    const int past = (int)(nk - nq);
    // a wave's 32 queries of one head: the heads that share the key head side by side
    const int part = SPLIT > 1 ? wave / kUnits : 0;              // which of SPLIT tiles at a time is the wave's
    const uint32_t unit = (uint32_t)(block * kUnits + (SPLIT > 1 ? wave % kUnits : wave));
    const int i0 = (int)(unit / (uint32_t)group) * 32;           // the wave's first query
    const int head = kvh * group + (int)(unit % (uint32_t)group);
    const int qi = i0 + ln;                                      // the lane's
    int end = (int)nk;                                           // keys that the workgroup needs
    if (a.causal) {
        const int64_t e = (int64_t)((uint32_t)(block * kUnits + kUnits - 1) / (uint32_t)group) * 32 + 32 + past;
        end = (int)(e < nk ? e : nk);
    }
    const uint16_t* q = static_cast<const uint16_t*>(a.q) + (q0 + (qi < nq ? qi : nq - 1)) * a.ld_q + head * a.hs_q;
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
    float m = -__builtin_inff(), nref = 0.f, l = 0.f;            // reference, minus it (0 while there is none), sum
    const float c = a.scale * 1.4426950408889634f;
    const int lim = a.causal && qi + past < nk - 1 ? qi + past : (int)nk - 1;    // the lane's last key

    // The lane's places in a tile. K: row ln, piece h; the other pieces are an
    // exclusive-or away, the other rows a constant. V: keys 4h + (lane % 16) / 4
    // and 8 further, columns 4 (lane % 4) and 16 for odd blocks of lanes.
    const int r4 = (lane & 15) >> 2, x4 = ((lane >> 4) & 1) * 2 + ((lane & 3) >> 1);
    const int kat = ln * D * 2 + 16 * (h ^ swizzle<CH>(ln));
    const int vat0 = (4 * h + r4) * D * 2 + 16 * (x4 ^ swizzle<CH>(4 * h + r4)) + 8 * (lane & 1);
    const int vat1 = (4 * h + r4 + 8) * D * 2 + 16 * (x4 ^ swizzle<CH>(4 * h + r4 + 8)) + 8 * (lane & 1);

    if (threadIdx.x == 0) special_at = 0;
    auto stage_all = [&](int kt, uint16_t* tk, uint16_t* tv) __attribute__((always_inline)) {
#pragma unroll
        for (int x = 0; x < SPLIT; ++x) {
            const int left = (int)nk - kt - x * kKeys, rows = left < kKeys ? left : kKeys;
            stage<D, WAVES>(kp + (int64_t)(kt + x * kKeys) * a.ld_k, a.ld_k, rows, tk + x * kTile);
            stage<D, WAVES>(vp + (int64_t)(kt + x * kKeys) * a.ld_v, a.ld_v, rows, tv + x * kTile);
        }
    };
    constexpr int kStep = SPLIT * kKeys;
    if (end > 0) stage_all(0, lk0, lv0);
    auto step = [&](int at, uint16_t* ck, uint16_t* cv, uint16_t* tk, uint16_t* tv) __attribute__((always_inline)) {
        // this tile is there, and everyone is done with the other buffer
        __builtin_amdgcn_s_waitcnt(0x0070);                      // vmcnt(0), lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
        const lds_bytes sk = (lds_bytes)ck + part * (2 * kTile), sv = (lds_bytes)cv + part * (2 * kTile);
        if (at + kStep < end) stage_all(at + kStep, tk, tv);
        // A zero weight does not take an inf or a NaN out of a product: where
        // the mask cuts through the tile, such values leave it and are added
        // below for the queries that see their keys.
        const bool cut = a.causal && at + kStep - 1 > first + past;
        if (__builtin_expect(cut, 0)) {
            bool any = false;
            for (int i = threadIdx.x; i < kStep * CH; i += 64 * WAVES) {
                u32x4 w = reinterpret_cast<const u32x4*>(cv)[i];
                const u32x4 s = {specials<TYPE>(w[0]), specials<TYPE>(w[1]), specials<TYPE>(w[2]), specials<TYPE>(w[3])};
                if (s[0] | s[1] | s[2] | s[3]) {
                    any = true;
                    reinterpret_cast<u32x4*>(cv)[i] = w & ~s;
                }
            }
            if (any) special_at = at + 1;
            __builtin_amdgcn_s_waitcnt(0xC07F);                  // lgkmcnt(0)
            __builtin_amdgcn_s_barrier();
        }
        const int kt = at + part * kKeys;
        if (i0 >= nq || (SPLIT > 1 && kt >= nk) || (a.causal && kt > i0 + 31 + past)) return;   // nothing here for the wave
        const bool masked = kt + kKeys > nk || (a.causal && kt + kKeys - 1 > i0 + past);
        __builtin_amdgcn_s_setprio(1);                           // a wave at its products goes first
        f32x16 st[2];
#pragma unroll
        for (int i = 0; i < 16; ++i) st[0][i] = st[1][i] = 0.f;
        if constexpr (kAhead) {
            auto row = [&](int x) { return read_row8(sk + (kat ^ (32 * (x >> 1))) + 32 * (x & 1) * D * 2); };
            uint4 ahead[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) ahead[x] = row(x);
#pragma unroll
            for (int x = 0; x < 2 * NK; ++x) {
                st[x & 1] = mfma<TYPE>(ahead[x & 3], qf[x >> 1], st[x & 1]);
                if (x + 4 < 2 * NK) ahead[x & 3] = row(x + 4);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < NK; ++s)
#pragma unroll
                for (int t = 0; t < 2; ++t)
                    st[t] = mfma<TYPE>(read_row8(sk + (kat ^ (32 * s)) + 32 * t * D * 2), qf[s], st[t]);
            // four reads ahead of the products
            __builtin_amdgcn_sched_group_barrier(0x100, 4, 0);
#pragma unroll
            for (int s = 0; s < 2 * NK - 4; ++s) {
                __builtin_amdgcn_sched_group_barrier(0x008, 1, 0);
                __builtin_amdgcn_sched_group_barrier(0x100, 1, 0);
            }
            __builtin_amdgcn_sched_group_barrier(0x008, 4, 0);
        }
        __builtin_amdgcn_s_setprio(0);
        if (__builtin_expect(masked, 0)) {
            const int left = lim - kt - 4 * h;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * t + 8 * (i >> 2) + (i & 3) > left) st[t][i] = -__builtin_inff();
        }
        float top = st[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, st[t][i]);
        top = half_max(top) * c;
        // the reference follows the maximum only when it is 2^8 behind: sums
        // and weights have the room, and the rescaling is rare
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + 8.f) != 0, 0)) {
            const float mn = __builtin_fmaxf(m, top);
            const float keep = mn == -__builtin_inff() ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            nref = mn == -__builtin_inff() ? 0.f : -mn;
            l *= keep;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= keep;
        }
        uint4 pf[4];
#pragma unroll
        for (int s = 0; s < 4; ++s) {
            float p[8];
#pragma unroll
            for (int e = 0; e < 8; ++e)
                p[e] = __builtin_amdgcn_exp2f(__builtin_fmaf(st[s >> 1][8 * (s & 1) + e], c, nref));
            pf[s] = make_uint4(pack2<TYPE>(p[0], p[1]), pack2<TYPE>(p[2], p[3]), pack2<TYPE>(p[4], p[5]),
                               pack2<TYPE>(p[6], p[7]));
            l = add_pair<TYPE>(pf[s].x, l);
            l = add_pair<TYPE>(pf[s].y, l);
            l = add_pair<TYPE>(pf[s].z, l);
            l = add_pair<TYPE>(pf[s].w, l);
        }
        if constexpr (kAhead) {
            auto columns = [&](int x) {
                const int at = 16 * (x / ND) * D * 2, d = 64 * (x % ND);
                const uint2 lo = read_column4(sv + (vat0 ^ d) + at), hi = read_column4(sv + (vat1 ^ d) + at);
                return make_uint4(lo.x, lo.y, hi.x, hi.y);
            };
            uint4 ahead[4];
#pragma unroll
            for (int x = 0; x < 4; ++x) ahead[x] = columns(x);
#pragma unroll
            for (int x = 0; x < 4 * ND; ++x) {
                o[x % ND] = mfma<TYPE>(ahead[x & 3], pf[x / ND], o[x % ND]);
                if (x + 4 < 4 * ND) ahead[x & 3] = columns(x + 4);
                __builtin_amdgcn_sched_barrier(0);
            }
        } else {
#pragma unroll
            for (int s = 0; s < 4; ++s) {
#pragma unroll
                for (int d = 0; d < ND; ++d) {
                    const uint2 lo = read_column4(sv + (vat0 ^ (64 * d)) + 16 * s * D * 2);
                    const uint2 hi = read_column4(sv + (vat1 ^ (64 * d)) + 16 * s * D * 2);
                    o[d] = mfma<TYPE>(make_uint4(lo.x, lo.y, hi.x, hi.y), pf[s], o[d]);
                }
            }
        }
        if (__builtin_expect(cut && special_at == at + 1, 0)) {
            for (int kr = 0; kr < kKeys && kt + kr < nk; ++kr) {
                const uint16_t* row = vp + (int64_t)(kt + kr) * a.ld_v + 4 * h;
                const bool seen = kt + kr <= lim;
#pragma unroll
                for (int d = 0; d < ND; ++d)
#pragma unroll
                    for (int i = 0; i < 16; i += 4) {
                        const u32x2 w = *reinterpret_cast<const u32x2*>(row + 32 * d + 2 * i);
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const uint32_t b = w[e >> 1] >> (16 * (e & 1)) & 0xFFFFu;
                            if (seen && (specials<TYPE>(b) & 0xFFFFu)) o[d][i + e] += widen<TYPE>((uint16_t)b);
                        }
                        __builtin_amdgcn_sched_barrier(0);
                    }
            }
        }
    };
    for (int at = 0; at < end; at += 2 * kStep) {
        step(at, lk0, lv0, lk1, lv1);
        if (at + kStep < end) step(at + kStep, lk1, lv1, lk0, lv0);
    }
    l += __shfl_xor(l, 32);
    if constexpr (SPLIT == 2) {
        // the second half's sums to the first, in the place of the tiles
        __shared__ float sh_m[kUnits][32], sh_l[kUnits][32];
        const int u = wave % kUnits;
        float4* held = reinterpret_cast<float4*>((u < 2 ? lk0 : lv0) + (u & 1) * kTile) + lane;
        __syncthreads();
        if (part == 1) {
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; i += 4)
                    held[16 * (16 * d + i)] = make_float4(o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]);
            if (h == 0) {
                sh_m[u][ln] = m;
                sh_l[u][ln] = l;
            }
        }
        __syncthreads();
        if (part == 1) return;
        const float m1 = sh_m[u][ln], both = __builtin_fmaxf(m, m1), base = both == -__builtin_inff() ? 0.f : both;
        const float f0 = __builtin_amdgcn_exp2f(m - base), f1 = __builtin_amdgcn_exp2f(m1 - base);
        l = l * f0 + sh_l[u][ln] * f1;
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4) {
                const float4 x = held[16 * (16 * d + i)];
                o[d][i] = o[d][i] * f0 + x.x * f1;
                o[d][i + 1] = o[d][i + 1] * f0 + x.y * f1;
                o[d][i + 2] = o[d][i + 2] * f0 + x.z * f1;
                o[d][i + 3] = o[d][i + 3] * f0 + x.w * f1;
            }
    }
    if (qi >= nq) return;
    // No weight at all: zeros for a query without keys; where its keys all score
    // -inf the softmax is 0 / 0.
    const float inv = 1.0f / l, none = lim < 0 ? 0.f : __builtin_nanf("");
    using O = Val<OUT>;
    typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (q0 + qi) * a.ld_out + head * a.hs_out;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {                        // columns 32 d + 2 i + 4 h and the next three
            float x[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) x[e] = l == 0.f ? none : o[d][i + e] * inv;
            if constexpr (OUT == kTypeF32)
                *reinterpret_cast<float4*>(out + 32 * d + 2 * i + 4 * h) = make_float4(x[0], x[1], x[2], x[3]);
            else
                *reinterpret_cast<uint2*>(out + 32 * d + 2 * i + 4 * h) =
                    make_uint2(pack2<OUT>(x[0], x[1]), pack2<OUT>(x[2], x[3]));
        }
}

template <int TYPE, int OUT, int D, int WAVES, int SPLIT>
hipError_t launch_one(PrefillArgs a, hipStream_t stream) {
    constexpr int kUnits = WAVES / SPLIT;
    a.blocks = ((a.max_q + 31) / 32 * (a.q_heads / a.kv_heads) + kUnits - 1) / kUnits;
    const int64_t grid = a.blocks * a.seqs * a.kv_heads;
    // Workgroups that all run at once go from the longest rows of any sequence to
    // the shortest (16 sequences of 512, 14 heads of 64: 20 us against 24); more
    // of them sequence by sequence, whose keys then stay in the L2 caches (24 of
    // 17 to 1500 tokens after up to 1200, 32 heads of 128: 521 us against 605).
    a.together = grid <= 1024;
    attn_prefill_kernel<TYPE, OUT, D, WAVES, SPLIT><<<(unsigned)grid, 64 * WAVES, 0, stream>>>(a);
    return hipGetLastError();
}

template <int TYPE, int OUT>
hipError_t launch_typed(const PrefillArgs& a, hipStream_t stream) {
    // Where every wave's 32 queries have a SIMD of their own to spare, two waves
    // share them, a tile each at a time: with at most 512 such units in workgroups
    // of four waves, with at most 1024 of eight (1024 tokens, 14 heads of 64: 12.8
    // us against 20.1; 1000 after 1000, 32 heads of 128: 41.5 against 47.6; 100
    // after 1500, twice: 27.5 against 35.2; 384, 16 heads: 12.0 against 13.5). Below
    // 384 keys the joining costs what it gains (333: 13.3 both, 128: 11.6, 11.0),
    // and with more units the waves are there without it (512, four times, 28 heads:
    // 26.0 against 20.7).
    // Else eight waves share a key tile on long prompts of 128-wide heads (32 heads,
    // 4096 tokens: 145 us against 154; 8192: 502 against 522; packed sequences the
    // same); four leave fewer idle where there are few rounds of workgroups (2048
    // tokens: 54 against 62, 2500: 68 against 76) and suit 64-wide heads, whose bound
    // is the exponentials (8192 tokens, 14 heads: 164 against 177).
    const int64_t units = (a.max_q + 31) / 32 * a.q_heads * a.seqs;
    const bool half = a.max_k >= 384 && units <= 1024, little = units <= 512;
    switch (a.head_dim) {
        case 64:
            if (half) return little ? launch_one<TYPE, OUT, 64, 4, 2>(a, stream) : launch_one<TYPE, OUT, 64, 8, 2>(a, stream);
            return launch_one<TYPE, OUT, 64, 4, 1>(a, stream);
        case 128:
            if (half) return little ? launch_one<TYPE, OUT, 128, 4, 2>(a, stream) : launch_one<TYPE, OUT, 128, 8, 2>(a, stream);
            return a.max_q > 1024 && units > 3200 ? launch_one<TYPE, OUT, 128, 8, 1>(a, stream) : launch_one<TYPE, OUT, 128, 4, 1>(a, stream);
        case 256: return launch_one<TYPE, OUT, 256, 4, 1>(a, stream);
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

hipError_t launch_attn_prefill(PrefillArgs a, hipStream_t stream) {
    if (a.type == kTypeBF16)
        return a.out_type == kTypeF32 ? launch_typed<kTypeBF16, kTypeF32>(a, stream)
                                      : launch_typed<kTypeBF16, kTypeBF16>(a, stream);
    return a.out_type == kTypeF32 ? launch_typed<kTypeF16, kTypeF32>(a, stream)
                                  : launch_typed<kTypeF16, kTypeF16>(a, stream);
}

}  // namespace frq
