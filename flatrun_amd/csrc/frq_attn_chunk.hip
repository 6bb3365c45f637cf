// Attention of chunks of new tokens against the 4-bit paged cache (frq_kv4.h),
// which holds the new tokens' keys too: of a sequence with n queries and length
// len, query i sees the keys j <= i + len - n,
//   S[i, j] = scale q_i . k_j,  out_i = sum_j softmax(S)[i, j] v_j.
//
// The queries of the heads that share a key head stand side by side as rows,
// 16 to a column tile of v_mfma_f32_16x16x32_f16. The products are
// S^T = K Q^T and O^T = V^T P^T: the cache's tiles lie in the order of both left
// operands, so that a lane unpacks what it loaded and nothing of K or V passes
// through LDS; and S^T leaves a lane the eight tokens of a query that are its
// k-slots in P^T. No value goes to another lane until the end.
//
// Numbers: k and v are code times scale, rounded to fp16 (2^-12 of themselves);
// q stands under a power of two per row that makes its 8 (bf16) or 11 (fp16)
// bits exact down to 2^-28 of the row's largest; weights are fp16 numbers under
// 2^5, at most 2^12 (2^-12 of themselves, or 2^-30 of the row's largest), summed
// as they are rounded; scores, maxima and sums are fp32. A tile with a scale
// beyond 8188, whose values pass fp16, is worked on at an eighth of its values.
//
// What bounds it: few rows, the loads of the cache beside the unpacking, some 260
// vector instructions a tile of 32 tokens and 128 channels whatever the rows, and 45
// a column tile for its softmax. 17 tokens after 131000, 16 heads of 128 over 8: 51
// us and 5 for the joining, 3.0 TB/s, vector instructions 58 % of the time, matrix cores
// 24 %. 32 sequences of 2 to 9 tokens after 100 to 8000: 66 and 6 us, 2.2 TB/s; the
// short ones leave a wave of two on a SIMD. 5 tokens after 1500, 14 heads over 2 of
// 64: 8.5 and 5.4. Many rows, the matrix cores at the clock that the power leaves:
// 2048 tokens after 32768, 32 heads over 8: 34 us to unpack and 1050 to 1085 for the
// products (1.13 TF of them), matrix cores 58 % busy, vector 36, LDS 29. 8 chunks of
// 201 to 512 after 300 to 4096, 28 heads over 4: 13.5 and 105 to 118.
#include "frq_kernels.h"
#include "frq_kv4.h"

namespace frq {
namespace {

using half2v = _Float16 __attribute__((ext_vector_type(2)));
using half8v = _Float16 __attribute__((ext_vector_type(8)));
using float4v = float __attribute__((ext_vector_type(4)));
using us2 = unsigned short __attribute__((ext_vector_type(2)));

constexpr int kWaves = 4;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kUnder = 5.f, kLag = 7.f;      // of the weights' powers of two: see the head of the file
constexpr float kInf = __builtin_inff();
// Rows of a key head from which on keys are unpacked once, for a kernel whose waves
// share copies of them. After 32768 tokens, 32 heads of 128 over 8, both: 128 rows 81
// us that way and 71 without, 512 rows 117 and 147, 2048 rows 300 and 376; 128 rows
// of 256-wide heads 55 and 40.
constexpr int kHeldRows = 256;
// Bytes of them: with the parts (at most 140 MB) and the words below the 1 GiB up to
// which a stream's scratch doubles, so that contexts that grow do not leave a buffer
// behind at every step.
constexpr size_t kHeldMost = (size_t)864 << 20;

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
__device__ __forceinline__ half8v join(half2v a, half2v b, half2v c, half2v d) {
    return half8v{a[0], a[1], b[0], b[1], c[0], c[1], d[0], d[1]};
}
__device__ __forceinline__ half2v pair_of(uint32_t w) { return __builtin_bit_cast(half2v, w); }
__device__ __forceinline__ uint32_t bits_of(half2v x) { return __builtin_bit_cast(uint32_t, x); }
// (half h of a, half h of b)
__device__ __forceinline__ half2v halves(uint32_t a, uint32_t b, int h) {
    return pair_of(__builtin_amdgcn_perm(b, a, h ? 0x07060302u : 0x05040100u));
}

// A scale, half hi of w, of a token that is behind the end (it becomes zero) or
// not: 1 beyond 8188, 2 no number.
__device__ __forceinline__ int clean_half(uint32_t& w, int hi, bool past_end) {
    const uint32_t s = (hi ? w >> 16 : w) & 0x7FFFu;
    if (past_end) w &= hi ? 0xFFFFu : 0xFFFF0000u;
    return past_end || s <= 0x6FFF ? 0 : s < 0x7C00 ? 1 : 2;
}
__device__ __forceinline__ uint32_t eighth(uint32_t w) { return bits_of(pair_of(w) * (half2v){0.125f16, 0.125f16}); }

// A lane's share of a tile's K or V scales, to look for what is not ordinary.
template <int NG>
struct Flat {
    uint32_t w[(NG + 3) / 4];
    __device__ __forceinline__ void load(const uint8_t* scales, int lane) {
        if constexpr (NG == 2) {
            w[0] = reinterpret_cast<const uint16_t*>(scales)[lane];
        } else {
#pragma unroll
            for (int i = 0; i < NG / 4; ++i) w[i] = reinterpret_cast<const uint32_t*>(scales)[64 * i + lane];
        }
    }
    __device__ __forceinline__ bool large() const {                  // beyond 8188, an inf or a NaN
        us2 x = __builtin_bit_cast(us2, w[0] & 0x7FFF7FFFu);
        if constexpr (NG == 8) x = __builtin_elementwise_max(x, __builtin_bit_cast(us2, w[1] & 0x7FFF7FFFu));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(x, (us2){0x6FFF, 0x6FFF})) != 0;
    }
};

// The largest of x over the four lanes that hold a query.
__device__ __forceinline__ float quad_max(float x) {
    x = __builtin_fmaxf(x, __shfl_xor(x, 16));
    return __builtin_fmaxf(x, __shfl_xor(x, 32));
}

using const_ints = const __attribute__((address_space(4))) int32_t*;
__device__ __forceinline__ const_ints constant(const int32_t* p) { return (const_ints)(uintptr_t)p; }

// What a sequence and a workgroup's rows of it come to.
struct Span {
    int64_t q0;                // first query
    int nq, len, past;
    bool bad;                  // not what the caller said: NaN
    __device__ __forceinline__ bool read(const ChunkArgs& a, int seq) {
        const const_ints cu = constant(a.cu_q);
        q0 = cu[seq];
        const int64_t n = (int64_t)cu[seq + 1] - q0;
        len = constant(a.lens)[seq];
        len = len < 0 ? 0 : len;
        if (q0 < 0 || n <= 0 || q0 + n > a.tokens_q) return false;
        nq = (int)n;
        bad = n > a.max_q || len > a.max_len || (len > 0 && a.pages == 0);
        past = len - nq;
        return true;
    }
    // keys that rows up to `row` see, `group` rows to a token
    __device__ __forceinline__ int keys(int row, int group) const {
        const int i = row / group, e = past + (i < nq ? i : nq - 1) + 1;
        return e < 0 ? 0 : e;
    }
};

// Block `t` of all sequences' blocks of kRows rows, those of the longest sequence
// first, so that the last workgroups to start are short ones (8 chunks of 201 to
// 512 after 300 to 4096: 172 us without). Up to 64 sequences, a lane each. false:
// there is none.
__device__ __forceinline__ bool longest_first(const ChunkArgs& a, int t, int group, int kRows, int lane, int& seq, int& block) {
    int blocks = 0, len = -1;
    if (lane < a.seqs) {
        const int64_t n = (int64_t)a.cu_q[lane + 1] - a.cu_q[lane];
        len = a.lens[lane];
        blocks = n <= 0 ? 0 : n > a.max_q ? (int)a.blocks : (int)((n * group + kRows - 1) / kRows);
    }
    int start = 0;
    for (int i = 0; i < a.seqs; ++i) {
        const int l = __builtin_amdgcn_readlane(len, i), b = __builtin_amdgcn_readlane(blocks, i);
        start += l > len || (l == len && i < lane) ? b : 0;
    }
    const uint64_t here = __builtin_amdgcn_ballot_w64(start <= t && t < start + blocks);
    if (here == 0) return false;
    seq = (int)__builtin_ctzll(here);
    block = __builtin_amdgcn_readlane(blocks, seq) - 1 - (t - __builtin_amdgcn_readlane(start, seq));
    return true;
}

// LDS of a workgroup of R column tiles.
template <int NG, int R>
struct FewShared {
    __attribute__((aligned(16))) float o[2][R * 2 * NG][64][4];      // [R NG][64] queries until the sums' turn comes
    float m[kWaves][16 * R], l[kWaves][16 * R];
};

// A workgroup's part of a row block: the column tiles that have rows, R of MAX
// (32 sequences of 2 to 9 tokens, 4 heads to a key head, after 100 to 8000: 67 us,
// 85 with all three tiles for every one).
template <int TYPE, int OUT, int NG, int R, int MAX>
__device__ __forceinline__ void few_rows(const ChunkArgs& a, FewShared<NG, MAX>& sh, const Span& sp, int seq, int kvh, int block, int split,
                                         int group) {
    using T = Val<TYPE>;
    using O = Val<OUT>;
    constexpr int D = 32 * NG, kTile = kv_tile_bytes(NG), kRows = 16 * MAX;
    constexpr bool kHeld = NG * R <= 8;            // queries in registers, or in LDS
    half8v (*sh_q)[64] = reinterpret_cast<half8v(*)[64]>(&sh.o[0][0][0][0]);
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int row0 = block * kRows, rows = sp.nq * group;
    const int end = sp.keys(row0 + kRows - 1, group);                // keys that the workgroup's rows see
    const int tiles = (end + kKvTile - 1) / kKvTile;
    const int first = split * (int)a.share;
    const int last = tiles < first + (int)a.share ? tiles : first + (int)a.share;
    if (first >= tiles && split) return;                             // nothing here: the joining knows
    const int whole = sp.keys(row0, group);                          // keys below this one every row sees

    const const_ints table = constant(a.table) + (int64_t)seq * a.ld_table;
    const uint32_t page_tiles = (uint32_t)a.page_tokens / kKvTile;
    const int64_t page_bytes = a.kv_heads * (int64_t)page_tiles * kTile;
    const uint8_t* heads = static_cast<const uint8_t*>(a.cache) + (int64_t)kvh * page_tiles * kTile;
    bool bad = false;
    // Pages are looked up a step before their tile is asked for. Past the last
    // tile that one is asked for again: a load that may not have been issued
    // would make the compiler wait for those after it.
    auto page_index = [&](int tile) { return (uint32_t)(((uint64_t)(uint32_t)tile * a.per_page) >> 36); };
    auto look_up = [&](int tile) { return table[page_index(tile < last ? tile : last - 1)]; };
    auto address = [&](int tile, int page) {
        if ((uint32_t)page >= (uint64_t)a.pages) {
            bad = true;
            page = 0;
        }
        tile = tile < last ? tile : last - 1;
        const uint32_t in = (uint32_t)tile - page_index(tile) * page_tiles;
        return heads + page * page_bytes + (int64_t)in * kTile;
    };
    uint32_t kc[2 * NG], ks[NG], vc[2 * NG], vs[4][NG];              // a tile's codes and scales as a lane holds them
    Flat<NG> fk, fv;
    auto fetch_k = [&](const uint8_t* t) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < 2 * NG; p += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(t + kv_word(p, lane));
            kc[p] = x.x; kc[p + 1] = x.y; kc[p + 2] = x.z; kc[p + 3] = x.w;
        }
#pragma unroll
        for (int p = 0; p < NG; p += 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(t + kv_ks_off(NG) + kv_scale(n, 0, NG) + 4 * p);
            ks[p] = x.x; ks[p + 1] = x.y;
        }
        fk.load(t + kv_ks_off(NG), lane);
    };
    auto fetch_v = [&](const uint8_t* t) __attribute__((always_inline)) {
#pragma unroll
        for (int p = 0; p < 2 * NG; p += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(t + kv_vc_off(NG) + kv_word(p, lane));
            vc[p] = x.x; vc[p + 1] = x.y; vc[p + 2] = x.z; vc[p + 3] = x.w;
        }
#pragma unroll
        for (int i = 0; i < 4; ++i)                                  // tokens 4j + i and 16 more
#pragma unroll
            for (int p = 0; p < NG; p += 2) {
                const uint2 x = *reinterpret_cast<const uint2*>(t + kv_vs_off(NG) + kv_scale(4 * j + i, 0, NG) + 4 * p);
                vs[i][p] = x.x; vs[i][p + 1] = x.y;
            }
        fv.load(t + kv_vs_off(NG), lane);
    };
    int tile = first + wave, page = 0;
    const uint8_t* at = nullptr;
    if (tile < last) {
        at = address(tile, look_up(tile));
        page = look_up(tile + kWaves);
        fetch_k(at);
        fetch_v(at);
    }

    // the lane's rows, one of each column tile: queries, and the last key they see
    half8v qf[kHeld ? R : 1][NG];
    float rs[R], m[R], nref[R], l[R];
    int lim[R];
#pragma unroll
    for (int c = 0; c < R; ++c) {
        int row = row0 + 16 * c + n;
        row = row < rows ? row : rows - 1;
        const int i = row / group;
        lim[c] = sp.past + i;
        const typename T::Elem* q = static_cast<const typename T::Elem*>(a.q) + (sp.q0 + i) * a.ld_q +
                                    (int64_t)(kvh * group + row - i * group) * D;
        float x[NG][8];
        uint32_t top = 0;                                            // bits of the largest |q|; inf and NaN above all
#pragma unroll
        for (int g = 0; g < NG; ++g) T::load8(q + 32 * g + 8 * j, x[g]);
#pragma unroll
        for (int g = 0; g < NG; ++g)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t b = __builtin_bit_cast(uint32_t, x[g][e]) & 0x7FFFFFFFu;
                top = top > b ? top : b;
            }
        uint32_t other = __shfl_xor(top, 16);
        top = top > other ? top : other;
        other = __shfl_xor(top, 32);
        top = top > other ? top : other;
        const int up = top ? 140 - (int)(top >> 23) : 0;             // the largest to [2^13, 2^14)
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            half8v y;
#pragma unroll
            for (int e = 0; e < 8; ++e) y[e] = (_Float16)__builtin_ldexpf(x[g][e], up);
            if constexpr (kHeld)
                qf[c][g] = y;
            else if (wave == c % kWaves)
                sh_q[c * NG + g][lane] = y;
        }
        rs[c] = top >= 0x7F800000u ? __builtin_nanf("") : __builtin_ldexpf(a.scale * kLog2e, -up);
        m[c] = -kInf;
        nref[c] = 0.f;
        l[c] = 0.f;
    }
    if constexpr (!kHeld) __syncthreads();
    float4v o[R][2 * NG];
#pragma unroll
    for (int c = 0; c < R; ++c)
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) o[c][i] = float4v{0, 0, 0, 0};

    for (; tile < last; tile += kWaves) {
        const uint8_t* next = address(tile + kWaves, page);
        page = look_up(tile + 2 * kWaves);
        const int kt = tile * kKvTile;
        const bool masked = kt + kKvTile > whole;
        float up = 1.f;
        // A scale beyond 8188, an inf or a NaN? What is behind the sequence's end
        // is nobody's and becomes zero.
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(fk.large()) != 0, 0)) {
            bool big = false;
#pragma unroll
            for (int x = 0; x < 2 * NG; ++x) {
                const int token = kt + 16 * (x / NG) + n;
                big |= clean_half(ks[x / 2], x & 1, token >= sp.len) == 1;
            }
            if (__builtin_amdgcn_ballot_w64(big)) {
                up = 8.f;
#pragma unroll
                for (int p = 0; p < NG; ++p) ks[p] = eighth(ks[p]);
            }
        }
        // scores of tokens 16u + 4j .. 4j + 3: K of 16 tokens and 32 channels at a time
        float4v s[R][2];
#pragma unroll
        for (int c = 0; c < R; ++c) s[c][0] = s[c][1] = float4v{0, 0, 0, 0};
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            half8v q[R];
#pragma unroll
            for (int c = 0; c < R; ++c) {
                if constexpr (kHeld)
                    q[c] = qf[c][g];
                else
                    q[c] = sh_q[c * NG + g][lane];
            }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                const uint32_t w = kc[u * NG + g], at2 = ks[(u * NG + g) / 2];
                const half2v d = halves(at2, at2, (u * NG + g) & 1);
                const half8v kf = join(low_pair(w) * d, high_pair(w) * d, low_pair(w >> 8) * d, high_pair(w >> 8) * d);
#pragma unroll
                for (int c = 0; c < R; ++c) s[c][u] = __builtin_amdgcn_mfma_f32_16x16x32_f16(kf, q[c], s[c][u], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        fetch_k(next);                                               // these registers are free again
        half8v pf[R];
#pragma unroll
        for (int c = 0; c < R; ++c) {
            const float by = rs[c] * up;
            if (masked) {
#pragma unroll
                for (int u = 0; u < 2; ++u)
#pragma unroll
                    for (int i = 0; i < 4; ++i)
                        if (kt + 16 * u + 4 * j + i > lim[c]) s[c][u][i] = -kInf;
            }
            float top = s[c][0][0];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; ++i) top = __builtin_fmaxf(top, s[c][u][i]);
            top *= by;
            if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m[c] + kLag) != 0, 0)) {
                // each row by its own scores alone
                const float all = quad_max(top), mn = all > m[c] + kLag ? all : m[c];
                const float keep = mn == -kInf ? 1.f : __builtin_amdgcn_exp2f(m[c] - mn);
                m[c] = mn;
                nref[c] = mn == -kInf ? 0.f : -mn;
                l[c] *= keep;
#pragma unroll
                for (int d = 0; d < 2 * NG; ++d) o[c][d] *= keep;
            }
            half2v p[4];
            float sum = 0.f;
            const float ref = nref[c] + kUnder;
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 4; i += 2) {
                    const float p0 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][u][i], by, ref));
                    const float p1 = __builtin_amdgcn_exp2f(__builtin_fmaf(s[c][u][i + 1], by, ref));
                    p[2 * u + i / 2] = half2v{(_Float16)p0, (_Float16)p1};
                    sum = __builtin_amdgcn_fdot2(p[2 * u + i / 2], (half2v){(_Float16)1.f, (_Float16)1.f}, sum, false);
                }
            l[c] += sum;
            pf[c] = join(p[0], p[1], p[2], p[3]);
        }
        // V of 16 channels at a time
        int odd = 0;                                                 // 1 a large scale, 2 blocks taken out of the product
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(fv.large()) != 0, 0)) {
            // A zero weight does not take a NaN out of a product: where rows
            // differ in what they see, a block that is no number leaves it, to be
            // added below for the rows that see it.
            bool any = false, big = false;
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int x = 0; x < 2 * NG; ++x) {
                    const int token = kt + 16 * (x / NG) + 4 * j + i;
                    const int f = clean_half(vs[i][x / 2], x & 1, token >= sp.len);
                    big |= f == 1;
                    any |= f == 2 && masked;
                    if (f == 2 && masked) vs[i][x / 2] &= x & 1 ? 0xFFFFu : 0xFFFF0000u;
                }
            odd = (__builtin_amdgcn_ballot_w64(big) ? 1 : 0) | (__builtin_amdgcn_ballot_w64(any) ? 2 : 0);
        }
        if (__builtin_expect(odd & 1, 0)) {                          // values past fp16: all at an eighth for this tile
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int p = 0; p < NG; ++p) vs[i][p] = eighth(vs[i][p]);
#pragma unroll
            for (int c = 0; c < R; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NG; ++d) o[c][d] *= 0.125f;
        }
#pragma unroll
        for (int g = 0; g < NG; ++g) {
            const uint32_t w0 = vc[2 * g], w1 = vc[2 * g + 1];
            half2v d[4];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int i = 0; i < 2; ++i) {
                    const int p = (u * NG + g) / 2, h = (u * NG + g) & 1;
                    d[2 * u + i] = halves(vs[2 * i][p], vs[2 * i + 1][p], h);
                }
            const half8v va = join(low_pair(w0) * d[0], low_pair(w0 >> 8) * d[1], low_pair(w1) * d[2], low_pair(w1 >> 8) * d[3]);
            const half8v vb = join(high_pair(w0) * d[0], high_pair(w0 >> 8) * d[1], high_pair(w1) * d[2], high_pair(w1 >> 8) * d[3]);
#pragma unroll
            for (int c = 0; c < R; ++c) {
                o[c][2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(va, pf[c], o[c][2 * g], 0, 0, 0);
                o[c][2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(vb, pf[c], o[c][2 * g + 1], 0, 0, 0);
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(odd & 1, 0)) {
#pragma unroll
            for (int c = 0; c < R; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NG; ++d) o[c][d] *= 8.f;
        }
        fetch_v(next);
        if (__builtin_expect(odd & 2, 0)) {
            for (int t = 0; t < kKvTile && kt + t < sp.len; ++t)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint16_t b = *reinterpret_cast<const uint16_t*>(at + kv_vs_off(NG) + kv_scale(t, g, NG));
                    if ((b & 0x7C00) == 0x7C00) {
#pragma unroll
                        for (int c = 0; c < R; ++c)
                            if (kt + t <= lim[c]) o[c][2 * g] += __builtin_nanf(""), o[c][2 * g + 1] += __builtin_nanf("");
                    }
                }
        }
        at = next;
    }
    if (__builtin_amdgcn_ballot_w64(bad)) {
#pragma unroll
        for (int c = 0; c < R; ++c) l[c] = __builtin_nanf("");
    }

    // the waves' sums, under the largest of their references: 2 and 3 to 0 and 1, 1 to 0
#pragma unroll
    for (int c = 0; c < R; ++c) {
        l[c] += __shfl_xor(l[c], 16);
        l[c] += __shfl_xor(l[c], 32);
        if (j == 0) {
            sh.m[wave][16 * c + n] = m[c];
            sh.l[wave][16 * c + n] = l[c];
        }
    }
    __syncthreads();
#pragma unroll
    for (int c = 0; c < R; ++c) {
        float mm = sh.m[0][16 * c + n];
#pragma unroll
        for (int w = 1; w < kWaves; ++w) mm = __builtin_fmaxf(mm, sh.m[w][16 * c + n]);
        const float base = mm == -kInf ? 0.f : mm, f = __builtin_amdgcn_exp2f(m[c] - base);
#pragma unroll
        for (int d = 0; d < 2 * NG; ++d) o[c][d] *= f;
        float sum = 0.f;
#pragma unroll
        for (int w = 0; w < kWaves; ++w) sum += sh.l[w][16 * c + n] * __builtin_amdgcn_exp2f(sh.m[w][16 * c + n] - base);
        l[c] = sum;
        m[c] = mm;
    }
#pragma unroll
    for (int half = 2; half; half >>= 1) {
        if (wave >= half && wave < 2 * half)
#pragma unroll
            for (int c = 0; c < R; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NG; ++d) *reinterpret_cast<float4v*>(sh.o[wave - half][c * 2 * NG + d][lane]) = o[c][d];
        __syncthreads();
        if (wave < half)
#pragma unroll
            for (int c = 0; c < R; ++c)
#pragma unroll
                for (int d = 0; d < 2 * NG; ++d) o[c][d] += *reinterpret_cast<const float4v*>(sh.o[wave][c * 2 * NG + d][lane]);
        __syncthreads();
    }
    if (wave) return;
#pragma unroll
    for (int c = 0; c < R; ++c) {
        const int row = row0 + 16 * c + n;
        if (row >= rows) continue;
        if (a.splits > 1) {
            float* part = a.part + (((int64_t)(seq * a.kv_heads + kvh) * a.blocks + block) * a.splits + split) * kRows * (D + 4) +
                          (16 * c + n) * (D + 4);
#pragma unroll
            for (int d = 0; d < 2 * NG; ++d) *reinterpret_cast<float4v*>(part + 16 * d + 4 * j) = o[c][d];
            if (j == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m[c], l[c]);
            continue;
        }
        // zeros for a query without keys; no weight at all elsewhere is 0 / 0
        const int i = row / group;
        const float inv = 1.0f / l[c];
        typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (sp.q0 + i) * a.ld_out + (int64_t)(kvh * group + row - i * group) * D;
#pragma unroll
        for (int d = 0; d < 2 * NG; ++d) {
            typename O::Elem y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = O::one(lim[c] < 0 ? 0.f : l[c] == 0.f ? __builtin_nanf("") : o[c][d][e] * inv);
            __builtin_memcpy(__builtin_assume_aligned(out + 16 * d + 4 * j, 4 * sizeof(y[0])), y, sizeof(y));
        }
    }
}

template <int TYPE, int OUT, int NG, int R>
__global__ void __launch_bounds__(64 * kWaves, NG == 8 ? 1 : 2) attn_chunk_kernel(ChunkArgs a) {
    using O = Val<OUT>;
    constexpr int D = 32 * NG, kRows = 16 * R;
    __shared__ FewShared<NG, R> sh;
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    uint32_t id = blockIdx.x;
    // Workgroup i goes to XCD i % 8: the parts go round from row to row, else an XCD
    // would have all the last ones, which short sequences do not have.
    int split = (int)(id % (uint32_t)a.splits);
    id /= (uint32_t)a.splits;
    split = (int)(((uint32_t)split + id) % (uint32_t)a.splits);
    const int kvh = (int)(id % (uint32_t)a.kv_heads);
    id /= (uint32_t)a.kv_heads;
    const int seq = (int)(id / (uint32_t)a.blocks), block = (int)(a.blocks - 1 - id % (uint32_t)a.blocks);
    Span sp;
    if (!sp.read(a, seq)) return;
    if (sp.bad) {
        if (split) return;
        for (int64_t i = block; i < sp.nq; i += a.blocks) {
            typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (sp.q0 + i) * a.ld_out + (int64_t)kvh * group * D;
            for (int e = threadIdx.x; e < group * D; e += 64 * kWaves) out[e] = O::one(__builtin_nanf(""));
        }
        return;
    }
    const int rest = sp.nq * group - block * kRows;
    if (rest <= 0) return;
    if (rest <= 16)
        few_rows<TYPE, OUT, NG, 1, R>(a, sh, sp, seq, kvh, block, split, group);
    else if (R > 2 && rest <= 32)
        few_rows<TYPE, OUT, NG, (R > 2 ? 2 : R), R>(a, sh, sp, seq, kvh, block, split, group);
    else
        few_rows<TYPE, OUT, NG, R, R>(a, sh, sp, seq, kvh, block, split, group);
}

// --------------------------------------------------------------- many rows
//
// Where hundreds of rows read the same keys, unpacking them for every 64 would be
// half of the work: one kernel unpacks every key and value of the call once, into
// scratch, and a second one has W waves of 32 rows each share what it copies from
// there, 64 tokens at a time, to LDS, on v_mfma_f32_32x32x16_f16.
using float16v = float __attribute__((ext_vector_type(16)));
constexpr int kKeys = 64;

// Four words of a tile's K (k < NG / 2) or V codes and their scales, as a lane
// holds them: of K the words (u, g) of token 16u + n, of V (g, u) of tokens 16u +
// 4j .. 4j + 3. Word x: K u = (4k + x) / NG, g = (4k + x) % NG; V g = 2v + x / 2, u = x % 2.
template <int NG>
struct Unit {
    uint32_t code[4], scale[8];
    __device__ __forceinline__ void load(const uint8_t* t, int unit, int lane) {
        const int n = lane & 15, j = lane >> 4;
        const bool v = unit >= NG / 2;
        const int k = v ? unit - NG / 2 : unit;
        const uint4 x = *reinterpret_cast<const uint4*>(t + (v ? kv_vc_off(NG) : 0) + kv_word(4 * k, lane));
        code[0] = x.x; code[1] = x.y; code[2] = x.z; code[3] = x.w;
        if (v) {
#pragma unroll
            for (int i = 0; i < 4; ++i)
#pragma unroll
                for (int u = 0; u < 2; ++u)            // groups 2k and 2k + 1
                    scale[2 * i + u] = *reinterpret_cast<const uint32_t*>(t + kv_vs_off(NG) + kv_scale(4 * j + i + 16 * u, 2 * k, NG));
        } else {
#pragma unroll
            for (int x2 = 0; x2 < 2; ++x2) {           // words 2 x2 and 2 x2 + 1
                const int w = 4 * k + 2 * x2;
                scale[x2] = *reinterpret_cast<const uint32_t*>(t + kv_ks_off(NG) + kv_scale(n + 16 * (w / NG), w % NG, NG));
            }
        }
    }
    __device__ __forceinline__ bool large(bool v) const {            // beyond 8188, an inf or a NaN
        us2 x = __builtin_bit_cast(us2, scale[0] & 0x7FFF7FFFu);
        x = __builtin_elementwise_max(x, __builtin_bit_cast(us2, scale[1] & 0x7FFF7FFFu));
        if (v)
#pragma unroll
            for (int i = 2; i < 8; ++i) x = __builtin_elementwise_max(x, __builtin_bit_cast(us2, scale[i] & 0x7FFF7FFFu));
        return __builtin_bit_cast(uint32_t, __builtin_elementwise_sub_sat(x, (us2){0x6FFF, 0x6FFF})) != 0;
    }
};

// A unit's values to where the products read them: K and V of 64 tokens, `half`
// the unit's tile of the two.
template <int NG>
__device__ __forceinline__ void put_unit(const Unit<NG>& r, int unit, int half, int lane, _Float16* kb, _Float16* vb) {
    const int n = lane & 15, j = lane >> 4;
    if (unit >= NG / 2) {
        const int k = unit - NG / 2;
#pragma unroll
        for (int w = 0; w < 4; ++w) {                                // group g, tokens 16u + 4j + i
            const int g = 2 * k + w / 2, u = w & 1, hi = w / 2;
            const half2v d0 = halves(r.scale[u], r.scale[2 + u], hi), d1 = halves(r.scale[4 + u], r.scale[6 + u], hi);
            const uint32_t c = r.code[w];
            // operand of group g and tokens 32 half + 16u ..: lane 32 (j & 1) + channel, its four tokens j / 2
            half2v* to = reinterpret_cast<half2v*>(vb + ((g * 4 + 2 * half + u) * 64 + 32 * (j & 1) + n) * 8 + 4 * (j >> 1));
            const uint2 low = make_uint2(bits_of(low_pair(c) * d0), bits_of(low_pair(c >> 8) * d1));
            const uint2 high = make_uint2(bits_of(high_pair(c) * d0), bits_of(high_pair(c >> 8) * d1));
            *reinterpret_cast<uint2*>(to) = low;
            *reinterpret_cast<uint2*>(to + 16 * 4) = high;           // 16 channels on
        }
    } else {
#pragma unroll
        for (int w = 0; w < 4; ++w) {                                // token 16u + n, channels 32g + 8j ..
            const int p = 4 * unit + w, u = p / NG, g = p % NG;
            const half2v d = halves(r.scale[w / 2], r.scale[w / 2], w & 1);
            const uint32_t c = r.code[w];
            *reinterpret_cast<half8v*>(kb + ((4 * g + j) * kKeys + 32 * half + 16 * u + n) * 8) =
                join(low_pair(c) * d, high_pair(c) * d, low_pair(c >> 8) * d, high_pair(c >> 8) * d);
        }
    }
}
// What is not ordinary in a unit of tokens t0 ..: zeros behind the sequence's end,
// and 1 for a large scale, 2 for no number in V.
template <int NG>
__device__ __forceinline__ int clean_unit(Unit<NG>& r, int unit, int t0, int len, int lane) {
    const int n = lane & 15, j = lane >> 4;
    bool any = false, big = false;
    if (unit >= NG / 2) {
#pragma unroll
        for (int x = 0; x < 16; ++x) {
            const int f = clean_half(r.scale[x / 2], x & 1, t0 + 4 * j + x / 4 + 16 * (x / 2 & 1) >= len);
            big |= f == 1;
            any |= f == 2;
        }
    } else {
#pragma unroll
        for (int x = 0; x < 4; ++x) big |= clean_half(r.scale[x / 2], x & 1, t0 + n + 16 * ((4 * unit + x) / NG) >= len) == 1;
    }
    return (__builtin_amdgcn_ballot_w64(big) ? 1 : 0) | (__builtin_amdgcn_ballot_w64(any) ? 2 : 0);
}

// Every key and value of the call, 64 tokens of a key head to a workgroup, in the
// order in which LDS will hold them. A word beside them says what is not ordinary: 1 V at an eighth, 2 no number in V, 4 K at an
// eighth, 8 a page outside the cache.
constexpr int unpack_waves(int ng) { return ng == 2 ? 4 : 8; }
template <int NG>
__global__ void __launch_bounds__(64 * unpack_waves(NG)) attn_chunk_unpack_kernel(ChunkArgs a) {
    constexpr int W = unpack_waves(NG), kUnits = 2 * NG / W, kBuf = kKeys * 32 * NG;
    __shared__ int sh_flags;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const uint32_t id = blockIdx.x / (uint32_t)a.steps;
    const int step = (int)(blockIdx.x - id * (uint32_t)a.steps);
    const int seq = (int)(id / (uint32_t)a.kv_heads), kvh = (int)(id % (uint32_t)a.kv_heads);
    Span sp;
    if (!sp.read(a, seq) || sp.bad || step * kKeys >= sp.len) return;
    const uint32_t page_tiles = (uint32_t)a.page_tokens / kKvTile;
    const int half = kUnits * wave / NG, tiles = (sp.len + kKvTile - 1) / kKvTile, want = 2 * step + half;
    const int tile = want < tiles ? want : tiles - 1;
    const uint32_t in = (uint32_t)(((uint64_t)(uint32_t)tile * a.per_page) >> 36);
    int page = constant(a.table)[(int64_t)seq * a.ld_table + in];
    int f = 0;
    if ((uint32_t)page >= (uint64_t)a.pages) {
        f = 8;
        page = 0;
    }
    const uint8_t* t = static_cast<const uint8_t*>(a.cache) +
                       ((page * a.kv_heads + kvh) * (int64_t)page_tiles + ((uint32_t)tile - in * page_tiles)) * kv_tile_bytes(NG);
    Unit<NG> raw[kUnits];
#pragma unroll
    for (int x = 0; x < kUnits; ++x) raw[x].load(t, (kUnits * wave + x) % NG, lane);
    if (threadIdx.x == 0) sh_flags = 0;
    __syncthreads();
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
        const int unit = (kUnits * wave + x) % NG;
        const bool v = unit >= NG / 2;
        if (__builtin_amdgcn_ballot_w64(raw[x].large(v)) == 0) continue;
        const int c = clean_unit<NG>(raw[x], unit, want * kKvTile, sp.len, lane);
        f |= v ? c : (c & 1) << 2;
    }
    if (f && lane == 0) atomicOr(&sh_flags, f);
    __syncthreads();
    f = sh_flags;
    _Float16* to = static_cast<_Float16*>(a.held) + (int64_t)blockIdx.x * (2 * kBuf);
#pragma unroll
    for (int x = 0; x < kUnits; ++x) {
        const int unit = (kUnits * wave + x) % NG;
        if (f & (unit >= NG / 2 ? 1 : 4))
#pragma unroll
            for (int i = 0; i < 8; ++i) raw[x].scale[i] = eighth(raw[x].scale[i]);
        put_unit<NG>(raw[x], unit, half, lane, to, to + kBuf);
    }
    if (threadIdx.x == 0) a.held_flags[blockIdx.x] = f;
}

template <int TYPE, int OUT, int NG, int W>
__global__ void __launch_bounds__(64 * W, NG == 8 ? 1 : 2) attn_chunk_rows_kernel(ChunkArgs a) {
    using T = Val<TYPE>;
    using O = Val<OUT>;
    constexpr int D = 32 * NG, kRows = 32 * W, NK = D / 16, ND = NG, kBuf = kKeys * D;
    // a K and a V tile twice, used in turn: objects of their own, so that the
    // compiler sees that a read of one need not wait for the copies into the other
    __shared__ __attribute__((aligned(16))) _Float16 kb0[kBuf], kb1[kBuf], vb0[kBuf], vb1[kBuf];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int ln = lane & 31, h = lane >> 5;
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    uint32_t id = blockIdx.x;
    const int split = (int)(id % (uint32_t)a.splits);
    id /= (uint32_t)a.splits;
    const int kvh = (int)(id % (uint32_t)a.kv_heads);
    id /= (uint32_t)a.kv_heads;
    int seq = (int)(id / (uint32_t)a.blocks), block = (int)(a.blocks - 1 - id % (uint32_t)a.blocks);    // the longest rows first
    if (a.sorted && !longest_first(a, (int)id, group, kRows, lane, seq, block)) return;
    Span sp;
    if (!sp.read(a, seq)) return;
    if (sp.bad) {
        if (split) return;
        for (int64_t i = block; i < sp.nq; i += a.blocks) {
            typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (sp.q0 + i) * a.ld_out + (int64_t)kvh * group * D;
            for (int e = threadIdx.x; e < group * D; e += 64 * W) out[e] = O::one(__builtin_nanf(""));
        }
        return;
    }
    const int row0 = block * kRows, rows = sp.nq * group;
    if (row0 >= rows) return;
    const int end = sp.keys(row0 + kRows - 1, group);
    const int tiles = (end + kKvTile - 1) / kKvTile;
    const int first = split * (int)a.share;                          // even
    const int last = tiles < first + (int)a.share ? tiles : first + (int)a.share;
    if (first >= tiles && split) return;
    const int whole = sp.keys(row0, group);                          // keys below this one every row of the workgroup sees
    const int wrow = row0 + 32 * wave;                               // the wave's rows
    const int seen = wrow < rows ? sp.keys(wrow + 31, group) : 0, own = wrow < rows ? sp.keys(wrow, group) : 0;

    // the unpacked steps of the sequence and key head, and their words
    const int64_t steps0 = ((int64_t)seq * a.kv_heads + kvh) * a.steps;
    const _Float16* held = static_cast<const _Float16*>(a.held) + steps0 * (2 * kBuf);
    const const_ints words = constant(a.held_flags) + steps0;
    // Asynchronous copy of a step's K (or V), as it lies, 16 bytes a lane and turn.
    auto copy = [&](int tile, bool v, _Float16* to) __attribute__((always_inline)) {
        constexpr int kTurns = kBuf / 8 / (64 * W);
        const __amdgpu_buffer_rsrc_t r = buffer_rsrc(held + (int64_t)(tile / 2) * (2 * kBuf) + (v ? kBuf : 0), kBuf * 2);
#pragma unroll
        for (int i = 0; i < kTurns; ++i) {
            const int at = (i * W + wave) * 64;
            __builtin_amdgcn_raw_ptr_buffer_load_lds(r, (__attribute__((address_space(3))) void*)(to + at * 8), 16, (at + lane) * 16, 0, 0, 0);
        }
    };
    if (first < last) {
        copy(first, false, kb0);
        copy(first, true, vb0);
        if (first + 2 < last) copy(first + 2, false, kb1);
    }

    // the lane's row
    int row = wrow + ln;
    row = row < rows ? row : rows - 1;
    const int qi = row / group, head = kvh * group + row - qi * group, lim = sp.past + qi;
    half8v qf[NK];
    float rs;
    {
        const typename T::Elem* q = static_cast<const typename T::Elem*>(a.q) + (sp.q0 + qi) * a.ld_q + (int64_t)head * D;
        float x[NK][8];
        uint32_t top = 0;
#pragma unroll
        for (int s = 0; s < NK; ++s) T::load8(q + 16 * s + 8 * h, x[s]);
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) {
                const uint32_t b = __builtin_bit_cast(uint32_t, x[s][e]) & 0x7FFFFFFFu;
                top = top > b ? top : b;
            }
        const uint32_t other = __shfl_xor(top, 32);
        top = top > other ? top : other;
        const int up = top ? 140 - (int)(top >> 23) : 0;
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int e = 0; e < 8; ++e) qf[s][e] = (_Float16)__builtin_ldexpf(x[s][e], up);
        rs = top >= 0x7F800000u ? __builtin_nanf("") : __builtin_ldexpf(a.scale * kLog2e, -up);
    }
    float16v o[ND];
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; ++i) o[d][i] = 0.f;
    float m = -kInf, nref = 0.f, l = 0.f;

    // the waves meet, and what any of them has copied is there
    auto meet = [&]() __attribute__((always_inline)) {
        __builtin_amdgcn_s_waitcnt(0x0070);                          // vmcnt(0), lgkmcnt(0)
        __builtin_amdgcn_s_barrier();
    };
    bool bad = false;
    float16v sa[2], sb[2];
    float up = 1.f;                                                  // of the scores at hand
    int word = 0;                                                    // of the next step
    meet();
    if (first < last) {
        word = words[first / 2];
        up = word & 4 ? 8.f : 1.f;
#pragma unroll
        for (int i = 0; i < 16; ++i) sa[0][i] = sa[1][i] = 0.f;
#pragma unroll
        for (int s = 0; s < NK; ++s)
#pragma unroll
            for (int t = 0; t < 2; ++t) {
                const half8v kf = *reinterpret_cast<const half8v*>(kb0 + ((2 * s + h) * kKeys + 32 * t + ln) * 8);
                sa[t] = __builtin_amdgcn_mfma_f32_32x32x16_f16(kf, qf[s], sa[t], 0, 0, 0);
            }
    }
    // Softmax and P V of a step, whose scores st holds, and the scores of the next:
    // K is a step ahead of V, so that those products go on beside the exponentials.
    auto step = [&](int tile, float16v (&st)[2], float16v (&sn)[2], _Float16* k_next, _Float16* k_after, _Float16* v_now,
                    _Float16* v_next) __attribute__((always_inline)) {
        meet();                                                      // K of the next step and V of this one are there
        const int f = word;
        float up_next = 1.f;
        if (tile + 4 < last) copy(tile + 4, false, k_after);
        if (tile + 2 < last) {
            copy(tile + 2, true, v_next);
            word = words[tile / 2 + 1];
            up_next = word & 4 ? 8.f : 1.f;
        }
        bad |= (f & 8) != 0;
        if (__builtin_expect((f & 2) && tile * kKvTile + kKeys > whole, 0)) {
            // a zero weight does not take a NaN out of a product: it leaves V
            // and is added below for the rows that see it
            for (int i = threadIdx.x; i < kBuf / 2; i += 64 * W) {
                uint32_t& w = reinterpret_cast<uint32_t*>(v_now)[i];
                const uint32_t x = w;
                w = x & ~(((x & 0x7C00u) == 0x7C00u ? 0xFFFFu : 0u) | ((x & 0x7C000000u) == 0x7C000000u ? 0xFFFF0000u : 0u));
            }
            __syncthreads();
        }
        const float down = f & 1 ? 0.125f : 1.f, under = f & 1 ? kUnder + 3.f : kUnder;
        const float by = rs * up;
        up = up_next;
        const int kt = tile * kKvTile;
        if (kt >= seen) return;                                      // nothing here for the wave, nor further on
        if (__builtin_expect(kt + kKeys > own || kt + kKeys > last * kKvTile, 0)) {
            // of the split's own tiles, what the row sees
            const int e = last * kKvTile - 1, left = (lim < e ? lim : e) - kt - 4 * h;
#pragma unroll
            for (int t = 0; t < 2; ++t)
#pragma unroll
                for (int i = 0; i < 16; ++i)
                    if (32 * t + 8 * (i >> 2) + (i & 3) > left) st[t][i] = -kInf;
        }
        float top = st[0][0];
#pragma unroll
        for (int t = 0; t < 2; ++t)
#pragma unroll
            for (int i = 0; i < 16; ++i) top = __builtin_fmaxf(top, st[t][i]);
        top *= by;
        if (__builtin_expect(__builtin_amdgcn_ballot_w64(top > m + kLag) != 0, 0)) {
            const float all = __builtin_fmaxf(top, __shfl_xor(top, 32)), mn = all > m + kLag ? all : m;
            const float keep = mn == -kInf ? 1.f : __builtin_amdgcn_exp2f(m - mn);
            m = mn;
            nref = mn == -kInf ? 0.f : -mn;
            l *= keep;
#pragma unroll
            for (int d = 0; d < ND; ++d)
#pragma unroll
                for (int i = 0; i < 16; ++i) o[d][i] *= keep;
        }
        // The next step's scores (of whatever LDS holds, where there is none)
        // beside this one's exponentials, operands four products ahead.
        auto k_of = [&](int x) { return *reinterpret_cast<const half8v*>(k_next + ((2 * (x >> 1) + h) * kKeys + 32 * (x & 1) + ln) * 8); };
        auto v_of = [&](int x) { return *reinterpret_cast<const half8v*>(v_now + ((x % ND * 4 + x / ND) * 64 + lane) * 8); };
        constexpr int kPer = 16 / NK;                                // of the 32 scores to a product
        half8v ahead[4];
        uint32_t pw[16];
        float sum = 0.f, odd = 0.f;
        const float ref = nref + under;
        __builtin_amdgcn_sched_barrier(0);
#pragma unroll
        for (int x = 0; x < 4; ++x) ahead[x] = k_of(x);
#pragma unroll
        for (int i = 0; i < 16; ++i) sn[0][i] = sn[1][i] = 0.f;
#pragma unroll
        for (int x = 0; x < 2 * NK; ++x) {
            sn[x & 1] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[x & 3], qf[x >> 1], sn[x & 1], 0, 0, 0);
            ahead[x & 3] = x + 4 < 2 * NK ? k_of(x + 4) : v_of(x + 4 - 2 * NK);
#pragma unroll
            for (int y = 0; y < kPer; ++y) {
                const int i = x * kPer + y;
                const float p = __builtin_amdgcn_exp2f(__builtin_fmaf(st[i >> 4][i & 15], by, ref));
                if (i & 1) {
                    const half2v w = {(_Float16)odd, (_Float16)p};
                    pw[i / 2] = bits_of(w);
                    sum = __builtin_amdgcn_fdot2(w, (half2v){(_Float16)1.f, (_Float16)1.f}, sum, false);
                } else {
                    odd = p;
                }
            }
            __builtin_amdgcn_sched_barrier(0);
        }
        l = __builtin_fmaf(sum, down, l);
#pragma unroll
        for (int x = 0; x < 4 * ND; ++x) {
            const int s = x / ND, d = x % ND;
            const half8v pf = join(pair_of(pw[4 * s]), pair_of(pw[4 * s + 1]), pair_of(pw[4 * s + 2]), pair_of(pw[4 * s + 3]));
            o[d] = __builtin_amdgcn_mfma_f32_32x32x16_f16(ahead[x & 3], pf, o[d], 0, 0, 0);
            if (x + 4 < 4 * ND) ahead[x & 3] = v_of(x + 4);
            __builtin_amdgcn_sched_barrier(0);
        }
        if (__builtin_expect(f & 2, 0)) {
            const const_ints table = constant(a.table) + (int64_t)seq * a.ld_table;
            const uint32_t page_tiles = (uint32_t)a.page_tokens / kKvTile;
            for (int t = 0; t < kKeys && kt + t < sp.len; ++t) {
                const uint32_t at = (uint32_t)(kt + t) / kKvTile, in = (uint32_t)(((uint64_t)at * a.per_page) >> 36);
                const int page = table[in];
                if ((uint32_t)page >= (uint64_t)a.pages) break;
                const uint8_t* there = static_cast<const uint8_t*>(a.cache) +
                                       ((page * a.kv_heads + kvh) * (int64_t)page_tiles + (at - in * page_tiles)) * kv_tile_bytes(NG);
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint16_t b = *reinterpret_cast<const uint16_t*>(there + kv_vs_off(NG) + kv_scale(t % kKvTile, g, NG));
                    if ((b & 0x7C00) == 0x7C00 && kt + t <= lim) o[g] += __builtin_nanf("");
                }
            }
        }
    };
    for (int tile = first; tile < last; tile += 4) {
        step(tile, sa, sb, kb1, kb0, vb0, vb1);
        if (tile + 2 < last) step(tile + 2, sb, sa, kb0, kb1, vb1, vb0);
    }
    if (bad) l = __builtin_nanf("");
    l += __shfl_xor(l, 32);
    if (wrow + ln >= rows) return;
    if (a.splits > 1) {
        float* part = a.part + (((int64_t)(seq * a.kv_heads + kvh) * a.blocks + block) * a.splits + split) * kRows * (D + 4) +
                      (32 * wave + ln) * (D + 4);
#pragma unroll
        for (int d = 0; d < ND; ++d)
#pragma unroll
            for (int i = 0; i < 16; i += 4)
                *reinterpret_cast<float4v*>(part + 32 * d + 2 * i + 4 * h) = float4v{o[d][i], o[d][i + 1], o[d][i + 2], o[d][i + 3]};
        if (h == 0) *reinterpret_cast<float2*>(part + D) = make_float2(m, l);
        return;
    }
    const float inv = 1.0f / l;
    typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (sp.q0 + qi) * a.ld_out + (int64_t)head * D;
#pragma unroll
    for (int d = 0; d < ND; ++d)
#pragma unroll
        for (int i = 0; i < 16; i += 4) {                            // columns 32 d + 2 i + 4 h and the next three
            typename O::Elem y[4];
#pragma unroll
            for (int e = 0; e < 4; ++e) y[e] = O::one(lim < 0 ? 0.f : l == 0.f ? __builtin_nanf("") : o[d][i + e] * inv);
            __builtin_memcpy(__builtin_assume_aligned(out + 32 * d + 2 * i + 4 * h, 4 * sizeof(y[0])), y, sizeof(y));
        }
}

// A row's parts of all splits, joined in their order, four columns a thread. A
// workgroup has D / 4 threads for each of its rows (few splits), or eight (of
// 128) such sets on the splits of one row, which meet in LDS.
template <int OUT, int NG, bool ONE>
__global__ void __launch_bounds__(256) attn_chunk_join_kernel(ChunkArgs a, int kRows) {
    using O = Val<OUT>;
    constexpr int D = 32 * NG, kCols = D / 4, kSets = 256 / kCols;
    __shared__ __attribute__((aligned(16))) float vals[ONE ? kSets : 1][D];
    __shared__ float sums[kSets];
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    const int col = threadIdx.x % kCols, set = threadIdx.x / kCols;
    const uint32_t per = ONE ? (uint32_t)kRows : (uint32_t)((kRows + kSets - 1) / kSets);   // workgroups of a block
    const uint32_t unit = blockIdx.x / per;                          // block of a key head of a sequence
    const int r = (int)(blockIdx.x - unit * per) * (ONE ? 1 : kSets) + (ONE ? 0 : set);
    const uint32_t id = unit / (uint32_t)a.blocks;
    const int block = (int)(unit % (uint32_t)a.blocks), kvh = (int)(id % (uint32_t)a.kv_heads), seq = (int)(id / (uint32_t)a.kv_heads);
    Span sp;
    if (!sp.read(a, seq) || sp.bad) return;
    const int row0 = block * kRows, row = row0 + r;
    if (row >= sp.nq * group || r >= kRows) return;                  // where ONE the whole workgroup
    const int tiles = (sp.keys(row0 + kRows - 1, group) + kKvTile - 1) / kKvTile;
    const int share = (int)a.share, used = tiles <= share ? 1 : (tiles + share - 1) / share;
    const int64_t step = (int64_t)kRows * (D + 4);
    const float* p = a.part + (int64_t)unit * a.splits * step + r * (D + 4);
    float mm = -kInf;
    if constexpr (ONE) {
        for (int s = threadIdx.x & 63; s < used; s += 64) mm = __builtin_fmaxf(mm, p[s * step + D]);
#pragma unroll
        for (int i = 1; i < 64; i <<= 1) mm = __builtin_fmaxf(mm, __shfl_xor(mm, i));
    } else {
        for (int s = 0; s < used; ++s) mm = __builtin_fmaxf(mm, p[s * step + D]);
    }
    const float base = mm == -kInf ? 0.f : mm;
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int s = ONE ? set : 0; s < used; s += ONE ? kSets : 1) {
        const float4 x = *reinterpret_cast<const float4*>(p + s * step + 4 * col);
        const float2 ml = *reinterpret_cast<const float2*>(p + s * step + D);
        const float f = __builtin_amdgcn_exp2f(ml.x - base);
        sum = __builtin_fmaf(f, ml.y, sum);
        val.x = __builtin_fmaf(f, x.x, val.x);
        val.y = __builtin_fmaf(f, x.y, val.y);
        val.z = __builtin_fmaf(f, x.z, val.z);
        val.w = __builtin_fmaf(f, x.w, val.w);
    }
    if constexpr (ONE) {
        *reinterpret_cast<float4*>(&vals[set][4 * col]) = val;
        if (col == 0) sums[set] = sum;
        __syncthreads();
        if (set) return;
#pragma unroll
        for (int i = 1; i < kSets; ++i) {
            const float4 x = *reinterpret_cast<const float4*>(&vals[i][4 * col]);
            val.x += x.x;
            val.y += x.y;
            val.z += x.z;
            val.w += x.w;
            sum += sums[i];
        }
    }
    const int i = row / group;
    typename O::Elem* out = static_cast<typename O::Elem*>(a.out) + (sp.q0 + i) * a.ld_out + (int64_t)(kvh * group + row - i * group) * D;
    const bool none = sp.past + i < 0;
    const typename O::Elem y[4] = {O::one(none ? 0.f : val.x / sum), O::one(none ? 0.f : val.y / sum),
                                   O::one(none ? 0.f : val.z / sum), O::one(none ? 0.f : val.w / sum)};
    __builtin_memcpy(__builtin_assume_aligned(out + 4 * col, 4 * sizeof(y[0])), y, sizeof(y));
}

// R: column tiles of a workgroup, or minus the waves of 32 rows of one that works
// on unpacked keys.
template <int TYPE, int OUT, int NG, int R>
hipError_t launch_one(const ChunkArgs& a, hipStream_t stream) {
    constexpr int kRows = R > 0 ? 16 * R : -32 * R;
    const int64_t units = a.seqs * a.kv_heads * a.blocks;
    const unsigned grid = (unsigned)(units * a.splits);
    if constexpr (R > 0) {
        attn_chunk_kernel<TYPE, OUT, NG, R><<<grid, 64 * kWaves, 0, stream>>>(a);
    } else {
        attn_chunk_unpack_kernel<NG><<<(unsigned)(a.seqs * a.kv_heads * a.steps), 64 * unpack_waves(NG), 0, stream>>>(a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
        attn_chunk_rows_kernel<TYPE, OUT, NG, -R><<<grid, -64 * R, 0, stream>>>(a);
    }
    if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.splits == 1) return e;
    constexpr int kSets = 256 / (8 * NG);
    if (a.splits > 8)
        attn_chunk_join_kernel<OUT, NG, true><<<(unsigned)(units * kRows), 256, 0, stream>>>(a, kRows);
    else
        attn_chunk_join_kernel<OUT, NG, false><<<(unsigned)(units * ((kRows + kSets - 1) / kSets)), 256, 0, stream>>>(a, kRows);
    return hipGetLastError();
}

template <int TYPE, int OUT>
hipError_t launch_typed(const ChunkArgs& a, hipStream_t stream) {
    const auto run = [&](auto ng) {
        constexpr int kN = decltype(ng)::value;
        switch (a.tiles) {
            case -8:
                if constexpr (kN == 4) return launch_one<TYPE, OUT, kN, -8>(a, stream);
                return hipErrorInvalidValue;
            case -4: return launch_one<TYPE, OUT, kN, -4>(a, stream);
            case 1: return launch_one<TYPE, OUT, kN, 1>(a, stream);
            case 2: return launch_one<TYPE, OUT, kN, 2>(a, stream);
            default:
                if constexpr (kN <= 4) return a.tiles == 3 ? launch_one<TYPE, OUT, kN, 3>(a, stream) : launch_one<TYPE, OUT, kN, 4>(a, stream);
                return hipErrorInvalidValue;
        }
    };
    switch (a.head_dim) {
        case 64: return run(Int<2>{});
        case 128: return run(Int<4>{});
        case 256: return run(Int<8>{});
        default: return hipErrorInvalidValue;
    }
}

}  // namespace

// Rows of a workgroup.
static int64_t block_rows(const ChunkArgs& a) { return a.tiles > 0 ? 16 * a.tiles : -32 * a.tiles; }

static size_t part_bytes(const ChunkArgs& a) {
    if (a.splits == 1) return 0;
    return sizeof(float) * (size_t)(a.seqs * a.kv_heads * a.blocks * a.splits * block_rows(a)) * (size_t)(a.head_dim + 4);
}
static size_t held_bytes(const ChunkArgs& a) {
    return a.tiles < 0 ? (size_t)(a.seqs * a.kv_heads * a.steps) * (size_t)(256 * a.head_dim) : 0;
}

// How the rows are cut (a.tiles) and the keys split, by the steps of 64 tokens (some
// 2 us) that the slowest CU comes to, where every workgroup has as many keys as the
// longest sequence, four more for its start and end, and the parts, written and
// read at 4 TB/s.
// Two workgroups of four waves on a CU take a fourteenth longer than one of eight,
// one alone two thirds of that.
static int64_t cut(ChunkArgs* a, int64_t rows, int64_t slots, int64_t most) {
    a->blocks = (rows + block_rows(*a) - 1) / block_rows(*a);
    const int64_t units = a->seqs * a->kv_heads * a->blocks;
    const int64_t part = a->seqs * a->max_q * a->q_heads * (a->head_dim + 4);     // floats
    int64_t best = 0;
    for (int64_t s = 1; s <= most && (s == 1 || units * s <= 4 * slots); ++s) {
        const int64_t each = (a->steps + s - 1) / s, over = units * s % slots;
        const int64_t rounds = slots == 256 ? (units * s + 255) / 256 * 14
                                            : units * s / slots * 15 + (over == 0 ? 0 : over <= 256 ? 10 : 15);
        const int64_t cost = rounds * (each + 4) + (s > 1 ? 14 * (3 + s * part / 1000000) : 0);
        if (best && cost >= best) continue;
        best = cost;
        a->splits = s;
    }
    return best;
}

bool plan_attn_chunk(ChunkArgs* a) {
    const int64_t rows = a->max_q * (a->q_heads / a->kv_heads), keys = (a->max_len + kKvTile - 1) / kKvTile;
    const bool wide = a->head_dim == 256;
    a->steps = (keys + 1) / 2;
    a->tiles = -4;
    if (rows >= kHeldRows && a->seqs * a->kv_heads * a->steps < (int64_t)1 << 22 && held_bytes(*a) <= kHeldMost) {
        const int64_t cost4 = cut(a, rows, wide ? 256 : 512, 16);
        if (a->head_dim == 128) {
            // eight waves to a copy of the keys where that leaves no CU empty: 2048 tokens
            // after 32768 1059 us, with four 1163; 8 of 350 after 2200 161 and 140
            const int64_t splits4 = a->splits, blocks4 = a->blocks;
            a->tiles = -8;
            if (cut(a, rows, 256, 16) > cost4) a->tiles = -4, a->splits = splits4, a->blocks = blocks4;
        }
        a->share = 2 * ((a->steps + a->splits - 1) / a->splits);
    } else {
        a->tiles = rows <= 16 ? 1 : rows <= 32 || wide ? 2 : rows <= 48 ? 3 : 4;     // 256-wide: two fill the registers
        a->blocks = (rows + block_rows(*a) - 1) / block_rows(*a);
        const int64_t units = a->seqs * a->kv_heads * a->blocks;
        // two workgroups a CU; twice as many where sequences may end early (1536: 32
        // ragged sequences 62 us, not 71, 32 equal ones of 4000 42, not 37)
        int64_t splits = units >= 512 ? 1 : ((units >= a->kv_heads * 2 ? 1024 : 512) + units - 1) / units;
        // two tiles a wave at least: 5 tokens after 4000, 32 heads over 8: 12.7 us in a
        // graph, 16.1 with four; of 8 sequences after 100 to 4000: 21.1, 24.8 with one
        const int64_t most = (keys + 2 * kWaves - 1) / (2 * kWaves);
        splits = splits < most ? splits : most;
        a->share = splits > 1 ? (keys + splits - 1) / splits : keys;
    }
    a->share = a->share > 0 ? a->share : 1;
    a->splits = keys > a->share ? (keys + a->share - 1) / a->share : 1;
    const int64_t units = a->seqs * a->kv_heads * a->blocks;
    if (units >= (int64_t)1 << 22) return false;                     // a launch has fewer than 2^32 threads
    a->sorted = a->seqs > 1 && a->seqs <= 64;
    a->per_page = ((uint64_t)1 << 36) / ((uint64_t)a->page_tokens / kKvTile) + 1;
    return true;
}

size_t attn_chunk_scratch(const ChunkArgs& a) {
    return (part_bytes(a) + 255) / 256 * 256 + held_bytes(a) + (a.tiles < 0 ? sizeof(int32_t) * (size_t)(a.seqs * a.kv_heads * a.steps) : 0);
}

hipError_t launch_attn_chunk(ChunkArgs a, float* scratch, hipStream_t stream) {
    a.part = scratch;
    a.held = reinterpret_cast<char*>(scratch) + (part_bytes(a) + 255) / 256 * 256;
    a.held_flags = reinterpret_cast<int32_t*>(static_cast<char*>(a.held) + held_bytes(a));
    if (a.type == kTypeBF16)
        return a.out_type == kTypeF32 ? launch_typed<kTypeBF16, kTypeF32>(a, stream)
                                      : launch_typed<kTypeBF16, kTypeBF16>(a, stream);
    return a.out_type == kTypeF32 ? launch_typed<kTypeF16, kTypeF32>(a, stream)
                                  : launch_typed<kTypeF16, kTypeF16>(a, stream);
}

}  // namespace frq
