// Attention of one query token per sequence against the 4-bit paged cache
// (frq_kv4.h):
//   S[h, t] = scale q_h . k_t,  t < len;   out_h = sum_t softmax(S)[h, t] v_t.
//
// The cache is read as it is held, once for up to eight query heads that share
// a key head. Both products run on v_mfma_f32_16x16x32_f16 with fp32 precision:
// the codes c - 8 are exact fp16 integers, and q and the softmax weights go in
// as two fp16 numbers each, rows 2h and 2h + 1 of the product: the value and the
// rest, 22 bits together. The rests stand 2^12 higher and their rows' sums are
// taken back at the end, so that the parts hold small numbers too: fp16 steps of
// 2^-24 become 2^-36 (without that, tokens at 2^-24 of a large one's weight were
// off by a tenth each). q is put under a power of two per head that brings its
// largest element to [2^13, 2^14). A block of K has its scale on the product of
// one instruction; the scale of V goes into the weights. Each group of 32
// channels has sums of its own and so a power of two of its own, 2^(5 - E), 2^E
// twice to four times the largest |scale| of the first tile's tokens in the
// group: a weight times a scale is kept to 22 bits, or to 2^-40 of the reference's
// weight times the largest scale where that is coarser.
//
// A wave takes 32 tokens a step. S = q K^T gives a lane one token of each half
// and both numbers of two heads, so scores, weights and their scales need no
// other lane; the weights pass through LDS, a wave's own part of it, to stand
// as the second product's operand (transposing reads). The reference that the
// exponentials are taken from, and E, are those of a wave's first tile. A tile
// whose scores pass the reference by more than 2^8, or whose scales reach
// 2^(E + 1) in a group, ends the run: sums and reference go to LDS, where runs
// and later waves are joined under the larger one, and the wave starts anew from
// that tile. So the loop has no rescaling and no maximum over lanes. Two tiles
// are on their way while one is worked on, 9.2 KB a wave at 128 channels.
//
// The tiles of all sequences and key heads, one after another, are shared out
// evenly over the workgroups, whatever the lengths are; the four waves of a
// workgroup take its tiles in turn and meet in LDS. A row that several
// workgroups worked on is joined, in their order, by a second, small kernel
// (joined by the last workgroup to finish instead, the release between XCDs
// costs what the launch does: 131072 tokens 42 us, 64 ragged sequences the same).
// Short sequences have one workgroup per sequence and key head, and no joining.
//
// 131072 tokens of 8 key heads of 128, 32 query heads: 37 us and 4.6 for the
// joining, 151 MB at 4.1 TB/s (reads alone reach 6.1): 4 us until the first tile
// is there, 2 for the end, the rest at 4.9 TB/s. 64 sequences of 1 to 8192
// tokens: 73 and 6 us, 4.3 TB/s; vector instructions (unpacking, weights) are
// then issued 55 % of the time, the matrix cores work 11 %. 16 sequences of
// 2000 to 4096, 4 key heads: 16 and 4 us, of which the loads are a third. Powers
// of two by channel group and the raised rests are 24 of a tile's 144 vector
// instructions, 2 us of the first case; 256-wide heads, one wave to a SIMD, take
// a tenth longer by them (32768 tokens, 8 heads over 4: 34.7 us against 31.2).
// The comparisons further down were measured without them.
#include "frq_kernels.h"
#include "frq_kv4.h"

namespace frq {
namespace {

using half2v = _Float16 __attribute__((ext_vector_type(2)));
using half8v = _Float16 __attribute__((ext_vector_type(8)));
using float4v = float __attribute__((ext_vector_type(4)));

constexpr int kWaves = 4;
constexpr int kPad = 16;               // see Line
constexpr int kShareMin = 8;           // places of a workgroup, two tiles for each wave
// Tiles up to which a workgroup takes all of a pair and nothing is joined: with
// few pairs (two key heads, 22 tiles: 7.9 us against 9.3; 63 tiles: 22 against
// 13), and with at least one for every workgroup (64 sequences of 8 key heads,
// up to 63 tiles: 28.7 against 33.1; up to 256: 104 against 79).
constexpr int kWhole = 28, kWholeMany = 64;
// Two workgroups on each of 256 CUs at 128 channels (34 KB, 193 registers a
// lane); at 64 a CU would hold three, at 256 it holds one, and they run in turn.
constexpr int kGroups = 512;
constexpr float kLog2e = 1.4426950408889634f;
constexpr float kRest = 4096;          // the rests stand 2^12 higher than the values
constexpr int kTop = 5;                // of the exponents that weights stand under, see the head of the file

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

// kRest / p, p a power of two: exponents (127 + 12 - e) + (127 + e) are 254 + 12.
__device__ __forceinline__ float over_pow2(float p) {
    return __builtin_bit_cast(float, ((254u + 12u) << 23) - __builtin_bit_cast(uint32_t, p));
}

// The largest of x over the 16 lanes of a row.
__device__ __forceinline__ float row_max(float x) {
#pragma unroll
    for (int i = 1; i <= 8; i <<= 1) x = __builtin_fmaxf(x, __shfl_xor(x, i));
    return x;
}

// Codes and scales of a tile as a lane holds them: words p of the codes, and
// of the scales words u NG/2 + g/2.
template <int NG>
struct Half {
    uint32_t code[2 * NG], scale[NG];
    __device__ __forceinline__ void load(const uint8_t* codes, const uint8_t* scales, int lane) {
#pragma unroll
        for (int p = 0; p < 2 * NG; p += 4) {
            const uint4 x = *reinterpret_cast<const uint4*>(codes + kv_word(p, lane));
            code[p] = x.x; code[p + 1] = x.y; code[p + 2] = x.z; code[p + 3] = x.w;
        }
        scales += kv_scale(lane & 15, 0, NG);
#pragma unroll
        for (int p = 0; p < NG; p += 2) {
            const uint2 x = *reinterpret_cast<const uint2*>(scales + 4 * p);
            scale[p] = x.x; scale[p + 1] = x.y;
        }
    }
    __device__ __forceinline__ _Float16 scale_of(int u, int g) const {
        const int at = u * NG + g;
        return half_of(scale[at / 2], at & 1);
    }
};
using lds_bytes = __attribute__((address_space(3))) char*;
using short4v = short __attribute__((ext_vector_type(4)));
using uint2v = uint32_t __attribute__((ext_vector_type(2)));

// Lengths and pages do not change under the kernel: read through the constant
// address space, so that uniform reads are scalar ones, which neither wait for
// the tiles that are on their way nor make what follows a vector value.
using const_ints = const __attribute__((address_space(4))) int32_t*;
__device__ __forceinline__ const_ints constant(const int32_t* p) { return (const_ints)(uintptr_t)p; }

// The length that counts: 0 for none, -1 for one that is not what the caller
// said (longer than max_len, or no cache to hold it), whose row is NaN.
__device__ __forceinline__ int length_of(const DecodeArgs& a, int b) {
    const int len = constant(a.lens)[b];
    return len <= 0 ? 0 : len > a.max_len || a.pages == 0 ? -1 : len;
}
__device__ __forceinline__ int tiles_in(int len) { return len > 0 ? (int)((uint32_t)(len + kKvTile - 1) / kKvTile) : 0; }

__device__ __forceinline__ int places_in(int len) { return len > 0 ? tiles_in(len) + kPad : 0; }

// x summed over the lanes up to and with this one.
__device__ __forceinline__ int wave_scan(int x) {
    x += __builtin_amdgcn_update_dpp(0, x, 0x111, 0xF, 0xF, true);   // within rows of 16
    x += __builtin_amdgcn_update_dpp(0, x, 0x112, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x114, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x118, 0xF, 0xF, true);
    x += __builtin_amdgcn_update_dpp(0, x, 0x142, 0xA, 0xF, false);  // row 0 into 1, 2 into 3
    x += __builtin_amdgcn_update_dpp(0, x, 0x143, 0xC, 0xF, false);  // rows 0, 1 into 2, 3
    return x;
}

// What every workgroup works out of the lengths. The pairs (a key head, eight
// query heads) of all sequences stand in one line, a sequence's side by side,
// each as many places long as it has tiles and kPad more at its front: what
// starting and ending a pair costs in tiles' time (64 sequences of 1 .. 8192
// tokens, 8 key heads: 117 us without, 93 with 8, 87 with 16 or 24). The lengths
// of 64 sequences at a time are in the lanes. The host keeps the whole line below 2^31.
struct Line {
    int total, share;   // places of all, and of a workgroup
    int from;           // the sequence of lane 0
    int len, upto;      // the lane's length, and the places of a pair up to its end from `from` on
    __device__ __forceinline__ void read(const DecodeArgs& a, int at, int lane) {
        from = at;
        len = at + lane < a.batch ? length_of(a, at + lane) : 0;
        upto = wave_scan(places_in(len));
    }
    __device__ __forceinline__ int all() const { return __builtin_amdgcn_readlane(upto, 63); }
    __device__ __forceinline__ int before(int k) const { return k ? __builtin_amdgcn_readlane(upto, k - 1) : 0; }
    __device__ __forceinline__ void open(const DecodeArgs& a, int pairs, int lane) {
        read(a, 0, lane);
        int sum = all();
        for (int at = 64; at < a.batch; at += 64) {
            read(a, at, lane);
            sum += all();
        }
        if (a.batch > 64) read(a, 0, lane);
        total = sum * pairs;
        share = (int)(((uint32_t)total + (uint32_t)a.groups - 1) / (uint32_t)a.groups);
        share = share < kShareMin ? kShareMin : share;
    }
};

template <int TYPE, int NG>
__global__ void __launch_bounds__(64 * kWaves, NG == 8 ? 1 : 2) attn_decode_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    constexpr int D = 32 * NG, kTile = kv_tile_bytes(NG), kRow = D + 8;   // 16 banks from the row of the next j
    // the waves' weights [group][token][row], and their results
    __shared__ __attribute__((aligned(16))) char sh_p[kWaves * NG * 1024];
    __shared__ float sh_o[kWaves * 8 * kRow], sh_m[kWaves][8], sh_l[kWaves][8];

    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int n = lane & 15, j = lane >> 4;
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads);
    const int chunks = (group + 7) / 8, pairs = (int)a.kv_heads * chunks;
    const uint32_t page_tiles = (uint32_t)a.page_tokens / kKvTile;
    const int64_t page_bytes = a.kv_heads * (int64_t)page_tiles * kTile;

    // this workgroup's tiles: [at, end) of the line, or all of one pair
    Line line;
    int at = 0, end = 0, begin = 0, k = 0, b, pair, first = 0, last = 0, len, tiles;
    const bool shared = a.groups != 0;
    if (!shared) {
        b = (int)(blockIdx.x / (uint32_t)pairs);
        pair = (int)(blockIdx.x - (uint32_t)b * (uint32_t)pairs);
        len = length_of(a, b);
        last = tiles = tiles_in(len);
    } else {
        line.open(a, pairs, lane);
        at = (int)blockIdx.x * line.share;
        if ((uint32_t)at >= (uint32_t)line.total) return;
        end = line.total - at < line.share ? line.total : at + line.share;
        // the sequence that `at` is in: lane k of those in hand
        while (begin + line.all() * pairs <= at) {
            begin += line.all() * pairs;
            line.read(a, line.from + 64, lane);
        }
        k = (int)__builtin_ctzll(__builtin_amdgcn_ballot_w64(begin + line.upto * pairs > at));
    }
    const lds_bytes sp = (lds_bytes)sh_p + wave * (NG * 1024);
    // a token's row of weights, its pieces in an order by which half a wave's
    // writes touch every bank once
    const int row = lane >> 2;
    const lds_bytes sp_to = sp + n * 32 + (j ^ (n >> 3 << 1)) * 8, sp_from = sp + row * 32 + ((lane & 3) ^ (row >> 3 << 1)) * 8;

    for (;;) {
        if (shared) {                                                // tiles [first, last) of a pair of sequence b
            b = line.from + k;
            len = __builtin_amdgcn_readlane(line.len, k);
            tiles = tiles_in(len);
            const int in = at - begin - line.before(k) * pairs, places = tiles + kPad;
            pair = (int)((uint32_t)in / (uint32_t)places);
            first = in - pair * places - kPad;
            last = end - at < tiles - first ? first + (end - at) : tiles;
            at += last - first;
            if (last <= 0) break;                                    // all of it padding
            first = first > 0 ? first : 0;
        }
        bool bad = len < 0;
        const int kvh = chunks == 1 ? pair : pair / chunks, hc = chunks == 1 ? 0 : pair - kvh * chunks;
        const int rows = group - 8 * hc < 8 ? group - 8 * hc : 8;    // query heads here
        const const_ints table = constant(a.table) + (int64_t)b * a.ld_table;
        const uint8_t* heads = static_cast<const uint8_t*>(a.cache) + (int64_t)kvh * page_tiles * kTile;
        // Pages are looked up a step before their tile is asked for. Past the last
        // tile that one is asked for again: with loads that may not have been
        // issued in flight, the compiler would wait for the ones after them too.
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
        int tile = first + wave;
        Half<NG> k0, v0, k1, v1;                                     // this tile and the wave's next one
        auto fetch_k = [&](Half<NG>& k, const uint8_t* t) { k.load(t, t + kv_ks_off(NG), lane); };
        auto fetch_v = [&](Half<NG>& v, const uint8_t* t) { v.load(t + kv_vc_off(NG), t + kv_vs_off(NG), lane); };
        int page = 0;
        auto start = [&]() __attribute__((always_inline)) {
            const int p0 = look_up(tile), p1 = look_up(tile + kWaves);
            page = look_up(tile + 2 * kWaves);
            const uint8_t* t0 = address(tile, p0);
            const uint8_t* t1 = address(tile + kWaves, p1);
            fetch_k(k0, t0);                                         // in the order of their use
            __builtin_amdgcn_sched_barrier(0);
            fetch_v(v0, t0);
            __builtin_amdgcn_sched_barrier(0);
            fetch_k(k1, t1);
            __builtin_amdgcn_sched_barrier(0);
            fetch_v(v1, t1);
            __builtin_amdgcn_sched_barrier(0);
        };
        if (tile < last) start();

        // q: row n holds head n / 2, the value or (n odd) the rest
        half8v qf[NG];
        float rs;
        {
            const int row = n >> 1;
            float x[NG][8];
            uint32_t top = 0;                                        // bits of the largest |q|; inf and NaN above all
            const typename T::Elem* qp = static_cast<const typename T::Elem*>(a.q) + (int64_t)b * a.ld_q +
                                         ((int64_t)kvh * group + 8 * hc + (row < rows ? row : 0)) * D;
#pragma unroll
            for (int g = 0; g < NG; ++g) T::load8(qp + 32 * g + 8 * j, x[g]);
#pragma unroll
            for (int g = 0; g < NG; ++g)
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const uint32_t m = __builtin_bit_cast(uint32_t, x[g][c]) & 0x7FFFFFFFu;
                    top = top > m ? top : m;
                }
            uint32_t other = __shfl_xor(top, 16);
            top = top > other ? top : other;
            other = __shfl_xor(top, 32);
            top = top > other ? top : other;
            const int up = top ? 140 - (int)(top >> 23) : 0;         // the largest to [2^13, 2^14)
            const float part = n & 1 ? -kRest : 0.f, gain = n & 1 ? kRest : 1.f;
#pragma unroll
            for (int g = 0; g < NG; ++g) {
#pragma unroll
                for (int c = 0; c < 8; ++c) {
                    const float y = __builtin_ldexpf(x[g][c], up);
                    const _Float16 hi = (_Float16)y;
                    qf[g][c] = (_Float16)__builtin_fmaf((float)hi, part, y * gain);
                }
            }
            rs = top >= 0x7F800000u ? __builtin_nanf("") : __builtin_ldexpf(a.scale * kLog2e, -up);
        }
        // of the lane's two heads 2j and 2j + 1: rows 4j .. 4j + 3 of both products
        const float rs2[2] = {__shfl(rs, 4 * j), __shfl(rs, 4 * j + 2)};
        // what the lane's heads have in LDS: reference and sum of weights
        float held_ref[2] = {-__builtin_inff(), -__builtin_inff()}, held_l[2] = {0.f, 0.f};
        bool held = false;

        while (tile < last) {
        float ref[2] = {-__builtin_inff(), -__builtin_inff()}, l[2] = {0.f, 0.f};
        float under[NG];                                             // 2^(kTop - E) kRest of each group
        uint32_t cap[NG / 2];                                        // the largest |scale| bits that fit, of two groups
#pragma unroll
        for (int g = 0; g < NG; ++g) under[g] = 1.f;
#pragma unroll
        for (int p = 0; p < NG / 2; ++p) cap[p] = 0;
        int fresh = 1;
        float4v o[2 * NG];
#pragma unroll
        for (int i = 0; i < 2 * NG; ++i) o[i] = float4v{0, 0, 0, 0};
        if (held) start();                                           // once more from this tile

        // one tile; false if it does not fit the reference
        auto step = [&](Half<NG>& k, Half<NG>& v) __attribute__((always_inline)) {
            const uint8_t* next = address(tile + 2 * kWaves, page);
            page = look_up(tile + 3 * kWaves);
            // scores of tokens n and 16 + n for heads 2j, 2j + 1
            float s[2][2];
            float4v c[2][NG];
#pragma unroll
            for (int u = 0; u < 2; ++u)
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t w = k.code[u * NG + g];
                    const half8v kf = join(low_pair(w), high_pair(w), low_pair(w >> 8), high_pair(w >> 8));
                    c[u][g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(qf[g], kf, float4v{0, 0, 0, 0}, 0, 0, 0);
                    // products under way before one is waited for, and no more
                    // operands at a time than the registers have room for
                    if ((u * NG + g) % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                }
#pragma unroll
            for (int u = 0; u < 2; ++u) {
                float acc[4] = {0.f, 0.f, 0.f, 0.f};
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const float d = (float)k.scale_of(u, g);
#pragma unroll
                    for (int i = 0; i < 4; ++i) acc[i] = __builtin_fmaf(c[u][g][i], d, acc[i]);
                }
                s[u][0] = __builtin_fmaf(acc[1], 1 / kRest, acc[0]) * rs2[0];
                s[u][1] = __builtin_fmaf(acc[3], 1 / kRest, acc[2]) * rs2[1];
            }
            fetch_k(k, next);                              // these registers are free again
            const int left = len - tile * kKvTile;                   // valid tokens from here
            if (__builtin_expect(left < kKvTile, 0)) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    if (16 * u + n >= left) {
                        s[u][0] = s[u][1] = -__builtin_inff();
#pragma unroll
                        for (int p = 0; p < NG / 2; ++p) v.scale[u * (NG / 2) + p] = 0;
                    }
                }
            }
            auto weigh = [&]() __attribute__((always_inline)) {
#pragma unroll
                for (int u = 0; u < 2; ++u) {
                    const float p0 = __builtin_amdgcn_exp2f(s[u][0] - ref[0]), p1 = __builtin_amdgcn_exp2f(s[u][1] - ref[1]);
                    l[0] += p0;
                    l[1] += p1;
#pragma unroll
                    for (int g = 0; g < NG; ++g) {
                        const float d = __builtin_fmaf((float)v.scale_of(u, g), under[g], 0.f), y0 = p0 * d, y1 = p1 * d;
                        const _Float16 h0 = (_Float16)__builtin_fmaf(y0, 1 / kRest, 0.f), h1 = (_Float16)__builtin_fmaf(y1, 1 / kRest, 0.f);
                        const _Float16 r0 = (_Float16)__builtin_fmaf((float)h0, -kRest, y0), r1 = (_Float16)__builtin_fmaf((float)h1, -kRest, y1);
                        const half2v x = {h0, r0}, y = {h1, r1};
                        *(__attribute__((address_space(3))) uint2v*)(sp_to + g * 1024 + u * 512) =
                            uint2v{__builtin_bit_cast(uint32_t, x), __builtin_bit_cast(uint32_t, y)};
                    }
                }
                __builtin_amdgcn_fence(__ATOMIC_RELEASE, "wavefront");
                __builtin_amdgcn_wave_barrier();
                __builtin_amdgcn_fence(__ATOMIC_ACQUIRE, "wavefront");
                using tr = __attribute__((address_space(3))) short4v*;
                uint2v px[NG], py[NG];
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    px[g] = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(sp_from + g * 1024)));
                    py[g] = __builtin_bit_cast(uint2v, __builtin_amdgcn_ds_read_tr16_b64_v4i16((tr)(sp_from + g * 1024 + 512)));
                }
                __builtin_amdgcn_sched_barrier(0);                       // V is unpacked while they come
#pragma unroll
                for (int g = 0; g < NG; ++g) {
                    const uint32_t w0 = v.code[2 * g], w1 = v.code[2 * g + 1];
                    const half8v va = join(low_pair(w0), low_pair(w0 >> 8), low_pair(w1), low_pair(w1 >> 8));
                    const half8v vb = join(high_pair(w0), high_pair(w0 >> 8), high_pair(w1), high_pair(w1 >> 8));
                    const half8v pf = join(pair_of(px[g][0]), pair_of(px[g][1]), pair_of(py[g][0]), pair_of(py[g][1]));
                    o[2 * g] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, va, o[2 * g], 0, 0, 0);
                    o[2 * g + 1] = __builtin_amdgcn_mfma_f32_16x16x32_f16(pf, vb, o[2 * g + 1], 0, 0, 0);
                    if (g % 2 == 1) __builtin_amdgcn_sched_barrier(0);
                }
                fetch_v(v, next);
            };
            // a score 2^8 past its reference, or a scale past its group's E?
            using us2 = unsigned short __attribute__((ext_vector_type(2)));
            us2 big[NG / 2], over = {0, 0};
#pragma unroll
            for (int p = 0; p < NG / 2; ++p) {
                big[p] = __builtin_elementwise_max(__builtin_bit_cast(us2, v.scale[p] & 0x7FFF7FFFu),
                                                   __builtin_bit_cast(us2, v.scale[NG / 2 + p] & 0x7FFF7FFFu));
                over |= __builtin_elementwise_sub_sat(big[p], __builtin_bit_cast(us2, cap[p]));
            }
            const float t0 = __builtin_fmaxf(s[0][0], s[1][0]), t1 = __builtin_fmaxf(s[0][1], s[1][1]);
            asm("" : "+s"(fresh));                                 // no copy of the step for the first tile
            if (__builtin_expect(fresh != 0, 0)) {
#pragma unroll
                for (int p = 0; p < NG / 2; ++p) {
                    us2 top = {0, 0};                                // of the scales that are numbers
#pragma unroll
                    for (int u = 0; u < 2; ++u) {
                        const us2 x = __builtin_bit_cast(us2, v.scale[u * (NG / 2) + p] & 0x7FFF7FFFu);
                        top = __builtin_elementwise_max(top, (us2){x[0] < 0x7C00 ? x[0] : (unsigned short)0, x[1] < 0x7C00 ? x[1] : (unsigned short)0});
                    }
#pragma unroll
                    for (int i = 1; i <= 8; i <<= 1)                 // every row of lanes holds all tokens
                        top = __builtin_elementwise_max(top, __builtin_bit_cast(us2, __shfl_xor(__builtin_bit_cast(uint32_t, top), i)));
                    const uint32_t w = (uint32_t)__builtin_amdgcn_readfirstlane(__builtin_bit_cast(int, top));
                    uint32_t caps[2];
#pragma unroll
                    for (int i = 0; i < 2; ++i) {
                        // 2^E from twice to four times the largest, scales below 2^(E + 1) fit
                        const uint32_t h = i ? w >> 16 : w & 0xFFFFu;
                        const int e = h ? __builtin_amdgcn_frexp_expf((float)half_of(h, 0)) + 1 : -22;
                        const int ev = __builtin_amdgcn_readfirstlane(e);
                        under[2 * p + i] = pow2(kTop + 12 - ev);
                        caps[i] = ev >= 15 ? 0x7BFFu : ev >= -15 ? ((uint32_t)(ev + 16) << 10) - 1 : (1u << (ev + 25)) - 1;
                    }
                    cap[p] = caps[0] | caps[1] << 16;
                }
                // where all scores are -inf, below everything, so that they count nothing
                ref[0] = __builtin_fmaxf(row_max(t0), -3.4028235e38f);
                ref[1] = __builtin_fmaxf(row_max(t1), -3.4028235e38f);
                fresh = 0;
            } else {
                const bool past = (int)(t0 - ref[0] > 8.f) | (int)(t1 - ref[1] > 8.f) | (int)(__builtin_bit_cast(uint32_t, over) != 0);
                if (__builtin_expect(__builtin_amdgcn_ballot_w64(past) != 0, 0)) return false;
            }
            weigh();
            __builtin_amdgcn_wave_barrier();
            tile += kWaves;
            return true;
        };
        // Of two workgroups on a CU the one that came first goes first and is
        // done early (131072 tokens, 8 key heads: after 26 us, the other after
        // 34); the later half of the grid gets the higher priority instead,
        // which evens them out a little (41.1 us against 40.1 together).
        if (shared && blockIdx.x >= gridDim.x / 2) __builtin_amdgcn_s_setprio(1);
        while (tile < last && step(k0, v0) && tile < last && step(k1, v1)) {
        }
        // into LDS, under the larger of the references
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const float both = __builtin_fmaxf(held_ref[i], ref[i]), base = both == -__builtin_inff() ? 0.f : both;
            const float fo = __builtin_amdgcn_exp2f(held_ref[i] - base), fn = __builtin_amdgcn_exp2f(ref[i] - base);
            held_l[i] = held_l[i] * fo + l[i] * fn;
            held_ref[i] = both;
            float* to = sh_o + (wave * 8 + 2 * j + i) * kRow + n;
#pragma unroll
            for (int c = 0; c < 2 * NG; ++c) {
                const float x = __builtin_fmaf(o[c][2 * i + 1], 1 / kRest, o[c][2 * i]) * over_pow2(under[c / 2]) * fn;
                to[16 * c] = held ? to[16 * c] * fo + x : x;
            }
        }
        held = true;
        }
        if (__builtin_amdgcn_ballot_w64(bad)) held_l[0] = held_l[1] = __builtin_nanf("");
#pragma unroll
        for (int i = 0; i < 2; ++i) {
#pragma unroll
            for (int w = 1; w <= 8; w <<= 1) held_l[i] += __shfl_xor(held_l[i], w);
            if (n == 0) {
                sh_m[wave][2 * j + i] = held_ref[i];
                sh_l[wave][2 * j + i] = held_l[i];
            }
        }
        __syncthreads();
        // a row that is whole here is done, else its part goes to the joining: to
        // one place if it began before this workgroup, to another if it began here
        const bool whole = first == 0 && last == tiles;
        float* part = a.part + (2 * (int64_t)blockIdx.x + (first == 0)) * 8 * (D + 2);
        for (int i = threadIdx.x; i < rows * D; i += 64 * kWaves) {
            const int r = i / D, c = i - r * D;
            float mm = sh_m[0][r];
#pragma unroll
            for (int w = 1; w < kWaves; ++w) mm = __builtin_fmaxf(mm, sh_m[w][r]);
            const float base = mm == -__builtin_inff() ? 0.f : mm;
            float sum = 0.f, val = 0.f;
#pragma unroll
            for (int w = 0; w < kWaves; ++w) {
                const float f = __builtin_amdgcn_exp2f(sh_m[w][r] - base);
                sum += f * sh_l[w][r];
                val += f > 0.f ? f * sh_o[(w * 8 + r) * kRow + c] : 0.f;    // a wave without tiles wrote none
            }
            if (whole) {
                const int64_t h = (int64_t)kvh * group + 8 * hc + r;
                static_cast<typename T::Elem*>(a.out)[(int64_t)b * a.ld_out + h * D + c] = T::one(len == 0 ? 0.f : val / sum);
            } else {
                part[r * D + c] = val;
                if (c == 0) {
                    part[8 * D + 2 * r] = mm;
                    part[8 * D + 2 * r + 1] = sum;
                }
            }
        }
        if (!shared || at >= end) break;
        if (last == tiles && pair == pairs - 1) {                    // on to the next sequence that has any
            uint64_t more = __builtin_amdgcn_ballot_w64(line.len > 0) >> k >> 1;
            while (more == 0) {
                begin += line.all() * pairs;
                line.read(a, line.from + 64, lane);
                k = -1;
                more = __builtin_amdgcn_ballot_w64(line.len > 0);
            }
            k += 1 + (int)__builtin_ctzll(more);
        }
        __syncthreads();                                             // the next results go to the same place
    }
}

// Rows that more than one workgroup worked on, joined in their order, and rows
// that none did: 256 / (D / 4) parts at a time, four columns a thread.
template <int TYPE, int D>
__global__ void __launch_bounds__(256) attn_join_kernel(DecodeArgs a) {
    using T = Val<TYPE>;
    constexpr int kCols = D / 4, kAt = 256 / kCols;
    __shared__ float vals[kAt][D], sums[kAt];
    const int lane = threadIdx.x & 63;
    const uint32_t b = blockIdx.x / (uint32_t)a.q_heads, h = blockIdx.x - b * (uint32_t)a.q_heads;
    const int group = (int)((uint32_t)a.q_heads / (uint32_t)a.kv_heads), chunks = (group + 7) / 8;
    const int pairs = (int)a.kv_heads * chunks, kvh = (int)h / group, in = (int)h - kvh * group;
    const int pair = kvh * chunks + in / 8, row = in & 7;
    typename T::Elem* out = static_cast<typename T::Elem*>(a.out) + b * a.ld_out + (int64_t)h * D;
    const int len = length_of(a, (int)b), tiles = tiles_in(len);
    if (tiles == 0) {
        if (threadIdx.x < D) out[threadIdx.x] = T::one(len < 0 ? __builtin_nanf("") : 0.f);
        return;
    }
    Line line;
    line.open(a, pairs, lane);
    int start = pair * (tiles + kPad) + kPad;                        // of its first tile
    while ((int)b - line.from >= 64) {
        start += line.all() * pairs;
        line.read(a, line.from + 64, lane);
    }
    start += line.before((int)b - line.from) * pairs;
    const uint32_t w0 = (uint32_t)start / (uint32_t)line.share, w1 = (uint32_t)(start + tiles - 1) / (uint32_t)line.share;
    if (w0 == w1) return;                                            // one workgroup's: done
    const int used = (int)(w1 - w0) + 1;
    auto part = [&](int s) { return a.part + (2 * (int64_t)(w0 + s) + (s == 0)) * 8 * (D + 2); };
    float mm = -__builtin_inff();
    for (int s = lane; s < used; s += 64) mm = __builtin_fmaxf(mm, part(s)[8 * D + 2 * row]);
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) mm = __builtin_fmaxf(mm, __shfl_xor(mm, i));
    const float base = mm == -__builtin_inff() ? 0.f : mm;
    const int c = threadIdx.x % kCols, at = threadIdx.x / kCols;
    float4 val = make_float4(0.f, 0.f, 0.f, 0.f);
    float sum = 0.f;
#pragma unroll 4
    for (int s = at; s < used; s += kAt) {
        const float* p = part(s);
        const float4 o = *reinterpret_cast<const float4*>(p + row * D + 4 * c);
        const float f = __builtin_amdgcn_exp2f(p[8 * D + 2 * row] - base);
        sum = __builtin_fmaf(f, p[8 * D + 2 * row + 1], sum);
        val.x = __builtin_fmaf(f, o.x, val.x);
        val.y = __builtin_fmaf(f, o.y, val.y);
        val.z = __builtin_fmaf(f, o.z, val.z);
        val.w = __builtin_fmaf(f, o.w, val.w);
    }
    *reinterpret_cast<float4*>(&vals[at][4 * c]) = val;
    if (c == 0) sums[at] = sum;
    __syncthreads();
    if (threadIdx.x < D) {
        float v = 0.f, t = 0.f;
#pragma unroll
        for (int i = 0; i < kAt; ++i) {
            v += vals[i][threadIdx.x];
            t += sums[i];
        }
        out[threadIdx.x] = T::one(v / t);
    }
}

}  // namespace

bool plan_attn_decode(DecodeArgs* a) {
    const int64_t tiles = (a->max_len + kKvTile - 1) / kKvTile;
    const int64_t group = a->q_heads / a->kv_heads, pairs = a->batch * a->kv_heads * ((group + 7) / 8);
    if (pairs * (tiles + kPad + 1) >= ((int64_t)1 << 31) - (1 << 20)) return false;
    const int64_t most = (pairs * (tiles + kPad) + kShareMin - 1) / kShareMin;
    a->groups = tiles <= (pairs < kGroups ? kWhole : kWholeMany) ? 0 : (int)(most < kGroups ? most : kGroups);
    // a launch has fewer than 2^32 threads: 256 for a pair, or for a row that is joined
    return (a->groups ? a->batch * a->q_heads : pairs) < ((int64_t)1 << 24);
}

size_t attn_decode_scratch(const DecodeArgs& a) {
    return sizeof(float) * (size_t)a.groups * 2 * 8 * (size_t)(a.head_dim + 2);
}

hipError_t launch_attn_decode(DecodeArgs a, float* scratch, hipStream_t stream) {
    const int64_t group = a.q_heads / a.kv_heads, pairs = a.batch * a.kv_heads * ((group + 7) / 8);
    const unsigned grid = (unsigned)(a.groups ? a.groups : pairs);
    const uint64_t page_tiles = (uint64_t)a.page_tokens / kKvTile;
    a.per_page = ((uint64_t)1 << 36) / page_tiles + 1;
    a.part = scratch;
    return with_type(a.type, [&](auto ty) {
        constexpr int kT = decltype(ty)::value;
        const auto run = [&](auto ng) {
            constexpr int kN = decltype(ng)::value;
            attn_decode_kernel<kT, kN><<<grid, 64 * kWaves, 0, stream>>>(a);
            if (const hipError_t e = hipGetLastError(); e != hipSuccess || a.groups == 0) return e;
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
