// The residual's addition and the root-mean-square norm behind it, one pass:
//   h = x + r, rounded to the residual's type (the next block's residual)
//   y = h / sqrt(mean(h^2) + eps) * w
// y in fp32, fp16, bf16, or as Q8_0 blocks: of the fp32 values, 32 at a time,
// d = fp16(max|y| / 127), held to 65504, and the codes round_even(y / d); a block
// with an inf or a NaN has d = NaN.
//
// Every operand passes once: memory bounds it. 8192 rows of 4096, fp32 in and sum,
// bf16 out: 84 us, 5.6 TB/s; one row: 2.2 us. 4097 rows of 3584 in bf16, out in
// 8-bit blocks: 25.5 us, 4.0 TB/s, by vector instructions, 40 an element (27.3 us
// with a division an element and codes stored two bytes at a time).
//
// Sums and products are in 64 bits and rounded once: an fp32 sum of squares
// leaves the last bit of y to the order of the sum, and with it, now and then,
// a code of the 8-bit form. Memory bounds the kernel either way.
//
// A workgroup holds a row in registers, eight elements at a time a thread (sixteen
// of 16-bit rows in half the threads: the same 25.5 us); rows of up to 256 share
// one (100000 of 96, fp32: 24.8 us, 34.9 with a wave each). Rows of other sizes and
// alignments take a second kernel, an element a thread at a time, held in registers
// too up to 16384 (8192 of 4097, fp32 to bf16: 130 us, 180 read twice; 20000 of 1001:
// 53 and 85, where aligned rows of 1000 take 50).
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

constexpr int kQ8 = 8;                   // out_type: Q8_0 blocks, 34 bytes for 32 elements
constexpr int kQ8Bytes = 34;

// Sum over the workgroup, in a fixed order; part: one place a wave.
__device__ __forceinline__ double group_sum(double x, double* part) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
    const int waves = blockDim.x >> 6;
    if (waves > 1) {
        if ((threadIdx.x & 63) == 0) part[threadIdx.x >> 6] = x;
        __syncthreads();
        x = part[0];
        for (int w = 1; w < waves; ++w) x += part[w];
    }
    return x;
}

// fp16(top / 127), held to 65504, and the code of y: the exact quotient rounded
// once. Near a half the remainder decides: a quotient rounded to fp32 first would
// now and then be the half itself.
__device__ __forceinline__ uint16_t q8_scale(float top) { return f32_to_f16_bits(__builtin_fminf(top / 127.0f, 65504.f)); }
__device__ __forceinline__ int q8_code(float y, float d) {
    if (d == 0.f) return 0;
    const float q = __builtin_fminf(__builtin_fmaxf(y / d, -127.f), 127.f);
    float k = __builtin_rintf(q);
    if (__builtin_fabsf(q - k) > 0.499f) {
        const float half = k + (q > k ? 0.5f : -0.5f), left = __builtin_fmaf(-half, d, y);
        k = left > 0.f ? half + 0.5f : left < 0.f ? half - 0.5f : __builtin_rintf(half);
    }
    return (int)k;
}

// Eight codes. y times 1 / d is within 2^-22 of the quotient: where that may
// decide the rounding, at 5e-5 from a half and nearer, the remainder does (one
// wave in ten). 2^23 + 2^22 rounds to integers and leaves them in the low byte.
__device__ __forceinline__ void q8_codes(const float (&y)[8], float d, uint32_t& lo, uint32_t& hi) {
    const float magic = 12582912.f, one_over = d == 0.f ? 0.f : 1.0f / d;
    uint32_t c[8];
    float off = 0.f;
#pragma unroll
    for (int i = 0; i < 8; ++i) {
        const float q = __builtin_amdgcn_fmed3f(y[i] * one_over, -127.f, 127.f), m = q + magic;
        c[i] = __builtin_bit_cast(uint32_t, m);
        off = __builtin_fmaxf(off, __builtin_fabsf(q - (m - magic)));
    }
    if (off > 0.49995f || !(d < __builtin_inff())) {
#pragma unroll
        for (int i = 0; i < 8; ++i) c[i] = (uint32_t)q8_code(y[i], d);
    }
    lo = (c[0] & 255) | (c[1] & 255) << 8 | (c[2] & 255) << 16 | c[3] << 24;
    hi = (c[4] & 255) | (c[5] & 255) << 8 | (c[6] & 255) << 16 | c[7] << 24;
}

template <int TYPE>
__device__ __forceinline__ float round_to(float x) {
    if constexpr (TYPE == kTypeBF16) return __builtin_bit_cast(float, (uint32_t)f32_to_bf16_bits(x) << 16);
    if constexpr (TYPE == kTypeF16) return f16_bits_to_f32(f32_to_f16_bits(x));
    return x;
}

// Eight elements a thread, CH times; a row to a workgroup or, where `lanes` of a
// wave hold it (SMALL), several.
template <int X, int R, int OUT, int CH, bool SMALL>
__global__ void __launch_bounds__(1024) norm_rows_kernel(NormArgs a, int lanes) {
    using TX = Val<X>;
    using TR = Val<R>;
    __shared__ double part[16];
    const int tid = SMALL ? (int)threadIdx.x & (lanes - 1) : (int)threadIdx.x;
    const int64_t row = SMALL ? (int64_t)blockIdx.x * (256 / lanes) + (int)threadIdx.x / lanes : blockIdx.x;
    if (SMALL && row >= a.rows) return;                  // all of a row's lanes, which meet nobody else
    const int hidden = (int)a.hidden, step = (int)blockDim.x * 8;
    const bool pairs = OUT == kQ8 && a.hidden % 64 == 0 && a.ld_out % 64 == 0 && (reinterpret_cast<uintptr_t>(a.out) & 3) == 0;
    float h[CH][8];
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = c * step + tid * 8;
        if (e < hidden) TX::load8(static_cast<const typename TX::Elem*>(a.x) + row * a.ld_x + e, h[c]);
    }
    if (a.residual) {
        float r[CH][8];
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e = c * step + tid * 8;
            if (e < hidden) TR::load8(static_cast<const typename TR::Elem*>(a.residual) + row * a.ld_res + e, r[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const int e = c * step + tid * 8;
            if (e >= hidden) break;
#pragma unroll
            for (int i = 0; i < 8; ++i) h[c][i] = round_to<R>(h[c][i] + r[c][i]);
            if (a.sum) TR::store8(static_cast<typename TR::Elem*>(a.sum) + row * a.ld_sum + e, h[c]);
        }
    }
    float w[CH][8];                      // on their way while the sum is made
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = c * step + tid * 8;
        if (a.weight && e < hidden) Val<kTypeF32>::load8(a.weight + e, w[c]);
    }
    double ss = 0.0;
#pragma unroll
    for (int c = 0; c < CH; ++c)
        if (c * step + tid * 8 < hidden)
#pragma unroll
            for (int i = 0; i < 8; ++i) ss = __builtin_fma((double)h[c][i], (double)h[c][i], ss);
    if constexpr (SMALL)
        for (int i = 1; i < lanes; i <<= 1) ss += __shfl_xor(ss, i);
    else
        ss = group_sum(ss, part);
    const double f = 1.0 / __builtin_sqrt(ss / (double)hidden + (double)a.eps);
#pragma unroll
    for (int c = 0; c < CH; ++c) {
        const int e = c * step + tid * 8;
        if (e >= hidden) break;                          // whole blocks of 32: four lanes go together
        float y[8];
#pragma unroll
        for (int i = 0; i < 8; ++i) y[i] = (float)((double)h[c][i] * f * (a.weight ? (double)w[c][i] : 1.0));
        if constexpr (OUT == kQ8) {
            uint32_t most = 0;           // |y| as integers: in order, NaN above infinity
#pragma unroll
            for (int i = 0; i < 8; ++i) {
                const uint32_t m = __builtin_bit_cast(uint32_t, y[i]) & 0x7FFFFFFFu;
                most = m > most ? m : most;
            }
            most = max(most, (uint32_t)__shfl_xor((int)most, 1));
            most = max(most, (uint32_t)__shfl_xor((int)most, 2));
            const uint16_t bits = most < 0x7F800000u ? q8_scale(__builtin_bit_cast(float, most)) : 0x7E00;
            uint32_t lo, hi;
            q8_codes(y, f16_bits_to_f32(bits), lo, hi);
            uint16_t* to = reinterpret_cast<uint16_t*>(static_cast<uint8_t*>(a.out) + (row * a.ld_out + e) / 32 * kQ8Bytes);
            const int j = tid & 3;
            if (pairs) {
                // two blocks are 17 words: the second's codes lie on words, the first's two bytes behind
                const bool second = tid & 4;
                const uint32_t before = (uint32_t)__shfl_up((int)hi, 1);
                uint32_t* words = reinterpret_cast<uint32_t*>(to + second) + 2 * j;
                if (second && j == 0) words[-1] = before >> 16 | (uint32_t)bits << 16;
                words[0] = second ? lo : (j ? before >> 16 : bits) | lo << 16;
                words[1] = second ? hi : lo >> 16 | hi << 16;
                continue;
            }
            if (j == 0) to[0] = bits;
            to[1 + 4 * j] = (uint16_t)lo;
            to[2 + 4 * j] = (uint16_t)(lo >> 16);
            to[3 + 4 * j] = (uint16_t)hi;
            to[4 + 4 * j] = (uint16_t)(hi >> 16);
        } else {
            using TO = Val<OUT>;
            TO::store8(static_cast<typename TO::Elem*>(a.out) + row * a.ld_out + e, y);
        }
    }
}

__device__ __forceinline__ float load_one(int type, const void* p, int64_t i) {
    if (type == kTypeF32) return static_cast<const float*>(p)[i];
    const uint16_t b = static_cast<const uint16_t*>(p)[i];
    return type == kTypeF16 ? f16_bits_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
}
__device__ __forceinline__ void store_one(int type, void* p, int64_t i, float x) {
    if (type == kTypeF32)
        static_cast<float*>(p)[i] = x;
    else
        static_cast<uint16_t*>(p)[i] = type == kTypeF16 ? f32_to_f16_bits(x) : f32_to_bf16_bits(x);
}

// CH elements of a row, `step` apart; those from n on are 0.
template <int CH>
__device__ __forceinline__ void load_some(int type, const void* p, int64_t base, int e, int step, int n, float (&x)[CH]) {
#pragma unroll
    for (int c = 0; c < CH; ++c) x[c] = 0.f;
    if (type == kTypeF32) {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (e + c * step < n) x[c] = static_cast<const float*>(p)[base + e + c * step];
    } else {
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (e + c * step < n) x[c] = __builtin_bit_cast(float, (uint32_t) static_cast<const uint16_t*>(p)[base + e + c * step]);
#pragma unroll
        for (int c = 0; c < CH; ++c) {
            const uint32_t b = __builtin_bit_cast(uint32_t, x[c]);
            x[c] = type == kTypeF16 ? f16_bits_to_f32(b) : __builtin_bit_cast(float, b << 16);
        }
    }
}

// Rows of any size and alignment, an element a thread at a time: CH times, held in
// registers, or (CH 0) as often as it takes, a row twice. 32 lanes share a block.
template <int CH>
__global__ void __launch_bounds__(1024) norm_any_kernel(NormArgs a) {
    __shared__ double part[16];
    const int64_t row = blockIdx.x;
    const int nt = (int)blockDim.x;
    auto rounded = [&](float h) {
        return a.res_type == kTypeF32 ? h : a.res_type == kTypeF16 ? round_to<kTypeF16>(h) : round_to<kTypeBF16>(h);
    };
    auto sum_at = [&](int64_t e) {
        const float x = load_one(a.x_type, a.x, row * a.ld_x + e);
        return a.residual ? rounded(x + load_one(a.res_type, a.residual, row * a.ld_res + e)) : x;
    };
    auto put = [&](int64_t e, float h, double f) {
        const float y = (float)((double)h * f * (a.weight ? (double)a.weight[e] : 1.0));
        if (a.out_type != kQ8) return store_one(a.out_type, a.out, row * a.ld_out + e, y);
        float top = __builtin_fabsf(y) < __builtin_inff() ? __builtin_fabsf(y) : __builtin_inff();
#pragma unroll
        for (int i = 1; i < 32; i <<= 1) top = __builtin_fmaxf(top, __shfl_xor(top, i));
        const uint16_t bits = top < __builtin_inff() ? q8_scale(top) : 0x7E00;
        uint8_t* to = static_cast<uint8_t*>(a.out) + (row * a.ld_out + e) / 32 * kQ8Bytes;
        if ((e & 31) == 0) *reinterpret_cast<uint16_t*>(to) = bits;
        to[2 + (e & 31)] = (uint8_t)q8_code(y, f16_bits_to_f32(bits));
    };
    double ss = 0.0;
    if constexpr (CH > 0) {
        const int n = (int)a.hidden, e0 = (int)threadIdx.x;
        float h[CH];
        load_some<CH>(a.x_type, a.x, row * a.ld_x, e0, nt, n, h);
        if (a.residual) {
            float r[CH];
            load_some<CH>(a.res_type, a.residual, row * a.ld_res, e0, nt, n, r);
#pragma unroll
            for (int c = 0; c < CH; ++c) h[c] = rounded(h[c] + r[c]);
            if (a.sum)
#pragma unroll
                for (int c = 0; c < CH; ++c)
                    if (e0 + c * nt < n) store_one(a.res_type, a.sum, row * a.ld_sum + e0 + c * nt, h[c]);
        }
#pragma unroll
        for (int c = 0; c < CH; ++c) ss = __builtin_fma((double)h[c], (double)h[c], ss);
        const double f = 1.0 / __builtin_sqrt(group_sum(ss, part) / (double)n + (double)a.eps);
#pragma unroll
        for (int c = 0; c < CH; ++c)
            if (e0 + c * nt < n) put(e0 + c * nt, h[c], f);
        return;
    }
    for (int64_t e = threadIdx.x; e < a.hidden; e += nt) {
        const float h = sum_at(e);
        if (a.sum) store_one(a.res_type, a.sum, row * a.ld_sum + e, h);
        ss = __builtin_fma((double)h, (double)h, ss);
    }
    const double f = 1.0 / __builtin_sqrt(group_sum(ss, part) / (double)a.hidden + (double)a.eps);
    // the sum may stand where x or the residual stood
    for (int64_t e = threadIdx.x; e < a.hidden; e += nt) put(e, a.sum ? load_one(a.res_type, a.sum, row * a.ld_sum + e) : sum_at(e), f);
}

template <int X, int R, int OUT>
hipError_t launch_typed(const NormArgs& a, unsigned threads, hipStream_t stream) {
    if (threads < 64)
        norm_rows_kernel<X, R, OUT, 1, true><<<(unsigned)((a.rows * threads + 255) / 256), 256, 0, stream>>>(a, (int)threads);
    else if (a.hidden <= (int64_t)threads * 8)
        norm_rows_kernel<X, R, OUT, 1, false><<<(unsigned)a.rows, threads, 0, stream>>>(a, 0);
    else
        norm_rows_kernel<X, R, OUT, 2, false><<<(unsigned)a.rows, threads, 0, stream>>>(a, 0);
    return hipGetLastError();
}

bool aligned(const void* p, int64_t ld, int type) {
    return (reinterpret_cast<uintptr_t>(p) & 15) == 0 && ld * (type == kTypeF32 ? 4 : 2) % 16 == 0;
}

hipError_t launch_part(const NormArgs& a, hipStream_t stream) {
    const bool wide = a.hidden % 8 == 0 && a.hidden <= 16384 && aligned(a.x, a.ld_x, a.x_type) &&
                      (!a.residual || aligned(a.residual, a.ld_res, a.res_type)) &&
                      (!a.sum || aligned(a.sum, a.ld_sum, a.res_type)) && (reinterpret_cast<uintptr_t>(a.weight) & 15) == 0 &&
                      (a.out_type == kQ8 || aligned(a.out, a.ld_out, a.out_type));
    if (!wide) {
        unsigned threads = 64;
        while (threads < 1024 && (int64_t)threads * 8 < a.hidden) threads *= 2;
        if (a.hidden <= (int64_t)threads * 8)
            norm_any_kernel<8><<<(unsigned)a.rows, threads, 0, stream>>>(a);
        else if (a.hidden <= (int64_t)threads * 16)
            norm_any_kernel<16><<<(unsigned)a.rows, threads, 0, stream>>>(a);
        else
            norm_any_kernel<0><<<(unsigned)a.rows, threads, 0, stream>>>(a);
        return hipGetLastError();
    }
    unsigned threads = 8;
    while (threads < 1024 && (int64_t)threads * 8 < a.hidden) threads *= 2;
    return with_type(a.x_type, [&](auto x) {
        return with_type(a.residual ? a.res_type : kTypeF32, [&](auto r) {
            constexpr int kX = decltype(x)::value, kR = decltype(r)::value;
            if (a.out_type == kQ8) return launch_typed<kX, kR, kQ8>(a, threads, stream);
            return with_type(a.out_type, [&](auto o) { return launch_typed<kX, kR, decltype(o)::value>(a, threads, stream); });
        });
    });
}

}  // namespace

hipError_t launch_add_rms_norm(const NormArgs& all, hipStream_t stream) {
    constexpr int64_t kMost = (int64_t)1 << 21;          // rows of 1024 threads: a launch has fewer than 2^32
    NormArgs a = all;
    const auto size = [](int type) { return type == kTypeF32 ? 4 : 2; };
    for (int64_t at = 0; at < all.rows; at += kMost) {
        a.rows = all.rows - at < kMost ? all.rows - at : kMost;
        a.x = static_cast<const char*>(all.x) + at * a.ld_x * size(a.x_type);
        if (a.residual) a.residual = static_cast<const char*>(all.residual) + at * a.ld_res * size(a.res_type);
        if (a.sum) a.sum = static_cast<char*>(all.sum) + at * a.ld_sum * size(a.res_type);
        a.out = static_cast<char*>(all.out) +
                (a.out_type == kQ8 ? at * a.ld_out / 32 * kQ8Bytes : at * a.ld_out * size(a.out_type));
        if (const hipError_t e = launch_part(a, stream); e != hipSuccess) return e;
    }
    return hipSuccess;
}

}  // namespace frq
