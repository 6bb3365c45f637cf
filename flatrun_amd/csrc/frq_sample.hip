// One token per row of logits:
//   w_i = exp((x_i - max x) / T);  sorted by x, equal ones by index, the first
//   top_k stay, of these the shortest run whose weights sum to top_p of theirs,
//   of these the ones with w >= min_p;  the token is the first index i at which
//   the sum of the weights that stayed exceeds u times all of it.
//
// Nothing is sorted. All three cuts take the list's lower end away, so what
// stays is: the logits above one value, and the first few that equal it. That
// value is found from histograms: 2048 bins of 1/64 in (max - x) / T, and below
// them, within one bin, the bits of x, eight at a time.
//
// Weights are whole numbers of 2^-kFrac: computed in 64 bits, rounded once.
// Sums of them are exact whatever their order, so every pass sees the same
// ones, the atomics of a histogram decide nothing, and a border lies where sums
// in 64 bits have it. A weight below 2^-45 of the largest is nothing.
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

constexpr int kThreads = 1024, kWaves = kThreads / 64;
constexpr int kBins = 2048;                  // of 1/64 each: exp(-32) is below 2^-45
constexpr int kStep = 256;                   // logits a wave takes at a time, four a lane
constexpr int kFrac = 44;

// Order of x as a number, larger first; equal ones (0 and -0) alike. NaN and
// -inf, which are never drawn, are 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -__builtin_inff() ? k : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u));
}

// A row's parameters, the largest logit, and the weights under them.
struct Row {
    double per_t;                            // T, to divide by
    float top, min_p, top_p;
    int64_t top_k;
    uint32_t top_key;
    bool greedy;
    __device__ __forceinline__ double depth(uint32_t key) const {        // (max - x) / T
        return key == top_key ? 0.0 : ((double)top - (double)of_key(key)) / per_t;
    }
};

__device__ __forceinline__ uint64_t wave_sum(uint64_t x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor((unsigned long long)x, i);
    return x;
}
__device__ __forceinline__ uint64_t wave_scan(uint64_t x, int lane) {    // up to and with the lane's
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const uint64_t y = __shfl_up((unsigned long long)x, i);
        if (lane >= i) x += y;
    }
    return x;
}

template <int TYPE>
__device__ __forceinline__ float load_logit(const void* row, int64_t i) {
    if constexpr (TYPE == kTypeF32) return static_cast<const float*>(row)[i];
    const uint16_t b = static_cast<const uint16_t*>(row)[i];
    if constexpr (TYPE == kTypeF16) return f16_bits_to_f32(b);
    return __builtin_bit_cast(float, (uint32_t)b << 16);
}

struct Shared {
    unsigned long long sum[kBins];
    uint32_t count[kBins];
    unsigned long long group[4096];          // of 256 logits
    unsigned long long wave[kWaves];
    uint32_t key[kWaves], index[kWaves];
    unsigned long long before, at;           // a search's answer
    uint32_t found;
};

// The first of `n` entries at which the running sum of f(i) passes `target`
// (less than the whole): its number in sh.found, what stands before it in
// sh.before. The whole workgroup calls.
template <typename F>
__device__ __forceinline__ void search(Shared& sh, int n, unsigned long long target, F&& f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (n + kThreads - 1) / kThreads;
    const int from = (int)threadIdx.x * per;
    unsigned long long mine = 0;
    for (int i = 0; i < per && from + i < n; ++i) mine += f(from + i);
    const unsigned long long upto = wave_scan(mine, lane);
    __syncthreads();
    if (lane == 63) sh.wave[wave] = upto;
    __syncthreads();
    unsigned long long base = upto - mine;
    for (int w = 0; w < wave; ++w) base += sh.wave[w];
    if (base <= target && target < base + mine) {
        for (int i = 0; i < per && from + i < n; ++i) {
            const unsigned long long x = f(from + i);
            if (target < base + x) {
                sh.found = (uint32_t)(from + i);
                sh.before = base;
                sh.at = x;
                break;
            }
            base += x;
        }
    }
    __syncthreads();
}

// Sum over the workgroup of a value a thread.
__device__ __forceinline__ unsigned long long group_sum(Shared& sh, unsigned long long x) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    x = wave_sum(x);
    __syncthreads();
    if (lane == 0) sh.wave[wave] = x;
    __syncthreads();
    x = 0;
    for (int w = 0; w < kWaves; ++w) x += sh.wave[w];
    return x;
}

template <int TYPE>
__global__ void __launch_bounds__(kThreads) sample_row_kernel(SampleArgs a) {
    __shared__ Shared sh;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    const int64_t r = blockIdx.x;
    const int n = (int)a.vocab, groups = (n + kStep - 1) / kStep;
    constexpr int kSize = TYPE == kTypeF32 ? 4 : 2;
    const char* row = static_cast<const char*>(a.logits) + r * a.ld * kSize;
    const double one = (double)((uint64_t)1 << a.frac);

    // every logit once: f(index, key), keys of a group of 256 by one wave
    auto each = [&](auto&& f) {
        for (int g = wave; g < groups; g += kWaves)
#pragma unroll
            for (int i = 0; i < kStep / 64; ++i) {
                const int e = g * kStep + i * 64 + lane;
                if (e < n) f(e, key_of(load_logit<TYPE>(row, e)));
            }
    };

    // the largest, the lowest index of equals
    Row p;
    uint32_t best = 0, where = 0;
    each([&](int e, uint32_t k) {
        if (k > best) { best = k; where = (uint32_t)e; }
    });
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const uint32_t k = __shfl_xor(best, i), w = __shfl_xor(where, i);
        if (k > best || (k == best && w < where)) { best = k; where = w; }
    }
    if (lane == 0) { sh.key[wave] = best; sh.index[wave] = where; }
    __syncthreads();
    best = 0, where = 0;
    for (int w = 0; w < kWaves; ++w)
        if (sh.key[w] > best || (sh.key[w] == best && sh.index[w] < where)) { best = sh.key[w]; where = sh.index[w]; }
    const float t = a.temperatures ? a.temperatures[r] : a.temperature;
    p.top_key = best;
    p.top = of_key(best);
    p.per_t = (double)__builtin_fminf(t, 3.4028235e38f);
    p.greedy = !(t > 0.f);
    p.top_k = a.top_ks ? a.top_ks[r] : a.top_k;
    p.top_p = a.top_ps ? a.top_ps[r] : a.top_p;
    p.min_p = a.min_ps ? a.min_ps[r] : a.min_p;
    if (best == 0 || p.greedy) {                 // nothing to draw, or the largest
        if (threadIdx.x == 0) {
            a.tokens[r] = best ? (int32_t)where : -1;
            if (a.probs) a.probs[r] = best ? 1.f : 0.f;
        }
        return;
    }
    const double min_w = p.min_p > 0.f ? (double)__builtin_fminf(p.min_p, 1.f) : 0.0;
    const bool cut_k = p.top_k > 0 && p.top_k < n, cut_p = p.top_p < 1.f;
    auto weight = [&](double w) { return (unsigned long long)__builtin_rint(w * one); };
    auto weight_of = [&](uint32_t k) -> unsigned long long { return k ? weight(exp(-p.depth(k))) : 0ull; };

    // What stays: keys above `low`, and those equal to it up to index `last`.
    uint32_t low = 0;
    int last = n;
    if (cut_k || cut_p) {
        for (int i = threadIdx.x; i < kBins; i += kThreads) sh.sum[i] = 0, sh.count[i] = 0;
        __syncthreads();
        each([&](int, uint32_t k) {
            const double d = k ? p.depth(k) : 1e9;
            if (d < kBins / 64.0) {
                const int b = (int)(d * 64.0);
                atomicAdd(&sh.sum[b], weight(exp(-d)));
                atomicAdd(&sh.count[b], 1u);
            }
        });
        __syncthreads();
        // One border: in the order of the list, the entry at which the running
        // count (by_count) or weight passes `target`. Leaves the entry's key in
        // `low`, the index of the last equal one that stays in `last`, and
        // returns the weight up to and with it.
        unsigned long long all = 0, many = 0;
        for (int i = threadIdx.x; i < kBins; i += kThreads) all += sh.sum[i], many += sh.count[i];
        all = group_sum(sh, all);
        many = group_sum(sh, many);
        const int bins = kBins;
        auto border = [&](bool by_count, unsigned long long target) -> unsigned long long {
            // the bin (sh.sum and sh.count still hold the bins of depth)
            search(sh, bins, target, [&](int i) { return by_count ? (unsigned long long)sh.count[i] : sh.sum[i]; });
            const int bin = (int)sh.found;
            target -= sh.before;
            unsigned long long upto = 0;
            for (int i = threadIdx.x; i < bin; i += kThreads) upto += sh.sum[i];
            upto = group_sum(sh, upto);
            // within it the bits of the key, from the top
            __shared__ unsigned long long dsum[256];
            __shared__ uint32_t dcount[256];
            uint32_t prefix = 0;
            for (int shift = 24; shift >= 0; shift -= 8) {
                __syncthreads();
                for (int i = threadIdx.x; i < 256; i += kThreads) dsum[i] = 0, dcount[i] = 0;
                __syncthreads();
                each([&](int, uint32_t k) {
                    if (!k || (shift < 24 && (k >> (shift + 8)) != prefix)) return;
                    const double d = p.depth(k);
                    if (!(d < kBins / 64.0) || (int)(d * 64.0) != bin) return;
                    const int digit = 255 - (int)(k >> shift & 255);
                    atomicAdd(&dsum[digit], weight(exp(-d)));
                    atomicAdd(&dcount[digit], 1u);
                });
                __syncthreads();
                search(sh, 256, target, [&](int i) { return by_count ? (unsigned long long)dcount[i] : dsum[i]; });
                const int digit = (int)sh.found;
                target -= sh.before;
                unsigned long long over = threadIdx.x < digit ? dsum[threadIdx.x & 255] : 0;
                upto += group_sum(sh, over);
                prefix = prefix << 8 | (uint32_t)(255 - digit);
            }
            // the equal ones: the first `extra` by index stay
            const unsigned long long w = weight_of(prefix);
            const unsigned long long extra = (by_count ? target : target / w) + 1;
            low = prefix;
            __syncthreads();
            for (int g = wave; g < groups; g += kWaves) {
                unsigned long long c = 0;
                for (int i = 0; i < kStep / 64; ++i) {
                    const int e = g * kStep + i * 64 + lane;
                    c += __builtin_popcountll(__builtin_amdgcn_ballot_w64(e < n && key_of(load_logit<TYPE>(row, e < n ? e : 0)) == low));
                }
                if (lane == 0) sh.group[g] = c;
            }
            __syncthreads();
            search(sh, groups, extra - 1, [&](int i) { return sh.group[i]; });
            {
                const int g = (int)sh.found;
                unsigned long long left = extra - 1 - sh.before;             // equal ones of the group before the last
                int at = 0;
                for (int i = 0; i < kStep / 64; ++i) {
                    const int e = g * kStep + i * 64 + lane;
                    const uint64_t m = __builtin_amdgcn_ballot_w64(e < n && key_of(load_logit<TYPE>(row, e < n ? e : 0)) == low);
                    const unsigned long long c = (unsigned long long)__builtin_popcountll(m);
                    if (left < c) {
                        uint64_t rest = m;
                        for (unsigned long long s = 0; s < left; ++s) rest &= rest - 1;
                        at = g * kStep + i * 64 + (int)__builtin_ctzll(rest);
                        break;
                    }
                    left -= c;
                }
                last = at;
            }
            __syncthreads();
            return upto + extra * w;
        };
        if (cut_k && (unsigned long long)p.top_k < many) all = border(true, (unsigned long long)p.top_k - 1);
        if (cut_p) {
            const double want = __builtin_ceil((double)p.top_p * (double)all);
            unsigned long long target = want >= 1.0 ? (unsigned long long)want : 1;
            if (target > all) target = all;
            border(false, target - 1);           // not past top_k's: all of the weight ends there
        }
    }
    auto stays = [&](int e, uint32_t k) { return k > low || (k == low && e <= last); };
    auto kept = [&](int e, uint32_t k) -> unsigned long long {
        if (k == 0 || !stays(e, k)) return 0;
        const double w = exp(-p.depth(k));
        return w < min_w && k != p.top_key ? 0 : weight(w);
    };

    // the weights that stay, summed by group, and the draw
    __syncthreads();
    for (int g = wave; g < groups; g += kWaves) {
        unsigned long long s = 0;
        for (int i = 0; i < kStep / 64; ++i) {
            const int e = g * kStep + i * 64 + lane;
            if (e < n) s += kept(e, key_of(load_logit<TYPE>(row, e)));
        }
        s = wave_sum(s);
        if (lane == 0) sh.group[g] = s;
    }
    __syncthreads();
    unsigned long long all = 0;
    for (int i = threadIdx.x; i < groups; i += kThreads) all += sh.group[i];
    all = group_sum(sh, all);
    const double u = a.u[r];
    const double x = u > 0.0 ? u * (double)all : 0.0;
    unsigned long long target = x < (double)all ? (unsigned long long)x : all - 1;
    if (target > all - 1) target = all - 1;
    search(sh, groups, target, [&](int i) { return sh.group[i]; });
    if (wave == 0) {
        const int g = (int)sh.found;
        unsigned long long left = target - sh.before;
        for (int i = 0; i < kStep / 64; ++i) {
            const int e = g * kStep + i * 64 + lane;
            const unsigned long long w = e < n ? kept(e, key_of(load_logit<TYPE>(row, e))) : 0, upto = wave_scan(w, lane);
            const uint64_t m = __builtin_amdgcn_ballot_w64(left < upto);
            if (m) {
                if (lane == (int)__builtin_ctzll(m)) {
                    a.tokens[r] = e;
                    if (a.probs) a.probs[r] = (float)((double)w / (double)all);
                }
                break;
            }
            left -= __shfl((unsigned long long)upto, 63);
        }
    }
}

}  // namespace

hipError_t launch_sample(SampleArgs a, hipStream_t stream) {
    int bits = 0;
    while (((int64_t)1 << bits) < a.vocab) ++bits;
    a.frac = 62 - bits < kFrac ? 62 - bits : kFrac;          // the sum of a row stays below 2^62
    return with_type(a.type, [&](auto ty) {
        sample_row_kernel<decltype(ty)::value><<<(unsigned)a.rows, kThreads, 0, stream>>>(a);
        return hipGetLastError();
    });
}

}  // namespace frq
