// One token per row of logits:
//   w_i = exp((x_i - max x) / T);  sorted by x, equal ones by index, the first
//   top_k stay, of these the shortest run whose weights sum to top_p of theirs,
//   of these the ones with w >= min_p;  the token is the first index i at which
//   the sum of the weights that stayed exceeds u times all of it.
//
// Nothing is sorted. All three cuts take the list's lower end away, so what
// stays is the logits above one place of the list. A histogram over the depth
// log2(e) (max - x) / T, 2048 bins of 1/44, says which bins stay whole and in
// which one or two the cuts lie; the logits of those, some hundreds, are listed
// and ranked against each other. top_k alone decides by counts; where it leaves
// up to kShort, all of them are listed and only they are weighed. Where a list
// is too long (thousands of logits within 1/44 of each other) the cuts are found
// from the bits of x, eight at a time, in further passes over the row.
//
// Weights are whole numbers of 2^-kFrac, computed in 64 bits and rounded once.
// Sums of them are exact whatever their order: every pass sees the same ones,
// atomics decide nothing, and a border lies where sums in 64 bits have it. In
// fp32 one draw in some hundred would fall on the other side of a border of a
// flat row of 10^5 logits.
//
// Passes over a row: its largest; the histogram (not without top_k and top_p);
// the sums of what stays by group of 1024, and the list; the group that the draw
// falls into. One workgroup does them all where there are rows for the GPU, else
// each pass is a launch of slices of all rows.
//
// What bounds it: one row, the launches and the chain of each (152064 fp32 logits,
// top_k 50 and top_p: 3.8, 5.0, 7.3 and 9.1 us); 64 rows of 131072 from the whole,
// the 64-bit weights (16 us of vector instructions, 67 % of the time) between a pass
// at 5.3 TB/s for the largest (6.3) and the draw (8.5). 256 rows of 152064, each with
// parameters of its own: 138 us for up to three passes; the slowest rows, with a
// top_p of their own, weigh every logit twice, and vector instructions fill 39 %
// (in slices, with the shares evened out, 146 to 184).
#include "frq_kernels.h"
#include "frq_vals.h"

namespace frq {
namespace {

constexpr int kBins = 2048, kPerBit = 44;    // depths up to 46.5: 2^-46 is no weight any more
constexpr int kFrac = 44;
constexpr int kGroup = 1024;                 // logits a wave takes at a time, four by four a lane
constexpr int kGroups = 1024;                // of a row, at most
constexpr int kList = 2048;                  // logits that are listed
constexpr int kShort = 1024;                 // top_k up to which all that stay are listed, and a bin more
constexpr int kRowThreads = 1024, kSliceThreads = 256, kPickThreads = 512;
constexpr float kInf = __builtin_inff();
using u64 = unsigned long long;

// Order of x as a number, larger first; equal ones (0 and -0) alike. NaN and
// -inf, which are never drawn, are 0.
__device__ __forceinline__ uint32_t key_of(float x) {
    const uint32_t b = __builtin_bit_cast(uint32_t, x + 0.f);
    const uint32_t k = b ^ ((uint32_t)((int32_t)b >> 31) | 0x80000000u);
    return x > -kInf ? k : 0u;
}
__device__ __forceinline__ float of_key(uint32_t k) {
    return __builtin_bit_cast(float, k ^ (~(uint32_t)((int32_t)k >> 31) | 0x80000000u));
}
// The list's order: larger logits first, then lower indices.
__device__ __forceinline__ u64 place_of(uint32_t key, int index) { return (u64)~key << 32 | (uint32_t)index; }

__device__ __forceinline__ u64 wave_sum(u64 x) {
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) x += __shfl_xor(x, i);
    return x;
}
__device__ __forceinline__ u64 wave_scan(u64 x, int lane) {          // up to and with the lane's
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const u64 y = __shfl_up(x, i);
        if (lane >= i) x += y;
    }
    return x;
}

// Four consecutive logits, as they are held.
template <int TYPE>
struct Raw {
    uint32_t w[TYPE == kTypeF32 ? 4 : 2];
    __device__ __forceinline__ void load(const void* row, int e) {
        __builtin_memcpy(w, static_cast<const char*>(row) + (int64_t)e * (TYPE == kTypeF32 ? 4 : 2), sizeof(w));
    }
    __device__ __forceinline__ void get(float (&x)[4]) const {
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            if constexpr (TYPE == kTypeF32)
                x[i] = __builtin_bit_cast(float, w[i]);
            else if constexpr (TYPE == kTypeF16)
                x[i] = f16_bits_to_f32(w[i / 2] >> (16 * (i & 1)) & 0xFFFFu);
            else
                x[i] = __builtin_bit_cast(float, i & 1 ? w[i / 2] & 0xFFFF0000u : w[i / 2] << 16);
        }
    }
};
// Four consecutive logits where the row may end; those from n on are -inf.
template <int TYPE>
__device__ __forceinline__ void load_end(const void* row, int e, int n, float (&x)[4]) {
#pragma unroll
    for (int i = 0; i < 4; ++i) {
        x[i] = -kInf;
        if (e + i >= n) continue;
        if constexpr (TYPE == kTypeF32) {
            x[i] = static_cast<const float*>(row)[e + i];
        } else {
            const uint16_t b = static_cast<const uint16_t*>(row)[e + i];
            x[i] = TYPE == kTypeF16 ? f16_bits_to_f32(b) : __builtin_bit_cast(float, (uint32_t)b << 16);
        }
    }
}

// A row's parameters, its largest logit, and weights under it.
struct Row {
    double per, top, least;                  // log2(e) / T; the largest; the least weight that min_p leaves, times 2^frac
    float top32, per32, finite;              // finite: the largest, 0 where that is inf
    int frac;
    double c[9];                             // of the polynomial in scaled(), in scalar registers
    float top_p;
    int64_t top_k;
    bool greedy, cut_k, cut_p, short_list;

    __device__ __forceinline__ void read(const SampleArgs& a, int64_t r) {
        const float t = a.temperatures ? a.temperatures[r] : a.temperature;
        const float least_p = a.min_ps ? a.min_ps[r] : a.min_p;
        top_p = a.top_ps ? a.top_ps[r] : a.top_p;
        top_k = a.top_ks ? a.top_ks[r] : a.top_k;
        greedy = !(t > 0.f);
        per = 1.4426950408889634 / (double)__builtin_fminf(t, 3.4028235e38f);
        per32 = (float)(per * kPerBit);
        frac = a.frac;
        const double k[9] = {-0x1.b63880a088780p-24, 0x1.63d136366f695p-20, -0x1.ffcb9515b5679p-17, 0x1.4308ac85aa8a7p-13,
                             -0x1.5d87fe86fe7f7p-10, 0x1.3b2ab7181b755p-7, -0x1.c6b08d7047e52p-5, 0x1.ebfbdff823cedp-3,
                             -0x1.62e42fefa39efp-1};
#pragma unroll
        for (int i = 0; i < 9; ++i) {
            c[i] = k[i];
            asm("" : "+s"(c[i]));            // else nine moves a weight
        }
        least = least_p > 0.f ? (double)__builtin_fminf(least_p, 1.f) * (double)((u64)1 << frac) : 0.0;
        cut_k = top_k > 0 && top_k < a.vocab;
        cut_p = top_p < 1.f;
        short_list = cut_k && top_k <= kShort;
    }
    __device__ __forceinline__ void largest_is(uint32_t key) {
        top32 = of_key(key);
        finite = top32 < kInf ? top32 : 0.f;
        top = (double)finite;
    }
    // The bin of x, in fp32: all that is asked of it is that a smaller x has no
    // smaller bin. kBins: no weight, or no number.
    __device__ __forceinline__ int bin(float x) const {
        const float d = x == top32 ? 0.f : (top32 - x) * per32;
        return d < (float)kBins ? (int)d : kBins;
    }
    // 2^(frac - t), t = log2(e) (max - x) / T, by whole steps of t and a
    // polynomial of degree 9 through Chebyshev's points of [-1/2, 1/2], within
    // 4e-14 of itself, for an x that has a bin.
    __device__ __forceinline__ double scaled(float x) const {
        const double t = (top - (double)(x == top32 ? finite : x)) * per;
        const double whole = t + 6755399441055744.0, r = t - (whole - 6755399441055744.0);     // 1.5 2^52
        double y = c[0];
#pragma unroll
        for (int i = 1; i < 9; ++i) y = __builtin_fma(y, r, c[i]);
        y = __builtin_fma(y, r, 1.0);
        const int n = frac - (int)(uint32_t)__builtin_bit_cast(u64, whole);
        const u64 bits = __builtin_bit_cast(u64, y);
        return __builtin_bit_cast(double, (u64)(((uint32_t)n << 20) + (uint32_t)(bits >> 32)) << 32 | (uint32_t)bits);
    }
    // A scaled weight as a whole number, to nearest: below 2^52.
    static __device__ __forceinline__ u64 count(double y) {
        return __builtin_bit_cast(u64, y + 4503599627370496.0) & 0x000FFFFFFFFFFFFFull;
    }
    // After min_p (of the logits that the other cuts leave).
    __device__ __forceinline__ u64 kept(double y) const { return y >= least ? count(y) : 0; }
    // The weight that top_p asks for of `all`: the run's sum reaches it.
    __device__ __forceinline__ u64 wanted(u64 all) const {
        const double want = __builtin_ceil((double)top_p * (double)all);
        const u64 w = want >= 1.0 ? (u64)want : 1;
        return w < all ? w : all;
    }
};

struct Shared {
    u64 wave[16];
    uint32_t key[16], index[16];
    u64 before, at;                          // a search's answer
    uint32_t found;
};

// Sum over the workgroup of a value a thread.
template <int NT>
__device__ __forceinline__ u64 group_sum(Shared& sh, u64 x) {
    x = wave_sum(x);
    __syncthreads();
    if ((threadIdx.x & 63) == 0) sh.wave[threadIdx.x >> 6] = x;
    __syncthreads();
    x = 0;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) x += sh.wave[w];
    return x;
}

// The first of `n` entries at which the running sum of f(i) passes `target`
// (less than the whole): its number in sh.found, what stands before it in
// sh.before, itself in sh.at. The whole workgroup calls.
template <int NT, typename F>
__device__ __forceinline__ void search(Shared& sh, int n, u64 target, F&& f) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, per = (n + NT - 1) / NT;
    const int from = (int)threadIdx.x * per;
    u64 mine = 0;
    for (int i = 0; i < per && from + i < n; ++i) mine += f(from + i);
    const u64 upto = wave_scan(mine, lane);
    __syncthreads();
    if (lane == 63) sh.wave[wave] = upto;
    __syncthreads();
    u64 base = upto - mine;
#pragma unroll
    for (int w = 0; w < NT / 64; ++w) base += w < wave ? sh.wave[w] : 0;
    if (base <= target && target < base + mine) {
        for (int i = 0; i < per && from + i < n; ++i) {
            const u64 x = f(from + i);
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

// Where the cuts lie: bins below `sure` stay whole; the logits of the bins
// [p_from, p_to] (top_p's cut) and of k_bin (top_k's) are listed.
struct Cuts {
    int sure, p_from, p_to, k_bin;
    u64 k_left;                              // logits of k_bin that stay
    u64 k_before, p_before, all;             // weights below k_bin, below p_from, and of all bins
    __device__ __forceinline__ bool listed(int b) const { return b == k_bin || (b >= p_from && b <= p_to); }
    __device__ __forceinline__ int last() const { return p_to > k_bin ? p_to : k_bin; }
    __device__ __forceinline__ void none() {
        sure = kBins;
        p_from = 1, p_to = 0, k_bin = -1;
        k_left = k_before = p_before = all = 0;
    }
    template <int NT>
    __device__ __forceinline__ void find_k(Shared& sh, const Row& p, const uint32_t* count) {
        u64 many = 0;
        for (int i = threadIdx.x; i < kBins; i += NT) many += count[i];
        many = group_sum<NT>(sh, many);
        if (!p.cut_k || (u64)p.top_k >= many) return;
        search<NT>(sh, kBins, (u64)p.top_k - 1, [&](int i) { return (u64)count[i]; });
        k_bin = (int)sh.found;
        k_left = (u64)p.top_k - sh.before;
        sure = k_bin;
    }
    // The bins that a short list takes, from counts alone.
    template <int NT>
    __device__ __forceinline__ void find_short(Shared& sh, const Row& p, const uint32_t* count) {
        none();
        find_k<NT>(sh, p, count);
        p_from = 0, p_to = k_bin >= 0 ? k_bin : kBins - 1, sure = 0, k_bin = -1;
    }
    template <int NT>
    __device__ __forceinline__ void find(Shared& sh, const Row& p, const u64* sum, const uint32_t* count) {
        none();
        find_k<NT>(sh, p, count);
        if (!p.cut_p) return;
        u64 low = 0;                                                 // what top_k leaves lies between low and high
        for (int i = threadIdx.x; i < kBins; i += NT) {
            all += sum[i];
            if (i < k_bin) low += sum[i];
        }
        all = group_sum<NT>(sh, all);
        k_before = group_sum<NT>(sh, low);
        low = k_bin >= 0 ? k_before : all;
        const u64 high = k_bin >= 0 ? low + sum[k_bin] : all;
        if (high == 0) return;
        search<NT>(sh, kBins, (low > 0 ? p.wanted(low) : 1) - 1, [&](int i) { return sum[i]; });
        p_from = sure = (int)sh.found;
        p_before = sh.before;
        search<NT>(sh, kBins, p.wanted(high) - 1, [&](int i) { return sum[i]; });
        p_to = (int)sh.found;
    }
};

// A listed logit: its place, and its weight below its bin.
struct Entry {
    u64 place, weight;
    __device__ __forceinline__ int bin() const { return (int)(weight >> 48); }
    __device__ __forceinline__ u64 w() const { return weight & 0xFFFFFFFFFFFFull; }
    __device__ __forceinline__ float value() const { return of_key(~(uint32_t)(place >> 32)); }
};

// Logits of the groups [from, to), wave by wave: f(group, index of the lane's
// first, x), x[i][j] at 256 i + j from there. The next group is asked for before
// one is worked on.
template <int TYPE, int NT, typename F>
__device__ __forceinline__ void each(const void* row, int n, int from, int to, F&& f) {
    constexpr int kStride = NT / 64;
    const int lane = threadIdx.x & 63, wave = __builtin_amdgcn_readfirstlane(threadIdx.x >> 6);
    const int full = n / kGroup < to ? n / kGroup : to;              // groups up to here are whole
    int g = from + wave;
    Raw<TYPE> raw[4];
    if (g < full)
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i].load(row, g * kGroup + 256 * i + 4 * lane);
    for (; g < full; g += kStride) {
        float x[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) raw[i].get(x[i]);
        if (g + kStride < full)
#pragma unroll
            for (int i = 0; i < 4; ++i) raw[i].load(row, (g + kStride) * kGroup + 256 * i + 4 * lane);
        f(g, g * kGroup + 4 * lane, x);
    }
    if (g < to) {
        float x[4][4];
#pragma unroll
        for (int i = 0; i < 4; ++i) load_end<TYPE>(row, g * kGroup + 256 * i + 4 * lane, n, x[i]);
        f(g, g * kGroup + 4 * lane, x);
    }
}

// The largest of the groups and, where asked for, the lowest index of equals, to
// every thread.
template <int TYPE, int NT>
__device__ __forceinline__ void largest(Shared& sh, const void* row, int n, int from, int to, bool where, uint32_t& key,
                                        uint32_t& index) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6;
    float best = -kInf;
    int at = -1;
    if (where)
        each<TYPE, NT>(row, n, from, to, [&](int, int e, const float (&x)[4][4]) {
            // a lane meets its indices in rising order: the first of equals stays
#pragma unroll
            for (int i = 0; i < 16; ++i)
                if (x[i / 4][i % 4] > best) best = x[i / 4][i % 4], at = e + i / 4 * 256 + i % 4;
        });
    else
        each<TYPE, NT>(row, n, from, to, [&](int, int, const float (&x)[4][4]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) best = __builtin_fmaxf(best, x[i / 4][i % 4]);
        });
    key = key_of(best);
    index = (uint32_t)at;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const uint32_t k = __shfl_xor(key, i), w = __shfl_xor(index, i);
        if (k > key || (k == key && w < index)) key = k, index = w;
    }
    __syncthreads();
    if (lane == 0) sh.key[wave] = key, sh.index[wave] = index;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w)
        if (sh.key[w] > key || (sh.key[w] == key && sh.index[w] < index)) key = sh.key[w], index = sh.index[w];
}

// Keeps a value's computation where it stands: what hides the 64-bit latency is
// that many go on side by side, not that some are left out.
__device__ __forceinline__ void here(u64& x) { asm volatile("" : "+v"(x)); }

// The histogram of the groups, into LDS that is zero.
template <int TYPE, int NT>
__device__ __forceinline__ void histogram(const Row& p, const void* row, int n, int from, int to, u64* sum, uint32_t* count) {
    if (p.short_list)                        // counts alone
        each<TYPE, NT>(row, n, from, to, [&](int, int, const float (&x)[4][4]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const int b = p.bin(x[i / 4][i % 4]);
                if (b < kBins) atomicAdd(&count[b], 1u);
            }
        });
    else
        each<TYPE, NT>(row, n, from, to, [&](int, int, const float (&x)[4][4]) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                u64 w[4];
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    w[j] = Row::count(p.scaled(x[i][j]));
                    here(w[j]);
                }
#pragma unroll
                for (int j = 0; j < 4; ++j) {
                    const int b = p.bin(x[i][j]);
                    if (b >= kBins) continue;
                    atomicAdd(&sum[b], w[j]);
                    if (p.cut_k) atomicAdd(&count[b], 1u);
                }
            }
        });
}

// Sums of what stays for certain, by group (not with a short list, where all that
// stays is listed), and the list: entries that fit in kList, all of them counted.
template <int TYPE, int NT>
__device__ __forceinline__ void sums_and_list(const Row& p, const Cuts& c, const void* row, int n, int from, int to, u64* group,
                                              Entry* list, uint32_t* listed) {
    const int lane = threadIdx.x & 63, last = c.last();
    each<TYPE, NT>(row, n, from, to, [&](int g, int e, const float (&x)[4][4]) {
        u64 s = 0;
        uint32_t any = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            int b[4], least = kBins;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                b[j] = p.bin(x[i][j]);
                least = b[j] < least ? b[j] : least;
                any |= (uint32_t)(b[j] >= c.sure && b[j] <= last) << (4 * i + j);
            }
            if (p.short_list || __builtin_amdgcn_ballot_w64(least < c.sure) == 0) continue;
#pragma unroll
            for (int j = 0; j < 4; ++j) {
                const double y = p.scaled(x[i][j]);
                u64 w = Row::count(y);
                here(w);
                s += b[j] < c.sure && y >= p.least ? w : 0;
            }
        }
        if (!p.short_list) {
            if (__builtin_amdgcn_ballot_w64(s != 0)) s = wave_sum(s);
            if (lane == 0) group[g] = s;
        }
        while (any) {                        // few
            const int i = __builtin_ctz(any);
            any &= any - 1;
            float y = 0.f;
#pragma unroll
            for (int o = 0; o < 16; ++o) y = o == i ? x[o / 4][o % 4] : y;
            const int b = p.bin(y);
            if (!c.listed(b)) continue;
            const uint32_t at = atomicAdd(listed, 1u);
            if (at < kList) list[at] = Entry{place_of(key_of(y), e + i / 4 * 256 + i % 4), Row::count(p.scaled(y)) | (u64)b << 48};
        }
    });
}

// LDS of a workgroup that finishes a row.
struct Finish {
    u64 sum[kBins], group[kGroups], dsum[256];
    uint32_t count[kBins], dcount[512], listed;
    Entry list[kList];
    u64 sort[2][kList];
};

// What stays of the list: those up to a place in its order, which is returned.
// Their weights are added to their groups. The list is put in order, by a bitonic
// network on one number an entry (key, index and number in the list), 32 steps of
// which leave the wave where there are 2048; then top_k counts and top_p sums.
template <int NT>
__device__ __forceinline__ u64 resolve(Shared& sh, Finish& f, const Row& p, const Cuts& c, int many) {
    constexpr int kPer = kList / NT;
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, t = (int)threadIdx.x;
    int size = 64;
    while (size < many) size *= 2;
    u64 v[kPer];
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
        const int i = x * NT + t;
        const u64 place = i < many ? f.list[i].place : 0;
        v[x] = i < many ? (place >> 32) << 32 | (u64)(uint32_t)place << 11 | (u64)i : ~(u64)0;
    }
    static_assert(kList <= 1 << 11, "the number of an entry has 11 bits, its index 20");
    if (size <= NT / 2) {                    // few: every entry counts those before it, NT / size threads an entry
        const int i = t & (size - 1), part = t / size, len = (many * size + NT - 1) / NT;
        uint32_t* before = f.dcount;
        if (t < size) before[t] = 0, f.sort[0][t] = v[0];
        __syncthreads();
        const u64 own = f.sort[0][i];
        uint32_t c = 0;
        const int to = (part + 1) * len < many ? (part + 1) * len : many;
        for (int j = part * len; j < to; ++j) c += f.sort[0][j] < own;
        if (i < many) atomicAdd(&before[i], c);
        __syncthreads();
        if (t < many) f.sort[1][before[t]] = v[0];
        __syncthreads();
        if (t < many) v[0] = f.sort[1][t];
    }
    int turn = 0;
    for (int k = 2; size > NT / 2 && k <= size; k *= 2)
        for (int j = k / 2; j; j /= 2) {
            if (j >= NT) {                                           // both in one thread
#pragma unroll
                for (int d = 1; d < kPer; d *= 2)
                    if (j == d * NT)
#pragma unroll
                        for (int x = 0; x < kPer; ++x) {
                            if (x & d) continue;
                            const bool rises = ((x * NT) & k) == 0, swap = (v[x] > v[x | d]) == rises;
                            const u64 a = swap ? v[x | d] : v[x], b = swap ? v[x] : v[x | d];
                            v[x] = a, v[x | d] = b;
                        }
                continue;
            }
            if (j >= 64) {
#pragma unroll
                for (int x = 0; x < kPer; ++x)
                    if (x * NT < size) f.sort[turn][x * NT + t] = v[x];
                __syncthreads();
            }
#pragma unroll
            for (int x = 0; x < kPer; ++x) {
                if (x * NT >= size) continue;
                const int i = x * NT + t;
                const u64 o = j >= 64 ? f.sort[turn][i ^ j] : __shfl_xor(v[x], j);
                const bool low = ((i & j) == 0) == ((i & k) == 0);   // keeps the smaller
                v[x] = low == (o < v[x]) ? o : v[x];
            }
            if (j >= 64) turn ^= 1;
        }
    // entry i of the order: its weight, and the weights before it
    Entry mine[kPer];
    u64 upto[kPer], whole = 0, first = 0;
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
        const int i = x * NT + t;
        mine[x] = Entry{~(u64)0, 0};
        upto[x] = 0;
        if (x * NT >= size) continue;
        if (i < many) mine[x] = f.list[v[x] & (kList - 1)];
        first += (u64)__builtin_popcountll(__builtin_amdgcn_ballot_w64(i < many && mine[x].bin() != c.k_bin));
        upto[x] = wave_scan(mine[x].w(), lane);
        __syncthreads();
        if (lane == 63) sh.wave[wave] = upto[x];
        __syncthreads();
        u64 base = whole;
#pragma unroll
        for (int w = 0; w < NT / 64; ++w) {
            base += w < wave ? sh.wave[w] : 0;
            whole += sh.wave[w];
        }
        upto[x] += base;
    }
    first = group_sum<NT>(sh, lane == 0 ? first : 0);                // entries of the bins above top_k's
    const u64 limit = p.short_list ? (u64)p.top_k : c.k_bin >= 0 ? first + c.k_left : ~(u64)0;
    u64 want = 0;
    if (p.cut_p) {
        u64 kept_k = 0;
#pragma unroll
        for (int x = 0; x < kPer; ++x)
            if ((u64)(x * NT + t) < limit && (p.short_list || mine[x].bin() == c.k_bin)) kept_k += mine[x].w();
        kept_k = group_sum<NT>(sh, kept_k);
        const u64 all = p.short_list ? kept_k : c.k_bin >= 0 ? c.k_before + kept_k : c.all;
        want = all > 0 ? p.wanted(all) : 0;
    }
    u64 to = 0;
#pragma unroll
    for (int x = 0; x < kPer; ++x) {
        const int i = x * NT + t, b = mine[x].bin();
        if (i >= many || (u64)i >= limit) continue;
        if (p.cut_p && (b < c.p_from || b > c.p_to || c.p_before + upto[x] - mine[x].w() >= want)) continue;
        to = mine[x].place;                                          // they rise
        const u64 w = p.kept(p.scaled(mine[x].value()));
        if (w) atomicAdd(&f.group[(uint32_t)mine[x].place / kGroup], w);
    }
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const u64 o = __shfl_xor(to, i);
        to = o > to ? o : to;
    }
    __syncthreads();
    if (lane == 0) sh.wave[wave] = to;
    __syncthreads();
    for (int w = 0; w < NT / 64; ++w) to = sh.wave[w] > to ? sh.wave[w] : to;
    return to;
}

// The draw from the groups' sums: what stays are bins below `sure` and places up
// to `to`. The whole workgroup calls.
template <int TYPE, int NT>
__device__ __forceinline__ void draw(Shared& sh, const SampleArgs& a, int64_t r, float number, const Row& p, int sure, u64 to, const void* row,
                                     const u64* group) {
    const int n = (int)a.vocab, groups = (n + kGroup - 1) / kGroup, lane = threadIdx.x & 63;
    u64 all = 0;
    for (int i = threadIdx.x; i < groups; i += NT) all += group[i];
    all = group_sum<NT>(sh, all);
    const double u = number, x = u > 0.0 ? u * (double)all : 0.0;
    u64 target = x < (double)all ? (u64)x : all - 1;
    target = target < all ? target : all - 1;
    search<NT>(sh, groups, target, [&](int i) { return group[i]; });
    if (threadIdx.x >= 64) return;
    u64 left = target - sh.before;
    float y[4][4];
#pragma unroll
    for (int q = 0; q < 4; ++q) load_end<TYPE>(row, (int)sh.found * kGroup + 256 * q + 4 * lane, n, y[q]);
#pragma unroll
    for (int q = 0; q < 4; ++q) {
        const int e = (int)sh.found * kGroup + 256 * q + 4 * lane;
        u64 w[4], mine = 0;
#pragma unroll
        for (int i = 0; i < 4; ++i) {
            const int b = p.bin(y[q][i]);
            w[i] = b < sure || (b < kBins && place_of(key_of(y[q][i]), e + i) <= to) ? p.kept(p.scaled(y[q][i])) : 0;
            mine += w[i];
        }
        const u64 upto = wave_scan(mine, lane);
        u64 base = upto - mine;
        if (base <= left && left < upto) {
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (base <= left && left < base + w[i]) {
                    a.tokens[r] = e + i;
                    if (a.probs) a.probs[r] = (float)((double)w[i] / (double)all);
                }
                base += w[i];
            }
        }
        const u64 whole = __shfl(upto, 63);
        if (left < whole) return;
        left -= whole;
    }
}

// A cut from the bits of x, for rows whose list is too long: eight bits at a time
// within a bin, then the indices of equal ones. Returns the last place that stays,
// and the weight up to it.
template <int TYPE, int NT>
__device__ __forceinline__ u64 border(Shared& sh, Finish& f, const Row& p, const void* row, int n, bool by_count, u64 target, u64& upto) {
    const int lane = threadIdx.x & 63, wave = threadIdx.x >> 6, groups = (n + kGroup - 1) / kGroup;
    search<NT>(sh, kBins, target, [&](int i) { return by_count ? (u64)f.count[i] : f.sum[i]; });
    const int bin = (int)sh.found;
    target -= sh.before;
    upto = 0;
    for (int i = threadIdx.x; i < bin; i += NT) upto += f.sum[i];
    upto = group_sum<NT>(sh, upto);
    uint32_t prefix = 0;
    for (int shift = 24; shift >= 0; shift -= 8) {
        __syncthreads();
        for (int i = threadIdx.x; i < 256; i += NT) f.dsum[i] = 0, f.dcount[i] = 0;
        __syncthreads();
        each<TYPE, NT>(row, n, 0, groups, [&](int, int, const float (&x)[4][4]) {
#pragma unroll
            for (int i = 0; i < 16; ++i) {
                const float y = x[i / 4][i % 4];
                const uint32_t k = key_of(y);
                if (p.bin(y) != bin || (shift < 24 && (k >> (shift + 8)) != prefix)) continue;
                const int digit = 255 - (int)(k >> shift & 255);
                atomicAdd(&f.dsum[digit], Row::count(p.scaled(y)));
                atomicAdd(&f.dcount[digit], 1u);
            }
        });
        __syncthreads();
        search<NT>(sh, 256, target, [&](int i) { return by_count ? (u64)f.dcount[i] : f.dsum[i]; });
        const int digit = (int)sh.found;
        target -= sh.before;
        upto += group_sum<NT>(sh, (int)threadIdx.x < digit ? f.dsum[threadIdx.x & 255] : 0);
        prefix = prefix << 8 | (uint32_t)(255 - digit);
    }
    // the equal ones: the first `extra` by index stay
    const u64 w = Row::count(p.scaled(of_key(prefix)));
    const u64 extra = (by_count ? target : target / w) + 1;
    upto += extra * w;
    __syncthreads();
    each<TYPE, NT>(row, n, 0, groups, [&](int g, int, const float (&x)[4][4]) {
        u64 c = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) c += (u64)__builtin_popcountll(__builtin_amdgcn_ballot_w64(key_of(x[i / 4][i % 4]) == prefix));
        if (lane == 0) f.group[g] = c;
    });
    __syncthreads();
    search<NT>(sh, groups, extra - 1, [&](int i) { return f.group[i]; });
    if (wave == 0) {
        u64 base = 0;
        const u64 left = extra - 1 - sh.before;                      // equal ones of the group before the last
        for (int q = 0; q < 4; ++q) {
            const int e = (int)sh.found * kGroup + 256 * q + 4 * lane;
            float x[4];
            load_end<TYPE>(row, e, n, x);
            u64 mine = 0;
#pragma unroll
            for (int i = 0; i < 4; ++i) mine += key_of(x[i]) == prefix;
            const u64 upto = wave_scan(mine, lane);
            u64 at = base + upto - mine;
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                if (key_of(x[i]) != prefix) continue;
                if (at == left) sh.at = place_of(prefix, e + i);
                ++at;
            }
            base += __shfl(upto, 63);
        }
    }
    __syncthreads();
    const u64 place = sh.at;
    __syncthreads();
    return place;
}

template <int TYPE, int NT>
__device__ __forceinline__ void long_way(Shared& sh, Finish& f, const SampleArgs& a, int64_t r, float u, Row p, const void* row) {
    const int n = (int)a.vocab, groups = (n + kGroup - 1) / kGroup, lane = threadIdx.x & 63;
    p.short_list = false;                    // weights of all bins
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += NT) f.sum[i] = 0, f.count[i] = 0;
    __syncthreads();
    histogram<TYPE, NT>(p, row, n, 0, groups, f.sum, f.count);
    __syncthreads();
    u64 all = 0, many = 0, to = ~(u64)0, upto = 0;
    for (int i = threadIdx.x; i < kBins; i += NT) all += f.sum[i], many += f.count[i];
    all = group_sum<NT>(sh, all);
    many = group_sum<NT>(sh, many);
    if (p.cut_k && (u64)p.top_k < many) {
        to = border<TYPE, NT>(sh, f, p, row, n, true, (u64)p.top_k - 1, upto);
        all = upto;
    }
    if (p.cut_p) to = border<TYPE, NT>(sh, f, p, row, n, false, p.wanted(all) - 1, upto);
    __syncthreads();
    each<TYPE, NT>(row, n, 0, groups, [&](int g, int e, const float (&x)[4][4]) {
        u64 s = 0;
#pragma unroll
        for (int i = 0; i < 16; ++i) {
            const float y = x[i / 4][i % 4];
            if (p.bin(y) < kBins && place_of(key_of(y), e + i / 4 * 256 + i % 4) <= to) s += p.kept(p.scaled(y));
        }
        s = wave_sum(s);
        if (lane == 0) f.group[g] = s;
    });
    __syncthreads();
    draw<TYPE, NT>(sh, a, r, u, p, 0, to, row, f.group);
}

// From the list (and, without a short list, the cuts and the groups' sums) to
// the token. The workgroup has met since they were written.
template <int TYPE, int NT>
__device__ __forceinline__ void finish(Shared& sh, Finish& f, const SampleArgs& a, int64_t r, float u, const Row& p, const Cuts& c, const void* row) {
    const int n = (int)a.vocab, groups = (n + kGroup - 1) / kGroup, many = (int)f.listed;
    if (many > kList) return long_way<TYPE, NT>(sh, f, a, r, u, p, row);
    if (p.short_list) {                      // resolve meets before it adds
        for (int i = threadIdx.x; i < groups; i += NT) f.group[i] = 0;
    }
    const u64 to = many ? resolve<NT>(sh, f, p, c, many) : 0;
    __syncthreads();
    draw<TYPE, NT>(sh, a, r, u, p, c.sure, to, row, f.group);
}

__device__ __forceinline__ void take(const SampleArgs& a, int64_t r, uint32_t key, uint32_t index) {
    if (threadIdx.x) return;
    a.tokens[r] = key ? (int32_t)index : -1;
    if (a.probs) a.probs[r] = key ? 1.f : 0.f;
}

// --------------------------------------------------- a row to a workgroup

template <int TYPE>
__device__ __forceinline__ const char* row_of(const SampleArgs& a, int64_t r) {
    return static_cast<const char*>(a.logits) + r * a.ld * (TYPE == kTypeF32 ? 4 : 2);
}

template <int TYPE>
__global__ void __launch_bounds__(kRowThreads) sample_row_kernel(SampleArgs a) {
    constexpr int NT = kRowThreads;
    __shared__ Shared sh;
    __shared__ Finish f;
    const int64_t r = blockIdx.x;
    const int n = (int)a.vocab, groups = (n + kGroup - 1) / kGroup;
    const char* row = row_of<TYPE>(a, r);
    if (threadIdx.x == 0) f.listed = 0;
    for (int i = threadIdx.x; i < kBins; i += NT) f.sum[i] = 0, f.count[i] = 0;
    Row p;
    p.read(a, r);
    uint32_t key, index;
    largest<TYPE, NT>(sh, row, n, 0, groups, p.greedy, key, index);
    if (key == 0 || p.greedy) return take(a, r, key, index);         // nothing to draw, or the largest
    p.largest_is(key);
    Cuts c;
    c.none();
    if (p.cut_k || p.cut_p) {
        histogram<TYPE, NT>(p, row, n, 0, groups, f.sum, f.count);
        __syncthreads();
        if (p.short_list)
            c.find_short<NT>(sh, p, f.count);
        else
            c.find<NT>(sh, p, f.sum, f.count);
    }
    const float u = a.u[r];
    sums_and_list<TYPE, NT>(p, c, row, n, 0, groups, f.group, f.list, &f.listed);
    __syncthreads();
    finish<TYPE, NT>(sh, f, a, r, u, p, c, row);
}

// ------------------------------------------------------ a row in slices

// Scratch of a row. The first launch clears what the others add to.
struct Held {
    u64 sum[kBins];
    uint32_t count[kBins];
    Entry list[kList];
    u64 group[kGroups];
    uint32_t key[64], index[64], listed;
};

struct Slice {
    int64_t r;
    int s, from, to;
    Held* held;
    __device__ __forceinline__ Slice(const SampleArgs& a) {
        const int groups = (int)((a.vocab + kGroup - 1) / kGroup), per = (groups + a.slices - 1) / a.slices;
        r = blockIdx.x / (uint32_t)a.slices;
        s = (int)(blockIdx.x - (uint32_t)r * (uint32_t)a.slices);
        from = s * per < groups ? s * per : groups;
        to = from + per < groups ? from + per : groups;
        held = static_cast<Held*>(a.scratch) + r;
    }
};

template <int TYPE>
__global__ void __launch_bounds__(kSliceThreads) sample_max_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ Shared sh;
    const Slice z(a);
    const char* row = row_of<TYPE>(a, z.r);
    Row p;
    p.read(a, z.r);
    if (!p.greedy && (p.cut_k || p.cut_p))
        for (int i = z.s * NT + (int)threadIdx.x; i < kBins; i += a.slices * NT) z.held->sum[i] = 0, z.held->count[i] = 0;
    if (z.s == 0 && threadIdx.x == 0) z.held->listed = 0;
    uint32_t key, index;
    largest<TYPE, NT>(sh, row, (int)a.vocab, z.from, z.to, p.greedy, key, index);
    if (threadIdx.x == 0) z.held->key[z.s] = key, z.held->index[z.s] = index;
}

// The row's largest from those of its slices.
__device__ __forceinline__ void largest_of(const SampleArgs& a, const Held* h, uint32_t& key, uint32_t& index) {
    const int lane = threadIdx.x & 63;
    key = lane < a.slices ? h->key[lane] : 0;
    index = lane < a.slices ? h->index[lane] : ~0u;
#pragma unroll
    for (int i = 1; i < 64; i <<= 1) {
        const uint32_t k = __shfl_xor(key, i), w = __shfl_xor(index, i);
        if (k > key || (k == key && w < index)) key = k, index = w;
    }
}

template <int TYPE>
__global__ void __launch_bounds__(kSliceThreads) sample_histogram_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ u64 sum[kBins];
    __shared__ uint32_t count[kBins];
    const Slice z(a);
    Row p;
    p.read(a, z.r);
    uint32_t key, index;
    largest_of(a, z.held, key, index);
    if (key == 0 || p.greedy || !(p.cut_k || p.cut_p)) return;
    p.largest_is(key);
    for (int i = threadIdx.x; i < kBins; i += NT) sum[i] = 0, count[i] = 0;
    __syncthreads();
    histogram<TYPE, NT>(p, row_of<TYPE>(a, z.r), (int)a.vocab, z.from, z.to, sum, count);
    __syncthreads();
    for (int i = threadIdx.x; i < kBins; i += NT) {
        if (sum[i]) atomicAdd(&z.held->sum[i], sum[i]);
        if (count[i]) atomicAdd(&z.held->count[i], count[i]);
    }
}

template <int TYPE>
__global__ void __launch_bounds__(kSliceThreads) sample_list_kernel(SampleArgs a) {
    constexpr int NT = kSliceThreads;
    __shared__ Shared sh;
    __shared__ u64 sum[kBins];
    __shared__ uint32_t count[kBins];
    const Slice z(a);
    Row p;
    p.read(a, z.r);
    uint32_t key, index;
    largest_of(a, z.held, key, index);
    if (key == 0 || p.greedy) return;
    p.largest_is(key);
    Cuts c;
    c.none();
    if (p.cut_k || p.cut_p) {
        for (int i = threadIdx.x; i < kBins; i += NT) sum[i] = z.held->sum[i], count[i] = z.held->count[i];
        __syncthreads();
        if (p.short_list)
            c.find_short<NT>(sh, p, count);
        else
            c.find<NT>(sh, p, sum, count);
    }
    sums_and_list<TYPE, NT>(p, c, row_of<TYPE>(a, z.r), (int)a.vocab, z.from, z.to, z.held->group, z.held->list, &z.held->listed);
}

template <int TYPE>
__global__ void __launch_bounds__(kPickThreads) sample_pick_kernel(SampleArgs a) {
    constexpr int NT = kPickThreads;
    __shared__ Shared sh;
    __shared__ Finish f;
    const int64_t r = blockIdx.x;
    const Held* h = static_cast<const Held*>(a.scratch) + r;
    const int groups = (int)((a.vocab + kGroup - 1) / kGroup);
    // all that does not hang on what another read says is asked for at once
    const float u = a.u[r];
    const uint32_t listed = h->listed;
    const Entry e0 = h->list[threadIdx.x];
    const u64 g0 = h->group[threadIdx.x];
    Row p;
    p.read(a, r);
    uint32_t key, index;
    largest_of(a, h, key, index);
    if (key == 0 || p.greedy) return take(a, r, key, index);
    p.largest_is(key);
    if (threadIdx.x == 0) f.listed = listed;
    f.list[threadIdx.x] = e0;
    for (int i = NT + threadIdx.x; i < (int)(listed < kList ? listed : kList); i += NT) f.list[i] = h->list[i];
    Cuts c;
    c.none();
    if (p.short_list) {                      // the list holds all that may stay
        c.sure = 0, c.p_from = 0, c.p_to = kBins - 1;
    } else {
        if (p.cut_k || p.cut_p)
            for (int i = threadIdx.x; i < kBins; i += NT) f.sum[i] = h->sum[i], f.count[i] = h->count[i];
        f.group[threadIdx.x] = g0;
        for (int i = NT + threadIdx.x; i < groups; i += NT) f.group[i] = h->group[i];
    }
    __syncthreads();
    if (!p.short_list && (p.cut_k || p.cut_p)) c.find<NT>(sh, p, f.sum, f.count);
    finish<TYPE, NT>(sh, f, a, r, u, p, c, row_of<TYPE>(a, r));
}

template <int TYPE>
hipError_t launch_typed(const SampleArgs& a, hipStream_t stream) {
    if (a.slices == 1) {
        sample_row_kernel<TYPE><<<(unsigned)a.rows, kRowThreads, 0, stream>>>(a);
        return hipGetLastError();
    }
    const unsigned grid = (unsigned)(a.rows * a.slices);
    // what the numbers given for all rows rule out is not launched
    const bool greedy = !a.temperatures && !(a.temperature > 0.f);
    const bool cuts = a.top_ks || a.top_ps || a.top_p < 1.f || (a.top_k > 0 && a.top_k < a.vocab);
    sample_max_kernel<TYPE><<<grid, kSliceThreads, 0, stream>>>(a);
    if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    if (!greedy && cuts) {
        sample_histogram_kernel<TYPE><<<grid, kSliceThreads, 0, stream>>>(a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    if (!greedy) {
        sample_list_kernel<TYPE><<<grid, kSliceThreads, 0, stream>>>(a);
        if (const hipError_t e = hipGetLastError(); e != hipSuccess) return e;
    }
    sample_pick_kernel<TYPE><<<(unsigned)a.rows, kPickThreads, 0, stream>>>(a);
    return hipGetLastError();
}

}  // namespace

void plan_sample(SampleArgs* a) {
    int bits = 0;
    while (((int64_t)1 << bits) < a->vocab) ++bits;
    a->frac = 62 - bits < kFrac ? 62 - bits : kFrac;         // the sum of a row stays below 2^62
    const int64_t groups = (a->vocab + kGroup - 1) / kGroup;
    // three workgroups a CU; whole rows from 128 on (256 rows: 138 us, 146 at best in slices)
    int64_t s = a->rows >= 128 ? 1 : 768 / (a->rows ? a->rows : 1);
    s = s < (groups + 3) / 4 ? s : (groups + 3) / 4;         // a group a wave
    s = s < 64 ? s : 64;
    a->slices = s > 1 ? (int)s : 1;
}

size_t sample_scratch(const SampleArgs& a) { return a.slices > 1 ? (size_t)a.rows * sizeof(Held) : 0; }

hipError_t launch_sample(SampleArgs a, void* scratch, hipStream_t stream) {
    a.scratch = scratch;
    return with_type(a.type, [&](auto ty) { return launch_typed<decltype(ty)::value>(a, stream); });
}

}  // namespace frq
