// One token per row of logits: temperature, top-k, top-p, min-p, and a draw from a given uniform number.
//
//   w_v = exp((l_v - m) / T), m = max l;  w = 1 where l_v = m, 0 where l_v is NaN or -inf or w < 2^-40
//   order: l descending, ties by the lower index; kept = the shortest of three prefixes of it:
//     the first k;  the first n whose weights reach p * (sum over the first k);  those with w >= min_p
//   token = the first kept v, in order of v, whose running sum of weights exceeds u * (sum kept)
//
// With 2^18 tokens of a flat distribution the running sums are 4e-6 apart, so fp32 sums would move
// the draw.  The weights are evaluated in fp64 and rounded to fixed point (a unit of 2^-50..2^-43 of the
// largest, so that V of them fit 63 bits): integer sums are exact in any order, hence the token
// depends neither on the split of the row nor on the order of the atomics below.
//
// A row is one cluster of CTAs; each keeps its slice of the row in shared memory, so the logits are read
// from HBM once and every later pass runs on chip.  The row is never sorted as a whole.  With top-k or top-p a
// histogram (counts; masses too for top-p alone), linear in the logit between the maximum and the 2^-40 floor,
// finds the bin that holds the border.  If at most SMP_LIST logits lie in that bin or above it, they
// are gathered into one CTA, sorted there, and everything else is done on that list.  Otherwise the border is
// narrowed down by further histograms over the integer keys of its bin until it is a single value
// (ties at that value are kept by index), and the kept weights are summed by blocks over the slices.
#pragma once
#include <cooperative_groups.h>
#include "engine.cuh"

namespace cce {

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = 2048;
constexpr int SMP_LIST = 1024;       // candidates that one CTA sorts
constexpr int SMP_BLK = 512;         // positions per block of the index-ordered search (16 per lane)
constexpr int SMP_MAX_CLUSTER = 16;  // above 8: allowed per kernel by an attribute
constexpr int SMP_SMEM = 224 * 1024; // dynamic shared memory at most: of the 227 KB of a CTA, the rest is static
constexpr double SMP_FLOOR_LOG2 = -40.0;
constexpr float SMP_LOWEST = -3.402823466e38f;

// A setting is an array with a value per row, or one value for all rows.
struct SampleParams {
    const void* logits;
    long long ld;      // elements between rows
    long long V;
    const float* u;    // [B]
    const float* temperature;  // [B] or null -> temperature_all; likewise below
    const long long* top_k;
    const float* top_p;
    const float* min_p;
    double temperature_all;
    long long top_k_all;  // <= 0: off
    double top_p_all;     // >= 1: off
    double min_p_all;     // <= 0: off
    long long* tokens;    // [B]
    float* logprobs;      // [B] or null
    int slice;            // positions per CTA: a multiple of SMP_BLK
    int frac_bits;        // weight 1 = 1 << frac_bits
};

typedef unsigned long long u64;

// The integer order of floats; +0 and -0 share a key.
__device__ __forceinline__ uint32_t order_key(float x) {
    const uint32_t b = __float_as_uint(x + 0.0f);
    return (b & 0x80000000u) ? ~b : (b | 0x80000000u);
}
__device__ __forceinline__ float order_value(uint32_t k) {
    return __uint_as_float((k & 0x80000000u) ? (k & 0x7fffffffu) : ~k);
}
// the largest float below x (key 0x7fffffff would be -0, which is not below +0)
__device__ __forceinline__ float just_below(float x) {
    const uint32_t k = order_key(x) - 1;
    return order_value(k == 0x7fffffffu ? k - 1 : k);
}

// 2^frac * exp((l - m) / T) rounded to an integer.  Table-driven (P. T. P. Tang, ACM TOMS 15(2), 1989):
// (l - m) * 64 log2(e) / T = 64 n + j + r with |r| <= 1/2, so the weight is 2^n * 2^(j/64) * e^z with
// z = r ln2 / 64, |z| < 0.0055, and four terms of the Taylor series leave a relative error of
// z^5/120 < 4e-14, below the rounding to 2^-43.  The product is added to 2^52, whose low bits then
// hold the rounded integer.  Nine fp64 operations: they bound the passes that need every weight.
constexpr int SMP_TABLE = 64;
struct WeightFn {
    double m, scale;      // maximum, 64 * log2(e) / T
    const double* table;  // shared memory: 2^(j/64)
    int frac;
    float peak;           // m as it is stored
    __device__ __forceinline__ u64 operator()(float l) const {
        constexpr double c = 0.010830424696249145;    // ln2 / 64
        constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
        const double d = double(l) - m;
        const double t = fma(d, scale, magic);
        const int i = __double2loint(t);
        const double r = fma(d, scale, magic - t);
        double e = fma(r, c * c * c * c / 24.0, c * c * c / 6.0);
        e = fma(e, r, c * c / 2.0);
        e = fma(e, r, c);
        e = fma(e, r, 1.0);
        const double tab = table[i & (SMP_TABLE - 1)];
        const double scaled =
            __hiloint2double(__double2hiint(tab) + ((i >> 6) + frac) * (1 << 20), __double2loint(tab));
        const double w = fma(e, scaled, 4503599627370496.0);  // 2^52
        const u64 q = (u64)__double_as_longlong(w) & 0xfffffffffffffull;
        return l == peak ? 1ull << frac : q;  // exact, also where the maximum is infinite
    }
};

// The dynamic shared memory of a CTA, in bytes from its start.
struct SampleLayout {
    int share;     // bins whose cluster-wide sums this CTA forms
    int max_blk;   // blocks of SMP_BLK positions a slice can touch (one more than it holds, by its alignment)
    int hist_mass, hist_cnt, own_mass, own_cnt, blk_mass, blk_tie, data, bytes;
    __host__ __device__ SampleLayout(int cluster, int slice, int elem_bytes) {
        share = SMP_BINS / cluster;
        max_blk = slice / SMP_BLK + 1;
        int o = 0;
        hist_mass = o, o += SMP_BINS * 8;  // later: two lists of SMP_LIST entries
        hist_cnt = o, o += SMP_BINS * 4;   // later: one list of SMP_LIST entries
        own_mass = o, o += share * 8;
        own_cnt = o, o += share * 4;
        blk_mass = o, o += max_blk * 8;
        blk_tie = o, o += max_blk * 4;
        data = (o + 15) / 16 * 16;
        bytes = data + max_blk * SMP_BLK * elem_bytes;
    }
};

struct SmpShared {
    double table[SMP_TABLE];
    u64 x[2][4][SMP_MAX_CLUSTER];  // exchange slots, written by the whole cluster
    u64 wa[SMP_WARPS], wb[SMP_WARPS];
    u64 r[4];
    float wf[SMP_WARPS];
    float l_floor, l_min;
    uint32_t n_local, n_list, base;
};

__device__ __forceinline__ u64 warp_sum_u64(u64 v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ u64 warp_scan_u64(u64 v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const u64 t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}
// In-place ascending sort of n (a power of two, at most 2 * SMP_THREADS) values by the whole CTA.
__device__ __forceinline__ void bitonic_sort(u64* v, int n) {
    for (int k = 2; k <= n; k <<= 1) {
        for (int j = k >> 1; j > 0; j >>= 1) {
            __syncthreads();
            const int t = threadIdx.x;
            if (t < n / 2) {
                const int a = 2 * t - (t & (j - 1)), b = a + j;
                const u64 x = v[a], y = v[b];
                if ((x > y) == ((a & k) == 0)) {
                    v[a] = y;
                    v[b] = x;
                }
            }
        }
    }
    __syncthreads();
}

// Positions with l > above are kept, and the first n_tie (in index order) of those with l == tie.
struct Cut {
    float above, tie;
    long long n_tie;
};

template <typename T>
struct Sampler {
    static constexpr int VE = 16 / int(sizeof(T));
    static constexpr int CHUNKS = SMP_BLK / VE / 32;  // 16-byte chunks per lane and block

    const SampleParams& p;
    SmpShared& sm;
    uint8_t* dyn;
    SampleLayout lay;
    cooperative_groups::cluster_group cl;
    int rank, size, buf = 0;
    long long row;
    int tid, warp, lane;
    // the slice: positions are counted from the 16-byte boundary at or below its first element, so that whole
    // 16-byte pieces of global memory land on 16-byte pieces of shared memory at any alignment; positions
    // outside the slice hold -inf
    uint4* data;
    long long start;
    int phase, n_blk;
    float mx, l_floor, l_min, bin_scale;
    double temp, top_p;
    float u;
    long long k;
    WeightFn weight;

    __device__ __forceinline__ Sampler(const SampleParams& p_, SmpShared& sm_, uint8_t* dyn_)
        : p(p_), sm(sm_), dyn(dyn_), lay(int(cooperative_groups::this_cluster().num_blocks()), p_.slice, int(sizeof(T))),
          cl(cooperative_groups::this_cluster()) {
        rank = int(cl.block_rank());
        size = int(cl.num_blocks());
        row = blockIdx.x / size;
        tid = threadIdx.x;
        warp = tid >> 5;
        lane = tid & 31;
        data = reinterpret_cast<uint4*>(dyn + lay.data);
    }
    __device__ __forceinline__ u64* hist_mass() const { return reinterpret_cast<u64*>(dyn + lay.hist_mass); }
    __device__ __forceinline__ uint32_t* hist_cnt() const { return reinterpret_cast<uint32_t*>(dyn + lay.hist_cnt); }
    __device__ __forceinline__ u64* blk_mass() const { return reinterpret_cast<u64*>(dyn + lay.blk_mass); }
    __device__ __forceinline__ uint32_t* blk_tie() const { return reinterpret_cast<uint32_t*>(dyn + lay.blk_tie); }

    // f(l, position) for every position of block b, a warp together
    template <typename F>
    __device__ __forceinline__ void each(int b, F f) const {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int q = (b * CHUNKS + c) * 32 + lane;
            const uint4 w = data[q];
            const T* x = reinterpret_cast<const T*>(&w);
#pragma unroll
            for (int i = 0; i < VE; ++i) f(float(x[i]), q * VE + i);
        }
    }
    // this warp's blocks of the slice
    template <typename F>
    __device__ __forceinline__ void each_of_slice(F f) const {
        for (int b = warp; b < n_blk; b += SMP_WARPS) each(b, f);
    }
    __device__ __forceinline__ long long token_at(int pos) const { return start + pos - phase; }

    // Four values of every CTA to all CTAs of the cluster: sm.x[buf][i][rank], i < 4 (the same in threads
    // 0..size-1).  Two buffers: a CTA that runs ahead writes the other one, and cannot come back to this one
    // before every CTA has passed the next barrier, hence read this one.
    __device__ __forceinline__ void exchange(u64 a, u64 b = 0, u64 c = 0, u64 d = 0) {
        buf ^= 1;
        if (size == 1) {
            if (tid == 0) {
                sm.x[buf][0][0] = a;
                sm.x[buf][1][0] = b;
                sm.x[buf][2][0] = c;
                sm.x[buf][3][0] = d;
            }
            __syncthreads();
            return;
        }
        if (tid < size) {
            SmpShared* dst = cl.map_shared_rank(&sm, tid);
            dst->x[buf][0][rank] = a;
            dst->x[buf][1][rank] = b;
            dst->x[buf][2][rank] = c;
            dst->x[buf][3][rank] = d;
        }
        cl.sync();
    }
    __device__ __forceinline__ u64 got(int i, int r) const { return sm.x[buf][i][r]; }
    // sum of two values over the CTA's threads, in every thread
    __device__ __forceinline__ void cta_sum(u64& a, u64& b) {
        a = warp_sum_u64(a);
        b = warp_sum_u64(b);
        __syncthreads();
        if (lane == 0) {
            sm.wa[warp] = a;
            sm.wb[warp] = b;
        }
        __syncthreads();
        a = b = 0;
#pragma unroll
        for (int w = 0; w < SMP_WARPS; ++w) {
            a += sm.wa[w];
            b += sm.wb[w];
        }
    }
    // inclusive scans of two values over the CTA's threads
    __device__ __forceinline__ void cta_scan(u64& a, u64& b) {
        a = warp_scan_u64(a, lane);
        b = warp_scan_u64(b, lane);
        __syncthreads();
        if (lane == 31) {
            sm.wa[warp] = a;
            sm.wb[warp] = b;
        }
        __syncthreads();
        for (int w = 0; w < warp; ++w) {
            a += sm.wa[w];
            b += sm.wb[w];
        }
    }

    __device__ __forceinline__ void write(long long token, float logprob) const {
        p.tokens[row] = token;
        if (p.logprobs) p.logprobs[row] = logprob;
    }
    // log of a kept logit's share of the kept weights
    __device__ __forceinline__ float log_share(float l, u64 total) const {
        const double y = l == mx ? 0.0 : (double(l) - double(mx)) / temp;
        return float(y - log(double(total) * exp2(-double(p.frac_bits))));
    }
    // the running sum that the drawn token is the first to exceed
    __device__ __forceinline__ u64 draw_target(u64 total) const {
        const double x = double(u) * double(total);
        if (!(x > 0.0)) return 0;
        return x >= double(total) ? total - 1 : min((u64)x, total - 1);
    }

    // ---- the slice to shared memory, and the row's maximum
    __device__ __forceinline__ void load() {
        start = (long long)rank * p.slice;
        const int n = int(max(0ll, min((long long)p.slice, p.V - start)));
        const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ld + start;
        phase = int((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
        n_blk = n > 0 ? (n + phase + SMP_BLK - 1) / SMP_BLK : 0;
        const T* src0 = src - phase;
        const int n_chunk = n_blk * (SMP_BLK / VE);
        const int lo = (phase + VE - 1) / VE, hi = (phase + n) / VE;  // chunks that lie in the slice as a whole
        float m = -INFINITY;
        constexpr int U = 4;  // loads in flight per thread
        for (int q0 = tid; q0 < n_chunk; q0 += U * SMP_THREADS) {
            uint4 v[U];
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int q = q0 + j * SMP_THREADS;
                if (q >= lo && q < hi) {
                    v[j] = __ldcs(reinterpret_cast<const uint4*>(src0) + q);
                } else {
                    T* x = reinterpret_cast<T*>(&v[j]);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const int pos = q * VE + i;
                        x[i] = (pos >= phase && pos < phase + n) ? src0[pos] : T(-INFINITY);
                    }
                }
            }
#pragma unroll
            for (int j = 0; j < U; ++j) {
                const int q = q0 + j * SMP_THREADS;
                if (q < n_chunk) data[q] = v[j];
                const T* x = reinterpret_cast<const T*>(&v[j]);
#pragma unroll
                for (int i = 0; i < VE; ++i) m = fmaxf(m, float(x[i]));  // drops NaN
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
        if (lane == 0) sm.wf[warp] = m;
        if (size > 1) cl.sync(); else __syncthreads();  // the cluster's CTAs run: their memory may be written
        m = -INFINITY;
#pragma unroll
        for (int w = 0; w < SMP_WARPS; ++w) m = fmaxf(m, sm.wf[w]);
        exchange(__float_as_uint(m));
        for (int r = 0; r < size; ++r) m = fmaxf(m, __uint_as_float(uint32_t(got(0, r))));
        mx = m + 0.0f;
    }

    // the first of the largest
    __device__ __forceinline__ void greedy() {
        uint32_t best = 0xffffffffu;
        each_of_slice([&](float l, int pos) {
            if (l == mx) best = min(best, uint32_t(pos));
        });
        best = __reduce_min_sync(0xffffffffu, best);
        __syncthreads();
        if (lane == 0) sm.wa[warp] = best;
        __syncthreads();
        for (int w = 0; w < SMP_WARPS; ++w) best = min(best, uint32_t(sm.wa[w]));
        exchange(best == 0xffffffffu ? ~0ull : u64(token_at(int(best))));
        if (rank == 0 && tid == 0) {
            u64 token = ~0ull;
            for (int r = 0; r < size; ++r) token = min(token, got(0, r));
            write((long long)token, 0.0f);
        }
    }

    // The smallest logit whose weight is at least 2^x (x <= 0): a first guess, then the neighbours.  A weight
    // that rounds to 1 in fp64, exp(z) with z >= -2^-54, counts as 1.
    __device__ __forceinline__ float lowest_with(double x, double k2) const {
        if (isinf(mx)) return mx;
        x = fmin(x, -8.0e-17);  // -2^-54 log2(e)
        float g = float(double(mx) + x / k2);
        if (!(g > SMP_LOWEST)) g = SMP_LOWEST;
        for (int it = 0; it < 4 && g < mx && (double(g) - double(mx)) * k2 < x; ++it) g = order_value(order_key(g) + 1);
        for (int it = 0; it < 4 && g > SMP_LOWEST; ++it) {
            const float below = just_below(g);
            if ((double(below) - double(mx)) * k2 < x) break;
            g = below;
        }
        return g;
    }

    // ---- histogram level 0: bins linear in the logit, bin 0 at the maximum (halves: the difference of two floats
    // may overflow).  The bin falls, or stays, as the logit grows.
    __device__ __forceinline__ int bin0(float l) const {
        return min(SMP_BINS - 1, int((0.5f * mx - 0.5f * l) * bin_scale));
    }
    __device__ __forceinline__ void clear_hist(bool mass) {
        for (int b = tid; b < SMP_BINS; b += SMP_THREADS) {
            hist_cnt()[b] = 0;
            if (mass) hist_mass()[b] = 0;
        }
        __syncthreads();
    }
    // Counts and masses of the bins over the cluster: this CTA's share to own_mass and own_cnt, the shares' totals
    // to got(0, r) (mass) and got(1, r) (count) of everyone.
    __device__ __forceinline__ void merge_hist(bool with_mass) {
        u64* mass = reinterpret_cast<u64*>(dyn + lay.own_mass);
        uint32_t* cnt = reinterpret_cast<uint32_t*>(dyn + lay.own_cnt);
        if (size > 1) cl.sync(); else __syncthreads();  // all histograms are complete
        u64 tm = 0, tc = 0;
        for (int b = tid; b < lay.share; b += SMP_THREADS) {
            u64 m = 0;
            uint32_t c = 0;
            for (int r = 0; r < size; ++r) {
                c += cl.map_shared_rank(hist_cnt(), r)[rank * lay.share + b];
                if (with_mass) m += cl.map_shared_rank(hist_mass(), r)[rank * lay.share + b];
            }
            mass[b] = m;
            cnt[b] = c;
            tm += m;
            tc += c;
        }
        cta_sum(tm, tc);
        exchange(tm, tc);
    }

    struct Border {
        int owner, bin;
        u64 mass_above, cnt_above, cnt;  // above the bin, and in it
    };
    // The bin where the running count (by_mass: mass) from the top reaches `target`, straight after merge_hist;
    // (am, ac): the mass and count above all of its bins.
    __device__ __forceinline__ Border find_border(bool by_mass, u64 target, u64 am, u64 ac) {
        const u64* mass = reinterpret_cast<const u64*>(dyn + lay.own_mass);
        const uint32_t* cnt = reinterpret_cast<const uint32_t*>(dyn + lay.own_cnt);
        int owner = 0;
        while (owner + 1 < size && (by_mass ? am + got(0, owner) : ac + got(1, owner)) < target) {
            am += got(0, owner);
            ac += got(1, owner);
            ++owner;
        }
        __syncthreads();
        if (rank == owner) {  // each thread scans `per` neighbouring bins
            const int per = max(1, lay.share / SMP_THREADS);
            u64 m = 0, c = 0;
            const int b0 = tid * per;
            if (b0 < lay.share)
                for (int i = 0; i < per; ++i) {
                    m += mass[b0 + i];
                    c += cnt[b0 + i];
                }
            u64 im = m, ic = c;
            cta_scan(im, ic);
            im += am;
            ic += ac;
            const u64 end = by_mass ? im : ic, begin = end - (by_mass ? m : c);
            if (begin < target && target <= end) {  // one thread
                u64 rm = im - m, rc = ic - c;
                for (int i = 0; i < per; ++i) {
                    const u64 nm = rm + mass[b0 + i], nc = rc + cnt[b0 + i];
                    if ((by_mass ? nm : nc) >= target) {
                        sm.r[0] = u64(owner * lay.share + b0 + i);
                        sm.r[1] = rm;
                        sm.r[2] = rc;
                        sm.r[3] = cnt[b0 + i];
                        break;
                    }
                    rm = nm;
                    rc = nc;
                }
            }
            __syncthreads();
        }
        exchange(sm.r[0], sm.r[1], sm.r[2], sm.r[3]);
        return Border{owner, int(got(0, owner)), got(1, owner), got(2, owner), got(3, owner)};
    }

    __device__ __forceinline__ void level0(bool with_mass) {
        clear_hist(with_mass);
        each_of_slice([&](float l, int) {
            if (l >= l_floor) {
                const int bin = bin0(l);
                atomicAdd(&hist_cnt()[bin], 1u);
                if (with_mass) atomicAdd(&hist_mass()[bin], weight(l));
            }
        });
        merge_hist(with_mass);
    }

    // The first key of [lo, hi] that fulfils a predicate which holds from some key on (hi if none before it does),
    // by all threads together
    template <typename F>
    __device__ __forceinline__ uint32_t first_key(uint32_t lo, uint32_t hi, F pred) {
        while (lo < hi) {
            const uint32_t step = (hi - lo) / SMP_THREADS + 1;
            const u64 at = u64(lo) + u64(tid) * step;
            const int below = __syncthreads_count(at < hi && !pred(uint32_t(at)));
            if (below == 0) return lo;
            const u64 next = u64(lo) + u64(below) * step;
            lo = lo + uint32_t(below - 1) * step + 1;
            hi = next < hi ? uint32_t(next) : hi;
        }
        return lo;
    }

    // From a level-0 border down to one value: that value, and the count and mass above it.
    struct Level {
        float value;
        u64 mass_above, cnt_above;
    };
    __device__ __forceinline__ Level descend(Border bd, bool by_mass, u64 target) {
        const uint32_t kmin = order_key(l_floor), kmax = order_key(mx);
        // the keys of bin bd.bin: from the first with bin0 <= bin, up to the one before the first with bin0 < bin
        uint32_t lo = first_key(kmin, kmax, [&](uint32_t q) { return bin0(order_value(q)) <= bd.bin; });
        uint32_t hi = bd.bin == 0 ? kmax : first_key(lo, kmax, [&](uint32_t q) { return bin0(order_value(q)) < bd.bin; }) - 1;
        while (hi > lo) {
            const int shift = max(0, 32 - __clz(hi - lo) - 11);  // (hi - lo) >> shift < SMP_BINS
            const float f_lo = order_value(lo), f_hi = order_value(hi);
            clear_hist(by_mass);
            each_of_slice([&](float l, int) {
                if (l >= f_lo && l <= f_hi) {
                    const int bin = int((hi - order_key(l)) >> shift);
                    atomicAdd(&hist_cnt()[bin], 1u);
                    if (by_mass) atomicAdd(&hist_mass()[bin], weight(l));
                }
            });
            merge_hist(by_mass);
            bd = find_border(by_mass, target, bd.mass_above, bd.cnt_above);
            const uint32_t top = hi - (uint32_t(bd.bin) << shift);
            lo = max(lo, top - ((1u << shift) - 1));
            hi = top;
        }
        return Level{order_value(lo), bd.mass_above, bd.cnt_above};
    }

    // ---- the whole rest on a list: every logit of bins 0..bin (at most SMP_LIST) goes to CTA `leader`, which sorts
    // them, applies the three prefixes and draws.  mass: of all weights (top-p without top-k).
    __device__ __forceinline__ void finish_on_list(int bin, int leader, u64 mass) {
        u64* local = hist_mass();               // this CTA's candidates; in the leader later the weights
        u64* list = hist_mass() + SMP_LIST;     // the leader's list: (key descending, index ascending)
        u64* by_index = reinterpret_cast<u64*>(hist_cnt());
        each_of_slice([&](float l, int pos) {
            if (l >= l_floor && bin0(l) <= bin)
                local[atomicAdd(&sm.n_local, 1u)] = u64(~order_key(l)) << 32 | u64(token_at(pos));
        });
        __syncthreads();
        const uint32_t n_local = sm.n_local;
        if (tid == 0 && n_local > 0) sm.base = atomicAdd(&cl.map_shared_rank(&sm, leader)->n_list, n_local);
        __syncthreads();
        u64* dst = cl.map_shared_rank(list, leader) + sm.base;
        for (uint32_t i = tid; i < n_local; i += SMP_THREADS) dst[i] = local[i];
        if (size > 1) cl.sync(); else __syncthreads();
        if (rank != leader) return;

        const int n = int(sm.n_list);
        int n2 = 2;
        while (n2 < n) n2 *= 2;
        for (int i = n + tid; i < n2; i += SMP_THREADS) list[i] = ~0ull;
        bitonic_sort(list, n2);

        const int n_k = k && k < n ? int(k) : n;
        u64 w[2];
        float l[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = 2 * tid + i;
            l[i] = j < n_k ? order_value(~uint32_t(list[j] >> 32)) : -INFINITY;
            w[i] = j < n_k ? weight(l[i]) : 0;
            if (j < n_k) local[j] = w[i];
        }
        u64 cum = w[0] + w[1], above_min = u64(l[0] >= l_min) + u64(l[1] >= l_min);
        cta_scan(cum, above_min);
        if (2 * tid < n_k && 2 * tid + 2 >= n_k) sm.r[0] = cum;  // sum over the first k
        if (tid == SMP_THREADS - 1) sm.r[1] = above_min;
        __syncthreads();
        int kept = max(1, int(min(u64(n_k), sm.r[1])));
        if (top_p < 1.0) {
            const u64 s = k ? sm.r[0] : mass;
            const double t = ceil(fmax(top_p, 0.0) * double(s));
            const u64 target = t < 1.0 ? 1ull : min((u64)t, s);
            // the first whose running sum reaches it
            int n_p = 0;
            n_p += __syncthreads_count(2 * tid < n_k && cum - w[1] < target);
            n_p += __syncthreads_count(2 * tid + 1 < n_k && cum < target);
            kept = min(kept, n_p + 1);
        }
        __syncthreads();
        // the kept weights' sum, and the kept candidates in order of their index
        if ((kept - 1) >> 1 == tid) sm.r[2] = (kept & 1) ? cum - w[1] : cum;
        n2 = 2;
        while (n2 < kept) n2 *= 2;
        for (int j = tid; j < n2; j += SMP_THREADS) by_index[j] = j < kept ? (list[j] << 32 | u64(j)) : ~0ull;
        bitonic_sort(by_index, n2);
        const u64 total = sm.r[2], target = draw_target(total);
        u64 v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = 2 * tid + i < kept ? local[uint32_t(by_index[2 * tid + i])] : 0;
        u64 run = v[0] + v[1], unused = 0;
        cta_scan(run, unused);
        if (run > target && run - v[0] - v[1] <= target) {  // one thread
            const u64 e = by_index[2 * tid + (run - v[1] > target ? 0 : 1)];
            write((long long)(e >> 32), log_share(order_value(~uint32_t(list[uint32_t(e)] >> 32)), total));
        }
    }

    // ---- the cut of top-k and top-p as a value and a number of ties, for borders too far down for a list
    __device__ __forceinline__ Cut cut_by_levels(Border bd, bool by_mass, u64 k_target, u64 p_target) {
        Cut cut{-INFINITY, 0.0f, 0};
        u64 mass = 0;
        if (k) {
            if (k_target) {
                const Level lv = descend(bd, false, k_target);
                cut = Cut{lv.value, lv.value, (long long)(k_target - lv.cnt_above)};
            }
            if (!(top_p < 1.0)) return cut;
            // the counts alone led here: now the masses, of the top-k and of every bin
            u64 s = 0, unused = 0;
            each_of_slice([&](float l, int) {
                if (l > cut.above && l >= l_floor) s += weight(l);
            });
            cta_sum(s, unused);
            exchange(s);
            for (int r = 0; r < size; ++r) mass += got(0, r);
            if (cut.n_tie > 0) mass += u64(cut.n_tie) * weight(cut.tie);
            const double t = ceil(fmax(top_p, 0.0) * double(mass));
            p_target = t < 1.0 ? 1ull : min((u64)t, mass);
            level0(true);
            bd = find_border(true, p_target, 0, 0);
        }
        const Level lv = descend(bd, true, p_target);
        const u64 w = weight(lv.value);
        long long need = (long long)((p_target - lv.mass_above + w - 1) / w);  // the mass above is short of the target
        if (cut.n_tie > 0 && lv.value == cut.tie) need = min(need, cut.n_tie);
        return Cut{lv.value, lv.value, need};
    }

    // ---- the draw over the slices: kept weights by blocks, ties counted apart
    __device__ __forceinline__ void draw(Cut cut) {
        if (cut.n_tie > 0 && cut.tie < l_min) cut.n_tie = 0;
        cut.above = fmaxf(cut.above, just_below(l_min));
        const bool ties = cut.n_tie > 0;
        u64 sum_m = 0, sum_t = 0;
        for (int b = warp; b < n_blk; b += SMP_WARPS) {
            u64 bm = 0;
            uint32_t bt = 0;
            each(b, [&](float l, int) {
                if (l > cut.above) bm += weight(l);
                if (ties && l == cut.tie) ++bt;
            });
            bm = warp_sum_u64(bm);
            if (ties) bt = __reduce_add_sync(0xffffffffu, bt);
            if (lane == 0) {
                blk_mass()[b] = bm;
                blk_tie()[b] = bt;
                sum_m += bm;
                sum_t += bt;
            }
        }
        cta_sum(sum_m, sum_t);
        exchange(sum_m, sum_t);

        // which CTA, which block, which position
        const u64 w_tie = ties ? weight(cut.tie) : 0;
        u64 total = 0, before = 0, mine = 0, ties_left = u64(cut.n_tie), my_ties = 0;
        for (int r = 0; r < size; ++r) {
            const u64 t = min(got(1, r), ties_left);
            const u64 m = got(0, r) + t * w_tie;
            if (r == rank) {
                before = total;
                mine = m;
                my_ties = ties_left;
            }
            total += m;
            ties_left -= t;
        }
        u64 target = draw_target(total);
        if (target < before || target >= before + mine || warp != 0) return;  // the owner's first warp goes on
        target -= before;
        for (int b0 = 0; b0 < n_blk; b0 += 32) {
            const int b = b0 + lane;
            const u64 t = b < n_blk && ties ? blk_tie()[b] : 0;
            const u64 t_incl = warp_scan_u64(t, lane), t_excl = t_incl - t;
            const u64 left = my_ties > t_excl ? my_ties - t_excl : 0;  // ties that this block may still keep
            const u64 m = (b < n_blk ? blk_mass()[b] : 0) + min(t, left) * w_tie;
            const u64 m_incl = warp_scan_u64(m, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, m_incl > target);
            if (!hit) {
                target -= __shfl_sync(0xffffffffu, m_incl, 31);
                const u64 seen = __shfl_sync(0xffffffffu, t_incl, 31);
                my_ties = my_ties > seen ? my_ties - seen : 0;
                continue;
            }
            const int f = __ffs(hit) - 1;
            target -= __shfl_sync(0xffffffffu, m_incl - m, f);
            my_ties = __shfl_sync(0xffffffffu, left, f);
            // inside block b0 + f every lane takes 16 consecutive positions
            const int pos0 = (b0 + f) * SMP_BLK + lane * (SMP_BLK / 32);
            const T* x = reinterpret_cast<const T*>(data) + pos0;
            u64 lt = 0;
            for (int i = 0; i < SMP_BLK / 32; ++i) lt += ties && float(x[i]) == cut.tie;
            const u64 lt_excl = warp_scan_u64(lt, lane) - lt;
            const u64 lane_ties = my_ties > lt_excl ? my_ties - lt_excl : 0;
            // the running sum over the lane's kept positions; returns the first that exceeds the target, or -1
            auto walk = [&](u64& run, bool stop) -> int {
                u64 seen = 0;
                for (int i = 0; i < SMP_BLK / 32; ++i) {
                    const float l = float(x[i]);
                    if (l > cut.above) run += weight(l);
                    else if (ties && l == cut.tie && seen++ < lane_ties) run += w_tie;
                    if (stop && run > target) return i;
                }
                return -1;
            };
            u64 lm = 0;
            walk(lm, false);
            const u64 incl = warp_scan_u64(lm, lane);
            const unsigned lane_hit = __ballot_sync(0xffffffffu, incl > target);
            if (lane == __ffs(lane_hit) - 1) {
                u64 run = incl - lm;
                const int i = walk(run, true);
                write(token_at(pos0 + i), log_share(float(x[i]), total));
            }
            break;
        }
    }

    __device__ __forceinline__ void run() {
        if (tid < SMP_TABLE) sm.table[tid] = exp2(double(tid) / SMP_TABLE);
        if (tid == 0) sm.n_local = sm.n_list = sm.base = 0;
        // the row's settings (the same in every thread, so the branches are uniform over the cluster)
        temp = p.temperature ? double(p.temperature[row]) : p.temperature_all;
        k = p.top_k ? p.top_k[row] : p.top_k_all;
        top_p = p.top_p ? double(p.top_p[row]) : p.top_p_all;
        const double min_p = p.min_p ? double(p.min_p[row]) : p.min_p_all;
        u = p.u[row];
        if (k <= 0 || k >= p.V) k = 0;
        load();
        if (!(mx > -INFINITY)) {  // nothing to draw from
            if (rank == 0 && tid == 0) write(-1, -INFINITY);
            return;
        }
        if (!(temp > 0.0) || k == 1) {
            greedy();
            return;
        }
        const double k2 = 1.4426950408889634074 / temp;  // exponents of 2 per unit of logit
        weight.m = double(mx);
        weight.peak = mx;
        weight.scale = SMP_TABLE * k2;
        weight.table = sm.table;
        weight.frac = p.frac_bits;
        if (warp == 0) {
            const double x = lane == 1 && min_p > 0.0 ? fmax(SMP_FLOOR_LOG2, log2(fmin(min_p, 1.0))) : SMP_FLOOR_LOG2;
            const float l = lowest_with(x, k2);
            if (lane == 0) sm.l_floor = l;
            if (lane == 1) sm.l_min = l;
        }
        __syncthreads();
        l_floor = sm.l_floor;
        l_min = sm.l_min;
        const bool want_p = top_p < 1.0;
        if (!k && !want_p) {
            draw(Cut{-INFINITY, 0.0f, 0});
            return;
        }
        bin_scale = fminf(float(SMP_BINS) / (0.5f * mx - 0.5f * l_floor), 1e30f);
        const bool by_mass = !k;  // top-k comes first: its counts decide
        level0(by_mass);
        u64 mass = 0, cnt = 0;
        for (int r = 0; r < size; ++r) {
            mass += got(0, r);
            cnt += got(1, r);
        }
        u64 target;
        if (by_mass) {
            const double t = ceil(fmax(top_p, 0.0) * double(mass));
            target = t < 1.0 ? 1ull : min((u64)t, mass);
        } else {
            target = min(u64(k), cnt);
        }
        const Border bd = find_border(by_mass, target, 0, 0);
        if (bd.cnt_above + bd.cnt <= SMP_LIST) {
            finish_on_list(bd.bin, bd.owner, mass);
            return;
        }
        if (by_mass)
            draw(cut_by_levels(bd, true, 0, target));
        else
            draw(cut_by_levels(bd, false, u64(k) < cnt ? u64(k) : 0, 0));
    }
};

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 2)
sample_kernel(const SampleParams p) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SmpShared sm;
    Sampler<T> s(p, sm, dyn);
    s.run();
}

}  // namespace cce
