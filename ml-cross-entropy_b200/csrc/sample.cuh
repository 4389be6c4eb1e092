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
// from HBM once and every later pass runs on chip.  No sort: a threshold (the k-th largest logit, or the
// logit where the mass reaches p) is found by a histogram of counts and masses over the slice, first
// linear in the logit between the maximum and the 2^-40 floor, then over the order-preserving integer keys of
// the bin that holds the threshold, until the bin is a single value; ties at that value are kept by index.
#pragma once
#include <cooperative_groups.h>
#include "engine.cuh"

namespace cce {

constexpr int SMP_THREADS = 512;
constexpr int SMP_WARPS = SMP_THREADS / 32;
constexpr int SMP_BINS = 2048;
constexpr int SMP_BLK = 512;         // positions per block of the final index-ordered search (16 per lane)
constexpr int SMP_MAX_CLUSTER = 8;
constexpr int SMP_SMEM = 225 * 1024;  // dynamic shared memory at most: of the 227 KB of a CTA, the rest is static
constexpr float SMP_FLOOR_LOG2 = -40.0f;

// One of the four settings: an array with a value per row, or one value for all rows.
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

// The integer order of floats (descending helpers below work on these keys); +0 and -0 share a key.
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
// (l - m) * 32 log2(e) / T = 32 n + j + r with |r| <= 1/2, so the weight is 2^n * 2^(j/32) * e^z with
// z = r ln2 / 32, |z| < 0.011, and five terms of the Taylor series leave a relative error of z^6/720 < 3e-15.
// The product is added to 2^52, whose low bits then hold the rounded integer.
struct WeightFn {
    double m, k32;        // maximum, 32 * log2(e) / T
    const double* table;  // shared memory: 2^(j/32), j < 32
    int frac;
    float peak;           // m as it is stored
    __device__ __forceinline__ unsigned long long operator()(float l) const {
        if (l == peak) return 1ull << frac;  // also where the maximum is infinite
        constexpr double c = 0.02166084939249829;  // ln2 / 32
        constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
        const double d = double(l) - m;
        const double t = fma(d, k32, magic);
        const int i = __double2loint(t);
        const double r = fma(d, k32, magic - t);
        double e = fma(r, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
        e = fma(e, r, c * c * c / 6.0);
        e = fma(e, r, c * c / 2.0);
        e = fma(e, r, c);
        e = fma(e, r, 1.0);
        const double tab = table[i & 31];
        const double scaled = __hiloint2double(__double2hiint(tab) + ((i >> 5) + frac) * (1 << 20), __double2loint(tab));
        const double w = fma(e, scaled, 4503599627370496.0);  // 2^52
        return (unsigned long long)__double_as_longlong(w) & 0xfffffffffffffull;
    }
};

// Positions with l > above are kept, and the first n_tie (in index order) of those with l == tie.
struct Cut {
    float above, tie;
    long long n_tie;
};

// The dynamic shared memory of a CTA, in bytes from its start.
struct SampleLayout {
    int share;     // bins whose cluster-wide sums this CTA forms
    int max_blk;   // blocks of SMP_BLK positions a slice can touch (one more than it holds, by its alignment)
    int hist_mass, own_mass, own_cnt, lv_mass, lv_cnt, blk_mass, hist_cnt, blk_tie, data, bytes;
    __host__ __device__ SampleLayout(int cluster, int slice, int elem_bytes) {
        share = SMP_BINS / cluster;
        max_blk = slice / SMP_BLK + 1;
        int o = 0;
        hist_mass = o, o += SMP_BINS * 8;
        own_mass = o, o += share * 8;  // level 0, kept for the second threshold
        own_cnt = o, o += share * 8;
        lv_mass = o, o += share * 8;   // the levels below it
        lv_cnt = o, o += share * 8;
        blk_mass = o, o += max_blk * 8;
        hist_cnt = o, o += SMP_BINS * 4;
        blk_tie = o, o += max_blk * 4;
        data = (o + 15) / 16 * 16;
        bytes = data + max_blk * SMP_BLK * elem_bytes;
    }
};

struct SmpShared {
    double table[32];
    unsigned long long xa[2][SMP_MAX_CLUSTER], xb[2][SMP_MAX_CLUSTER];  // exchange slots, written by the whole cluster
    unsigned long long xc[2][SMP_MAX_CLUSTER];
    unsigned long long wa[SMP_WARPS], wb[SMP_WARPS];
    unsigned long long ra, rb, rc, rd;
    float wf[SMP_WARPS];
};

template <typename T>
struct RowSlice {
    const uint4* data;  // shared memory, SMP_BLK-position blocks; positions outside the slice hold -inf
    int n_blk;
    static constexpr int VE = 16 / int(sizeof(T));
    static constexpr int CHUNKS = SMP_BLK / VE / 32;  // 16-byte chunks per lane and block
    // f(l, position) for every position of block b, a warp together
    template <typename F>
    __device__ __forceinline__ void each(int b, int lane, F f) const {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int q = (b * CHUNKS + c) * 32 + lane;
            const uint4 u = data[q];
            const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < VE; ++i) f(float(x[i]), q * VE + i);
        }
    }
};

__device__ __forceinline__ unsigned long long warp_sum_u64(unsigned long long v) {
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) v += __shfl_xor_sync(0xffffffffu, v, o);
    return v;
}
__device__ __forceinline__ unsigned long long warp_scan_u64(unsigned long long v, int lane) {  // inclusive
#pragma unroll
    for (int o = 1; o < 32; o <<= 1) {
        const unsigned long long t = __shfl_up_sync(0xffffffffu, v, o);
        if (lane >= o) v += t;
    }
    return v;
}

// The cluster's three-value exchange: thread 0 of each CTA gives (a, b, c), everyone reads all of them
// in sm.x?[buf][rank].  Two buffers: a CTA that runs ahead writes the other one, and cannot come back to
// this one before every CTA has passed the next barrier, hence read this one.
struct Exchange {
    cooperative_groups::cluster_group cl;
    SmpShared* sm;
    int rank, size, buf;
    __device__ __forceinline__ void operator()(unsigned long long a, unsigned long long b, unsigned long long c) {
        buf ^= 1;
        if (threadIdx.x < unsigned(size)) {
            SmpShared* dst = cl.map_shared_rank(sm, threadIdx.x);
            dst->xa[buf][rank] = a;
            dst->xb[buf][rank] = b;
            dst->xc[buf][rank] = c;
        }
        cl.sync();
    }
};

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS)
sample_kernel(const SampleParams p) {
    namespace cg = cooperative_groups;
    constexpr int VE = 16 / int(sizeof(T));
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SmpShared sm;
    cg::cluster_group cl = cg::this_cluster();
    const int rank = int(cl.block_rank()), size = int(cl.num_blocks());
    const int tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const long long row = blockIdx.x / size;

    const SampleLayout lay(size, p.slice, int(sizeof(T)));
    const int share = lay.share;
    unsigned long long* hist_mass = reinterpret_cast<unsigned long long*>(dyn + lay.hist_mass);
    unsigned long long* own_mass = reinterpret_cast<unsigned long long*>(dyn + lay.own_mass);
    unsigned long long* own_cnt = reinterpret_cast<unsigned long long*>(dyn + lay.own_cnt);
    unsigned long long* lv_mass = reinterpret_cast<unsigned long long*>(dyn + lay.lv_mass);
    unsigned long long* lv_cnt = reinterpret_cast<unsigned long long*>(dyn + lay.lv_cnt);
    unsigned long long* blk_mass = reinterpret_cast<unsigned long long*>(dyn + lay.blk_mass);
    uint32_t* hist_cnt = reinterpret_cast<uint32_t*>(dyn + lay.hist_cnt);
    uint32_t* blk_tie = reinterpret_cast<uint32_t*>(dyn + lay.blk_tie);
    uint4* data = reinterpret_cast<uint4*>(dyn + lay.data);

    // ---- the slice: positions are counted from the 16-byte boundary at or below its first element, so
    // that whole 16-byte pieces of global memory land on 16-byte pieces of shared memory at any alignment
    const long long start = (long long)rank * p.slice;
    const int n = int(max(0ll, min((long long)p.slice, p.V - start)));
    const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ld + start;
    const int phase = int((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
    RowSlice<T> rs;
    rs.data = data;
    rs.n_blk = n > 0 ? (n + phase + SMP_BLK - 1) / SMP_BLK : 0;
    float mx = -INFINITY;
    {
        const T lowest = T(-INFINITY);
        const T* src0 = src - phase;
        const int n_chunk = rs.n_blk * (SMP_BLK / VE);
        for (int q = tid; q < n_chunk; q += SMP_THREADS) {
            const int first = q * VE;
            uint4 v;
            T* x = reinterpret_cast<T*>(&v);
            if (first >= phase && first + VE <= phase + n) {
                v = __ldg(reinterpret_cast<const uint4*>(src0 + first));
            } else {
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    x[i] = (first + i >= phase && first + i < phase + n) ? src0[first + i] : lowest;
            }
            data[q] = v;
#pragma unroll
            for (int i = 0; i < VE; ++i) mx = fmaxf(mx, float(x[i]));  // drops NaN
        }
    }
    if (tid < 32) sm.table[tid] = exp2(double(tid) / 32.0);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    if (lane == 0) sm.wf[warp] = mx;
    cl.sync();  // every CTA of the cluster runs: its shared memory may be written from now on
    if (warp == 0) {
        mx = lane < SMP_WARPS ? sm.wf[lane] : -INFINITY;
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) mx = fmaxf(mx, __shfl_xor_sync(0xffffffffu, mx, o));
    }
    Exchange xch{cl, &sm, rank, size, 0};
    xch(__float_as_uint(mx), 0, 0);
    mx = -INFINITY;
    for (int r = 0; r < size; ++r) mx = fmaxf(mx, __uint_as_float(uint32_t(sm.xa[xch.buf][r])));
    mx += 0.0f;

    // the row's settings (the same in every thread, so the branches below are uniform over the cluster)
    const double temp = p.temperature ? double(p.temperature[row]) : p.temperature_all;
    long long k = p.top_k ? p.top_k[row] : p.top_k_all;
    const double top_p = p.top_p ? double(p.top_p[row]) : p.top_p_all;
    const double min_p = p.min_p ? double(p.min_p[row]) : p.min_p_all;
    const float u = p.u ? p.u[row] : 0.0f;
    if (k <= 0 || k >= p.V) k = 0;

    if (!(mx > -INFINITY)) {  // nothing to draw from
        if (rank == 0 && tid == 0) {
            p.tokens[row] = -1;
            if (p.logprobs) p.logprobs[row] = -INFINITY;
        }
        return;
    }
    if (!(temp > 0.0) || k == 1) {  // the first of the largest
        uint32_t best = 0xffffffffu;
        for (int b = warp; b < rs.n_blk; b += SMP_WARPS)
            rs.each(b, lane, [&](float l, int pos) {
                if (l == mx) best = min(best, uint32_t(pos - phase));
            });
        best = __reduce_min_sync(0xffffffffu, best);
        if (lane == 0) sm.wa[warp] = best;
        __syncthreads();
        best = 0xffffffffu;
        for (int w = 0; w < SMP_WARPS; ++w) best = min(best, uint32_t(sm.wa[w]));
        xch(best, 0, 0);
        if (rank == 0 && tid == 0) {
            long long token = -1;
            for (int r = size - 1; r >= 0; --r) {
                const uint32_t b = uint32_t(sm.xa[xch.buf][r]);
                if (b != 0xffffffffu) token = (long long)r * p.slice + b;
            }
            p.tokens[row] = token;
            if (p.logprobs) p.logprobs[row] = 0.0f;
        }
        return;
    }

    WeightFn weight;
    weight.m = double(mx);
    weight.peak = mx;
    const double k2 = 1.4426950408889634074 / temp;  // exponents of 2 per unit of logit
    weight.k32 = 32.0 * k2;
    weight.table = sm.table;
    weight.frac = p.frac_bits;

    // the smallest logit whose weight is at least 2^x (x <= 0): a first guess, then the neighbours.  A weight
    // that rounds to 1 in fp64, exp(z) with z >= -2^-54, counts as 1.
    auto lowest_with = [&](double x) -> float {
        if (isinf(mx)) return mx;
        x = fmin(x, -8.0e-17);  // -2^-54 log2(e)
        float g = float(double(mx) + x / k2);
        if (!(g > -3.402823466e38f)) g = -3.402823466e38f;
        for (int it = 0; it < 4 && g < mx && (double(g) - double(mx)) * k2 < x; ++it) g = order_value(order_key(g) + 1);
        for (int it = 0; it < 4 && g > -3.402823466e38f; ++it) {
            const float below = just_below(g);
            if ((double(below) - double(mx)) * k2 < x) break;
            g = below;
        }
        return g;
    };
    const float l_floor = lowest_with(double(SMP_FLOOR_LOG2));
    const float l_min = min_p > 0.0 ? fmaxf(l_floor, lowest_with(log2(fmin(min_p, 1.0)))) : l_floor;
    Cut cut{-INFINITY, 0.0f, 0};
    const bool want_p = top_p < 1.0;

    if (k || want_p) {
        // ---- level 0 of the histogram: bins linear in the logit, bin 0 at the maximum
        const float span = 0.5f * mx - 0.5f * l_floor;  // halves: the difference of two floats may overflow
        const float per = fminf(float(SMP_BINS) / span, 1e30f);
        auto bin0 = [&](float l) -> int { return min(SMP_BINS - 1, int((0.5f * mx - 0.5f * l) * per)); };
        auto clear_hist = [&]() {
            for (int b = tid; b < SMP_BINS; b += SMP_THREADS) {
                hist_mass[b] = 0;
                hist_cnt[b] = 0;
            }
            __syncthreads();
        };
        // Counts and masses of the bins over the cluster: this CTA's share to (mass, cnt), its totals to everyone.
        auto merge_hist = [&](unsigned long long* mass, unsigned long long* cnt) {
            cl.sync();  // all histograms are complete
            unsigned long long tm = 0, tc = 0;
            for (int b = tid; b < share; b += SMP_THREADS) {
                unsigned long long sm_ = 0, sc = 0;
                for (int r = 0; r < size; ++r) {
                    sm_ += cl.map_shared_rank(hist_mass, r)[rank * share + b];
                    sc += cl.map_shared_rank(hist_cnt, r)[rank * share + b];
                }
                mass[b] = sm_;
                cnt[b] = sc;
                tm += sm_;
                tc += sc;
            }
            tm = warp_sum_u64(tm);
            tc = warp_sum_u64(tc);
            if (lane == 0) {
                sm.wa[warp] = tm;
                sm.wb[warp] = tc;
            }
            __syncthreads();
            tm = tc = 0;
            for (int w = 0; w < SMP_WARPS; ++w) {
                tm += sm.wa[w];
                tc += sm.wb[w];
            }
            xch(tm, tc, 0);
        };
        // The bin where the running count (by_mass: mass) from the top reaches `target`; in all CTAs:
        // bin, and the count and mass above it.  Uses the totals that merge_hist left in the exchange.
        struct Border {
            int bin;
            unsigned long long mass_above, cnt_above;
        };
        auto find_border = [&](const unsigned long long* mass, const unsigned long long* cnt,
                               const unsigned long long (&tot_m)[SMP_MAX_CLUSTER],
                               const unsigned long long (&tot_c)[SMP_MAX_CLUSTER], bool by_mass,
                               unsigned long long target, unsigned long long base_m, unsigned long long base_c) -> Border {
            unsigned long long am = base_m, ac = base_c;
            int owner = size - 1;
            for (int r = 0; r < size; ++r) {
                if ((by_mass ? am + tot_m[r] : ac + tot_c[r]) >= target) {
                    owner = r;
                    break;
                }
                if (r + 1 < size) {
                    am += tot_m[r];
                    ac += tot_c[r];
                }
            }
            if (rank == owner && warp == 0) {
                int found = share - 1;
                for (int b0 = 0; b0 < share; b0 += 32) {
                    const unsigned long long vm = mass[b0 + lane], vc = cnt[b0 + lane];
                    const unsigned long long im = warp_scan_u64(vm, lane), ic = warp_scan_u64(vc, lane);
                    const unsigned hit = __ballot_sync(0xffffffffu, (by_mass ? am + im : ac + ic) >= target);
                    if (hit || b0 + 32 >= share) {
                        const int first = hit ? __ffs(hit) - 1 : 31;
                        found = b0 + first;
                        am += __shfl_sync(0xffffffffu, im - vm, first);
                        ac += __shfl_sync(0xffffffffu, ic - vc, first);
                        break;
                    }
                    am += __shfl_sync(0xffffffffu, im, 31);
                    ac += __shfl_sync(0xffffffffu, ic, 31);
                }
                if (lane == 0) {
                    sm.ra = (unsigned long long)(owner * share + found);
                    sm.rb = am;
                    sm.rc = ac;
                }
            }
            __syncthreads();
            xch(sm.ra, sm.rb, sm.rc);
            return Border{int(sm.xa[xch.buf][owner]), sm.xb[xch.buf][owner], sm.xc[xch.buf][owner]};
        };

        clear_hist();
        for (int b = warp; b < rs.n_blk; b += SMP_WARPS)
            rs.each(b, lane, [&](float l, int) {
                if (l >= l_floor) {
                    const int bin = bin0(l);
                    atomicAdd(&hist_cnt[bin], 1u);
                    if (want_p) atomicAdd(&hist_mass[bin], weight(l));
                }
            });
        merge_hist(own_mass, own_cnt);
        unsigned long long tot_m[SMP_MAX_CLUSTER], tot_c[SMP_MAX_CLUSTER];
        unsigned long long n_all = 0, m_all = 0;
        for (int r = 0; r < SMP_MAX_CLUSTER; ++r) {
            tot_m[r] = r < size ? sm.xa[xch.buf][r] : 0;
            tot_c[r] = r < size ? sm.xb[xch.buf][r] : 0;
            m_all += tot_m[r];
            n_all += tot_c[r];
        }

        // From the level-0 border down to one value.  On return: that value, the count and the mass
        // above it, in every thread of the cluster.
        struct Level {
            float value;
            unsigned long long mass_above, cnt_above;
        };
        auto descend = [&](bool by_mass, unsigned long long target) -> Level {
            Border bd = find_border(own_mass, own_cnt, tot_m, tot_c, by_mass, target, 0, 0);
            // the keys of level-0 bin bd.bin: bin0 falls as the key grows
            uint32_t lo, hi;
            {
                const uint32_t kmin = order_key(l_floor), kmax = order_key(mx);
                uint32_t a = kmin, b = kmax;  // smallest key with bin0 <= bin
                while (a < b) {
                    const uint32_t mid = a + (b - a) / 2;
                    if (bin0(order_value(mid)) <= bd.bin) b = mid; else a = mid + 1;
                }
                lo = a;
                a = lo, b = kmax;  // largest key with bin0 >= bin
                while (a < b) {
                    const uint32_t mid = b - (b - a) / 2;
                    if (bin0(order_value(mid)) >= bd.bin) a = mid; else b = mid - 1;
                }
                hi = a;
            }
            while (hi > lo) {
                const int bits = 32 - __clz(hi - lo);
                const int shift = max(0, bits - 11);  // (hi - lo) >> shift < 2048
                const float f_lo = order_value(lo), f_hi = order_value(hi);
                clear_hist();
                for (int b = warp; b < rs.n_blk; b += SMP_WARPS)
                    rs.each(b, lane, [&](float l, int) {
                        if (l >= f_lo && l <= f_hi) {
                            const int bin = int((hi - order_key(l)) >> shift);
                            atomicAdd(&hist_cnt[bin], 1u);
                            if (by_mass) atomicAdd(&hist_mass[bin], weight(l));
                        }
                    });
                merge_hist(lv_mass, lv_cnt);
                unsigned long long lm[SMP_MAX_CLUSTER], lc[SMP_MAX_CLUSTER];
                for (int r = 0; r < SMP_MAX_CLUSTER; ++r) {
                    lm[r] = r < size ? sm.xa[xch.buf][r] : 0;
                    lc[r] = r < size ? sm.xb[xch.buf][r] : 0;
                }
                bd = find_border(lv_mass, lv_cnt, lm, lc, by_mass, target, bd.mass_above, bd.cnt_above);
                const uint32_t top = hi - (uint32_t(bd.bin) << shift);
                lo = max(lo, top - ((1u << shift) - 1));
                hi = top;
            }
            return Level{order_value(lo), bd.mass_above, bd.cnt_above};
        };

        unsigned long long kept_mass = m_all;  // mass of the top-k (used by top-p only)
        if (k && (unsigned long long)k < n_all) {
            const Level lv = descend(false, (unsigned long long)k);
            cut.above = lv.value;
            cut.tie = lv.value;
            cut.n_tie = k - (long long)lv.cnt_above;
            if (want_p) {
                // mass above lv.value: the levels carried counts only, so take it from one more pass
                unsigned long long s = 0;
                for (int b = warp; b < rs.n_blk; b += SMP_WARPS)
                    rs.each(b, lane, [&](float l, int) {
                        if (l > lv.value) s += weight(l);
                    });
                s = warp_sum_u64(s);
                __syncthreads();
                if (lane == 0) sm.wa[warp] = s;
                __syncthreads();
                s = 0;
                for (int w = 0; w < SMP_WARPS; ++w) s += sm.wa[w];
                xch(s, 0, 0);
                kept_mass = (unsigned long long)cut.n_tie * weight(lv.value);
                for (int r = 0; r < size; ++r) kept_mass += sm.xa[xch.buf][r];
            }
        }
        if (want_p) {
            // the first n whose mass reaches p * kept_mass, at least one
            double t = ceil(fmax(top_p, 0.0) * double(kept_mass));
            unsigned long long target = t < 1.0 ? 1ull : (unsigned long long)t;
            target = min(target, kept_mass);
            const Level lv = descend(true, target);
            const unsigned long long w = weight(lv.value);
            const long long need = lv.mass_above >= target ? 0ll : (long long)((target - lv.mass_above + w - 1) / w);
            const long long limit = lv.value == cut.tie && cut.n_tie > 0 ? cut.n_tie : need;
            cut.above = lv.value;
            cut.tie = lv.value;
            cut.n_tie = min(need, limit);
        }
    }
    // the min-p prefix
    if (cut.n_tie > 0 && cut.tie < l_min) cut.n_tie = 0;
    cut.above = fmaxf(cut.above, just_below(l_min));

    // ---- masses of the kept positions by block, ties counted apart
    unsigned long long sum_m = 0;
    uint32_t sum_t = 0;
    const bool ties = cut.n_tie > 0;
    __syncthreads();
    for (int b = warp; b < rs.n_blk; b += SMP_WARPS) {
        unsigned long long bm = 0;
        uint32_t bt = 0;
        rs.each(b, lane, [&](float l, int) {
            if (l > cut.above) bm += weight(l);
            if (ties && l == cut.tie) ++bt;
        });
        bm = warp_sum_u64(bm);
        bt = __reduce_add_sync(0xffffffffu, bt);
        if (lane == 0) {
            blk_mass[b] = bm;
            blk_tie[b] = bt;
        }
        sum_m += bm;
        sum_t += bt;
    }
    if (lane == 0) {
        sm.wa[warp] = sum_m;
        sm.wb[warp] = sum_t;
    }
    __syncthreads();
    sum_m = 0;
    unsigned long long sum_tt = 0;
    for (int w = 0; w < SMP_WARPS; ++w) {
        sum_m += sm.wa[w];
        sum_tt += sm.wb[w];
    }
    xch(sum_m, sum_tt, 0);

    // ---- which CTA, which block, which position
    const unsigned long long w_tie = ties ? weight(cut.tie) : 0;
    unsigned long long total = 0, before = 0, mine = 0, ties_left = (unsigned long long)cut.n_tie, my_ties_left = 0;
    for (int r = 0; r < size; ++r) {
        const unsigned long long t = min(sm.xb[xch.buf][r], ties_left);
        const unsigned long long m = sm.xa[xch.buf][r] + t * w_tie;
        if (r == rank) {
            before = total;
            mine = m;
            my_ties_left = ties_left;
        }
        total += m;
        ties_left -= t;
    }
    const double x = double(u) * double(total);
    unsigned long long target = 0;
    if (x > 0.0) target = x >= double(total) ? total - 1 : (unsigned long long)x;
    if (target >= total) target = total - 1;
    if (target < before || target >= before + mine || warp != 0) return;  // the owner's first warp goes on
    target -= before;
    unsigned long long tl = my_ties_left;
    for (int b0 = 0; b0 < rs.n_blk; b0 += 32) {
        const int b = b0 + lane;
        const unsigned long long t = b < rs.n_blk && ties ? blk_tie[b] : 0;
        const unsigned long long t_incl = warp_scan_u64(t, lane), t_excl = t_incl - t;
        const unsigned long long left = tl > t_excl ? tl - t_excl : 0;  // ties that this block may still keep
        const unsigned long long m = (b < rs.n_blk ? blk_mass[b] : 0) + min(t, left) * w_tie;
        const unsigned long long m_incl = warp_scan_u64(m, lane);
        const unsigned hit = __ballot_sync(0xffffffffu, m_incl > target);
        if (!hit) {
            target -= __shfl_sync(0xffffffffu, m_incl, 31);
            const unsigned long long seen = __shfl_sync(0xffffffffu, t_incl, 31);
            tl = tl > seen ? tl - seen : 0;
            continue;
        }
        const int f = __ffs(hit) - 1;
        target -= __shfl_sync(0xffffffffu, m_incl - m, f);
        tl = __shfl_sync(0xffffffffu, left, f);
        // inside block b0 + f: every lane takes 16 consecutive positions
        const T* x16 = reinterpret_cast<const T*>(data) + (size_t)(b0 + f) * SMP_BLK + lane * (SMP_BLK / 32);
        unsigned long long lt = 0;
        for (int i = 0; i < SMP_BLK / 32; ++i) lt += ties && float(x16[i]) == cut.tie;
        const unsigned long long lt_excl = warp_scan_u64(lt, lane) - lt;
        const unsigned long long lane_left = tl > lt_excl ? tl - lt_excl : 0;
        unsigned long long lm = 0, tk = 0;
        for (int i = 0; i < SMP_BLK / 32; ++i) {
            const float l = float(x16[i]);
            if (l > cut.above) lm += weight(l);
            else if (ties && l == cut.tie && tk++ < lane_left) lm += w_tie;
        }
        const unsigned long long lm_incl = warp_scan_u64(lm, lane);
        const unsigned lane_hit = __ballot_sync(0xffffffffu, lm_incl > target);
        if (lane == __ffs(lane_hit) - 1) {
            unsigned long long run = lm_incl - lm;
            tk = 0;
            for (int i = 0; i < SMP_BLK / 32; ++i) {
                const float l = float(x16[i]);
                if (l > cut.above) run += weight(l);
                else if (ties && l == cut.tie && tk++ < lane_left) run += w_tie;
                if (run > target) {
                    p.tokens[row] = start + (long long)(b0 + f) * SMP_BLK + lane * (SMP_BLK / 32) + i - phase;
                    if (p.logprobs) {
                        const double y = l == mx ? 0.0 : (double(l) - double(mx)) / temp;
                        p.logprobs[row] = float(y - log(double(total) * exp2(-double(p.frac_bits))));
                    }
                    break;
                }
            }
        }
        break;
    }
}

}  // namespace cce
