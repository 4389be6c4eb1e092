// One token per row of logits: temperature, top-k, top-p, min-p, and a draw from a given uniform number.
//
//   w_v = exp((l_v - m) / T), m = max l;  w = 1 where l_v = m, 0 where l_v is NaN or -inf or w < 2^-40
//   order: l descending, ties by the lower index; kept = the shortest of three prefixes of it:
//     the first k;  the first n whose weights reach p * (sum over the first k);  those with w >= min_p
//   token = the first kept v, in order of v, whose running sum of weights exceeds u * (sum kept)
//
// With 2^18 tokens of a flat distribution the running sums are 4e-6 apart, so fp32 sums would move
// the draw.  The weights are evaluated in fp64 and rounded to fixed point (a unit of 2^-46..2^-42 of the
// largest, so that V of them fit 63 bits): integer sums are exact in any order, hence the token
// depends neither on the split of the row nor on the order of the atomics below.
//
// A row is one cluster of CTAs; each keeps its slice of the row in shared memory, so the logits are read
// from HBM once and every later pass runs on chip.  The row is never sorted as a whole.  With top-k or top-p a
// histogram of counts, linear in the logit between the maximum and the 2^-40 floor, tells where the border lies:
// the bin of the k-th logit exactly, the bin where the mass reaches p to within the width of a bin (the exact sum of all
// weights is formed in the same pass; exact masses per bin would need 64-bit atomics, 1.5 cycles per logit).
//  - At most SMP_LIST logits down to the border: they are gathered into one CTA, sorted, and the rest
//    is done on that list.
//  - top-p with more: the logits of some bins around the estimate are gathered and sorted, the weights above them are
//    summed exactly (by blocks, which the draw needs anyway), and the border is found, exactly, in the list.
//  - Otherwise (a large k, thousands of equal logits, an estimate that was off): further histograms narrow the
//    border down over the integer keys of its bin until it is a single value.
// A cluster barrier costs 0.5 to 0.8 us, a pass over a slice of 16384 logits 1 to 3 us: five to seven barriers are 3 to 5
// of the 17 us that 1 x 256000 fp32 with all filters takes on the device (64 x 128256 bf16, top-k and top-p: 34 us); how
// the rest divides among the passes has not been measured.  Throughput is the fp64 weights (0.4 cycles per logit and SM) and
// the atomics (0.3).
#pragma once
#include <cooperative_groups.h>
#include "engine.cuh"
#include "ptx_pair.cuh"

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

constexpr int SMP_TABLE = 16;
constexpr int SMP_MAX_FRAC = 46;

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
    double table[SMP_TABLE];  // see WeightFn
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
// (l - m) * 16 log2(e) / T = 16 n + j + r with |r| <= 1/2, so the weight is 2^n * 2^(j/16) * e^z with
// z = r ln2 / 16, |z| < 0.022, and five terms of the Taylor series leave a relative error of
// z^6/720 < 1.5e-13, about the rounding to 2^-43.  The product is added to 2^52, whose low bits then
// hold the rounded integer.  16 entries of 8 bytes are what the 32 banks serve at once, whichever the lanes ask for.
// The exponent n reaches the table's value by one addition: i << 16 is n << 20 plus j << 16, and the entry of j has
// that taken off.  A pass over every weight is bound by issuing its instructions (51 per logit with a branch for each and
// 64-bit integer sums, about 22 as below): the sums are kept in fp64, exact while 128 weights of at most 2^46 meet.
struct WeightFn {
    double m, scale;  // maximum (the largest finite number for an infinite one), 16 * log2(e) / T
    uint32_t table;   // shared memory: SampleParams::table
    // its entry j, on the host: 2^(frac + j/16), less j << 16 in its high word
    static double entry(int j, int frac) {
        const double x = exp2(double(j) / SMP_TABLE + double(frac));
        long long b;
        memcpy(&b, &x, 8);
        b -= (long long)j << 48;
        double y;
        memcpy(&y, &b, 8);
        return y;
    }
    // the rounded weight + 2^52; for m - l beyond the floor (or NaN, -inf) the result means nothing
    __device__ __forceinline__ double raised(float l) const {
        constexpr double c = 0.043321698784996581;    // ln2 / 16
        constexpr double magic = 6755399441055744.0;  // 1.5 * 2^52: adding it rounds to an integer
        const double d = double(fminf(l, -SMP_LOWEST)) - m;
        const double t = fma(d, scale, magic);
        const int i = __double2loint(t);
        const double r = fma(d, scale, magic - t);
        double e = fma(r, c * c * c * c * c / 120.0, c * c * c * c / 24.0);
        e = fma(e, r, c * c * c / 6.0);
        e = fma(e, r, c * c / 2.0);
        e = fma(e, r, c);
        e = fma(e, r, 1.0);
        double tab;
        asm("ld.shared.f64 %0, [%1];" : "=d"(tab) : "r"(table + ((i << 3) & ((SMP_TABLE - 1) << 3))));
        const double scaled = __hiloint2double(__double2hiint(tab) + i * (1 << 16), __double2loint(tab));
        return fma(e, scaled, 4503599627370496.0);
    }
    __device__ __forceinline__ u64 operator()(float l) const {
        return (u64)__double_as_longlong(raised(l)) & 0xfffffffffffffull;
    }
    // adds the weights of those of N logits that are at least `from` to sum; a warp together
    template <int N>
    __device__ __forceinline__ void sum_weights(const float (&l)[N], float from, double& sum) const {
        bool any = false;
#pragma unroll
        for (int i = 0; i < N; ++i) any |= l[i] >= from;
        if (__any_sync(0xffffffffu, any)) {
#pragma unroll
            for (int i = 0; i < N; ++i) {
                const double w = raised(l[i]) - 4503599627370496.0;
                asm("{\n\t.reg .pred p;\n\tsetp.ge.f32 p, %2, %3;\n\t@p add.rn.f64 %0, %0, %1;\n\t}" : "+d"(sum) : "d"(w), "f"(l[i]), "f"(from));
            }
        }
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
        hist_mass = o, o += SMP_BINS * 8;  // also two lists of SMP_LIST entries
        hist_cnt = o, o += SMP_BINS * 4;   // also one list of SMP_LIST entries
        own_mass = o, o += share * 8;
        own_cnt = o, o += share * 4;
        blk_mass = o, o += max_blk * 8;
        blk_tie = o, o += max_blk * 4;
        data = (o + 15) / 16 * 16;
        bytes = data + max_blk * SMP_BLK * elem_bytes;
    }
};

// Shared memory of a CTA's sums and scans.
struct CtaScratch {
    double table[SMP_TABLE];
    u64 wa[SMP_WARPS], wb[SMP_WARPS];
    u64 r[4];
};

struct SmpShared : CtaScratch {
    u64 x[2][4][SMP_MAX_CLUSTER];  // exchange slots, written by the whole cluster
    float wf[SMP_WARPS];
    uint32_t n_local, n_list, base, key[4];
    int lo, hi, all;
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
// In-place ascending sort of n values (a power of two from 64 to 2 * SMP_THREADS) by the whole CTA: bitonic; the
// steps within 64 neighbours stay in the registers of a warp (two values per lane), so that 1024 values need 10
// steps through shared memory instead of 55.
__device__ __forceinline__ void sort_pair(u64& a, u64& b, bool ascending) {
    if ((a > b) == ascending) {
        const u64 t = a;
        a = b;
        b = t;
    }
}
__device__ __forceinline__ void bitonic_sort(u64* v, int n) {
    const int tid = threadIdx.x, lane = tid & 31, e0 = (tid >> 5) * 64 + lane;
    const bool active = e0 < n;  // uniform over the warp
    u64 a = 0, b = 0;
    // the steps j = 32 .. 1 of stage k on the warp's 64 values
    auto inner = [&](int k) {
        for (int j = min(32, k >> 1); j > 0; j >>= 1) {
            if (j == 32) {
                sort_pair(a, b, (e0 & k) == 0);
            } else {
                const u64 pa = __shfl_xor_sync(0xffffffffu, a, j), pb = __shfl_xor_sync(0xffffffffu, b, j);
                const bool low = (lane & j) == 0;
                const bool up_a = (e0 & k) == 0, up_b = ((e0 + 32) & k) == 0;
                a = ((a < pa) == (up_a == low)) ? a : pa;
                b = ((b < pb) == (up_b == low)) ? b : pb;
            }
        }
    };
    __syncthreads();
    if (active) {
        a = v[e0];
        b = v[e0 + 32];
        for (int k = 2; k <= 64; k <<= 1) inner(k);
        v[e0] = a;
        v[e0 + 32] = b;
    }
    for (int k = 128; k <= n; k <<= 1) {
        for (int j = k >> 1; j >= 64; j >>= 1) {
            __syncthreads();
            if (tid < n / 2) {
                const int i = 2 * tid - (tid & (j - 1));
                u64 x = v[i], y = v[i + j];
                sort_pair(x, y, (i & k) == 0);
                v[i] = x;
                v[i + j] = y;
            }
        }
        __syncthreads();
        if (active) {
            a = v[e0];
            b = v[e0 + 32];
            inner(k);
            v[e0] = a;
            v[e0 + 32] = b;
        }
    }
    __syncthreads();
}
__device__ __forceinline__ int sort_size(int n) {
    int m = 64;
    while (m < n) m *= 2;
    return m;
}

// How the kernels of sample_stream.cuh go on with a row.
enum RowMode { ROW_DONE, ROW_GREEDY, ROW_SUM, ROW_LIST, ROW_WINDOW, ROW_BY_CLUSTER };
struct RowState {
    int mode;
    float edge, last;   // ROW_WINDOW: the logits from edge on lie above the window, those from last on in it; ROW_LIST: those
                        // from last on
    unsigned first;    // ROW_GREEDY: the lowest index of the largest logits
    unsigned n_list;
    u64 mass, target;  // top-p alone: all weights, and the running sum to reach
    // RowBase::prepare's results
    double scale;
    float mx, l_floor, l_min, bin_scale;
};

// What a row's kernels share: its settings, its thresholds, and the arithmetic on them.
struct RowBase {
    const SampleParams& p;
    CtaScratch& sc;
    long long row;
    int tid, warp, lane;
    int n_bins = SMP_BINS;  // of the histogram over the logits, set before prepare
    float mx, l_floor, l_min, bin_scale;
    double temp, top_p;
    float u;
    long long k;  // 0: off
    WeightFn weight;

    __device__ __forceinline__ RowBase(const SampleParams& p_, CtaScratch& sc_, long long row_) : p(p_), sc(sc_), row(row_) {
        tid = threadIdx.x;
        warp = tid >> 5;
        lane = tid & 31;
        // the same in every thread, so that the branches on them are uniform
        temp = p.temperature ? double(p.temperature[row]) : p.temperature_all;
        k = p.top_k ? p.top_k[row] : p.top_k_all;
        top_p = p.top_p ? double(p.top_p[row]) : p.top_p_all;
        u = p.u[row];
        if (k <= 0 || k >= p.V) k = 0;
    }
    __device__ __forceinline__ bool greedy_row() const { return !(temp > 0.0) || k == 1; }
    __device__ __forceinline__ void make_table() {
        if (tid < SMP_TABLE) sc.table[tid] = p.table[tid];
    }
    // from the row's maximum (above -inf): the weights and the thresholds
    __device__ __forceinline__ void prepare(float m) {
        mx = m + 0.0f;
        const double min_p = p.min_p ? double(p.min_p[row]) : p.min_p_all;
        // exponents of 2 per unit of logit; finite, for infinity x 0 would be the largest logit's exponent
        const double k2 = 1.4426950408889634074 / fmax(temp, 1e-300);
        weight.scale = SMP_TABLE * k2;
        set_weight();
        l_floor = l_min = lowest_with(SMP_FLOOR_LOG2, k2);
        if (min_p > 0.0) l_min = fmaxf(l_floor, lowest_with(fmax(SMP_FLOOR_LOG2, log2(fmin(min_p, 1.0))), k2));
        bin_scale = fminf(float(n_bins) / (0.5f * mx - 0.5f * l_floor), 1e30f);
    }
    __device__ __forceinline__ void set_weight() {
        weight.m = double(fminf(mx, -SMP_LOWEST));
        weight.table = smem_u32(sc.table);
    }
    // the same as another kernel left it
    __device__ __forceinline__ void prepare(const RowState& st) {
        mx = st.mx;
        l_floor = st.l_floor;
        l_min = st.l_min;
        bin_scale = st.bin_scale;
        weight.scale = st.scale;
        set_weight();
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
        return min(n_bins - 1, int((0.5f * mx - 0.5f * l) * bin_scale));
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

    // The smallest logit of bins 0..bin, by all threads together
    __device__ __forceinline__ float lowest_of_bins(int bin) {
        return order_value(first_key(order_key(l_floor), order_key(mx), [&](uint32_t q) { return bin0(order_value(q)) <= bin; }));
    }
    // the running sum that top-p has to reach, of the mass it is measured by
    __device__ __forceinline__ u64 p_target(u64 mass) const {
        const double t = ceil(fmax(top_p, 0.0) * double(mass));
        return t < 1.0 ? 1ull : min((u64)t, mass);
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

    // sum of two values over the CTA's threads, in every thread
    __device__ __forceinline__ void cta_sum(u64& a, u64& b) {
        a = warp_sum_u64(a);
        b = warp_sum_u64(b);
        __syncthreads();
        if (lane == 0) {
            sc.wa[warp] = a;
            sc.wb[warp] = b;
        }
        __syncthreads();
        a = b = 0;
#pragma unroll
        for (int w = 0; w < SMP_WARPS; ++w) {
            a += sc.wa[w];
            b += sc.wb[w];
        }
    }
    // inclusive scans of two values over the CTA's threads
    __device__ __forceinline__ void cta_scan(u64& a, u64& b) {
        a = warp_scan_u64(a, lane);
        b = warp_scan_u64(b, lane);
        __syncthreads();
        if (lane == 31) {
            sc.wa[warp] = a;
            sc.wb[warp] = b;
        }
        __syncthreads();
        for (int w = 0; w < warp; ++w) {
            a += sc.wa[w];
            b += sc.wb[w];
        }
    }

    // A logit and its token as one number: ascending = falling logits, ties by the lower index.
    __device__ __forceinline__ u64 rank_key(float l, long long token) const { return u64(~order_key(l)) << 32 | u64(token); }
    static __device__ __forceinline__ float key_logit(u64 key) { return order_value(~uint32_t(key >> 32)); }

    // A logit is kept when it is not below min-p's and its key not behind the cut.
    __device__ __forceinline__ bool is_kept(float l, long long token, u64 cut, float cut_l) const {
        return l >= l_min && (l > cut_l || (l == cut_l && rank_key(l, token) <= cut));
    }
    static __device__ __forceinline__ float cut_logit(u64 cut) { return cut == ~0ull ? -INFINITY : key_logit(cut); }

    // The rest of a row on the sorted list of its n largest logits (all that any prefix can keep; list in shared memory,
    // like the two others of SMP_LIST entries): applies the three prefixes and draws.  mass: of all weights, for top-p
    // without top-k.
    __device__ __forceinline__ void draw_from_list(const u64* list, int n, u64* weights, u64* by_index, u64 mass) {
        const int n_k = k && k < n ? int(k) : n;
        u64 w[2];
        float l[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) {
            const int j = 2 * tid + i;
            l[i] = j < n_k ? key_logit(list[j]) : -INFINITY;
            w[i] = j < n_k ? weight(l[i]) : 0;
            if (j < n_k) weights[j] = w[i];
        }
        u64 cum = w[0] + w[1], above_min = u64(l[0] >= l_min) + u64(l[1] >= l_min);
        cta_scan(cum, above_min);
        if (2 * tid < n_k && 2 * tid + 2 >= n_k) sc.r[0] = cum;  // sum over the first k
        if (tid == SMP_THREADS - 1) sc.r[1] = above_min;
        __syncthreads();
        int kept = max(1, int(min(u64(n_k), sc.r[1])));
        if (top_p < 1.0) {
            const u64 target = p_target(k ? sc.r[0] : mass);
            // the first whose running sum reaches it
            int n_p = __syncthreads_count(2 * tid < n_k && cum - w[1] < target);
            n_p += __syncthreads_count(2 * tid + 1 < n_k && cum < target);
            kept = min(kept, n_p + 1);
        }
        // the kept weights' sum, and the kept candidates in order of their index
        if ((kept - 1) >> 1 == tid) sc.r[2] = (kept & 1) ? cum - w[1] : cum;
        const int m = sort_size(kept);
        for (int j = tid; j < m; j += SMP_THREADS) by_index[j] = j < kept ? (list[j] << 32 | u64(j)) : ~0ull;
        bitonic_sort(by_index, m);
        const u64 total = sc.r[2], target = draw_target(total);
        u64 v[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) v[i] = 2 * tid + i < kept ? weights[uint32_t(by_index[2 * tid + i])] : 0;
        u64 run = v[0] + v[1], unused = 0;
        cta_scan(run, unused);
        if (run > target && run - v[0] - v[1] <= target) {  // one thread
            const u64 e = by_index[2 * tid + (run - v[1] > target ? 0 : 1)];
            write((long long)(e >> 32), log_share(key_logit(list[uint32_t(e)]), total));
        }
    }

};

template <typename T>
struct Sampler : RowBase {
    static constexpr int VE = 16 / int(sizeof(T));
    static constexpr int CHUNKS = SMP_BLK / VE / 32;  // 16-byte chunks per lane and block

    SmpShared& sm;
    uint8_t* dyn;
    SampleLayout lay;
    cooperative_groups::cluster_group cl;
    int rank, size, buf = 0;
    // the slice: positions are counted from the 16-byte boundary at or below its first element, so that whole
    // 16-byte pieces of global memory land on 16-byte pieces of shared memory at any alignment; positions
    // outside the slice hold -inf
    uint4* data;
    long long start;
    int phase, n_blk;

    __device__ __forceinline__ Sampler(const SampleParams& p_, SmpShared& sm_, uint8_t* dyn_, long long row_, int cluster)
        : RowBase(p_, sm_, row_), sm(sm_), dyn(dyn_), lay(cluster, p_.slice, int(sizeof(T))),
          cl(cooperative_groups::this_cluster()) {
        rank = int(cl.block_rank());
        size = cluster;
        data = reinterpret_cast<uint4*>(dyn + lay.data);
    }
    __device__ __forceinline__ u64* hist_mass() const { return reinterpret_cast<u64*>(dyn + lay.hist_mass); }
    __device__ __forceinline__ uint32_t* hist_cnt() const { return reinterpret_cast<uint32_t*>(dyn + lay.hist_cnt); }
    __device__ __forceinline__ u64* own_mass() const { return reinterpret_cast<u64*>(dyn + lay.own_mass); }
    __device__ __forceinline__ uint32_t* own_cnt() const { return reinterpret_cast<uint32_t*>(dyn + lay.own_cnt); }
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
    // f(logits of a 16-byte piece, first position), likewise
    template <typename F>
    __device__ __forceinline__ void each_piece(int b, F f) const {
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const int q = (b * CHUNKS + c) * 32 + lane;
            const uint4 w = data[q];
            const T* x = reinterpret_cast<const T*>(&w);
            float l[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) l[i] = float(x[i]);
            f(l, q * VE);
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
        __syncthreads();
        if (size > 1) cluster_wait();  // the cluster's CTAs run (they arrived as they started): their memory may be written
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

    __device__ __forceinline__ void clear_hist(bool mass) {
        for (int b = tid; b < SMP_BINS; b += SMP_THREADS) {
            hist_cnt()[b] = 0;
            if (mass) hist_mass()[b] = 0;
        }
        __syncthreads();
    }
    // The bins over the cluster: this CTA's share to own_cnt (and own_mass).
    __device__ __forceinline__ void merge_hist(bool with_mass) {
        u64* mass = own_mass();
        uint32_t* cnt = own_cnt();
        for (int b = tid; b < lay.share; b += SMP_THREADS) {
            cnt[b] = 0;
            mass[b] = 0;
        }
        if (size > 1) cl.sync(); else __syncthreads();  // all histograms are complete
        const int n = lay.share * size;  // = SMP_BINS: a thread reads a few bins of other CTAs
#pragma unroll
        for (int i0 = 0; i0 < SMP_BINS; i0 += SMP_THREADS) {
            const int i = i0 + tid, b = i % lay.share, r = i / lay.share;
            if (i < n) {
                const uint32_t c = cl.map_shared_rank(hist_cnt(), r)[rank * lay.share + b];
                if (c) {
                    atomicAdd(&cnt[b], c);
                    if (with_mass) atomicAdd(&mass[b], cl.map_shared_rank(hist_mass(), r)[rank * lay.share + b]);
                }
            }
        }
        __syncthreads();
    }
    // the shares' totals to got(0, r) (mass) and got(1, r) (count) of everyone
    __device__ __forceinline__ void exchange_totals() {
        u64 tm = 0, tc = 0;
        for (int b = tid; b < lay.share; b += SMP_THREADS) {
            tm += own_mass()[b];
            tc += own_cnt()[b];
        }
        cta_sum(tm, tc);
        exchange(tm, tc);
    }

    struct Border {
        int owner, bin;
        u64 mass_above, cnt_above, cnt;  // above the bin, and in it
    };
    // The bin where the running count (by_mass: mass) from the top reaches `target`, straight after exchange_totals;
    // (am, ac): the mass and count above all of its bins.
    __device__ __forceinline__ Border find_border(bool by_mass, u64 target, u64 am, u64 ac) {
        const u64* mass = own_mass();
        const uint32_t* cnt = own_cnt();
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
    // the counts of level 0, and the sum of this CTA's weights
    __device__ __forceinline__ u64 level0_counts_and_sum() {
        clear_hist(false);
        double sum = 0.0;
        for (int b = warp; b < n_blk; b += SMP_WARPS)
            each_piece(b, [&](const float (&l)[VE], int) {
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if (l[i] >= l_floor) atomicAdd(&hist_cnt()[bin0(l[i])], 1u);
                weight.sum_weights(l, l_floor, sum);
            });
        merge_hist(false);
        return u64(sum);
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
        return descend_keys(lo, hi, bd, by_mass, target);
    }
    // likewise from the keys lo..hi; bd: what lies above them
    __device__ __forceinline__ Level descend_keys(uint32_t lo, uint32_t hi, Border bd, bool by_mass, u64 target) {
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
            exchange_totals();
            bd = find_border(by_mass, target, bd.mass_above, bd.cnt_above);
            const uint32_t top = hi - (uint32_t(bd.bin) << shift);
            lo = max(lo, top - ((1u << shift) - 1));
            hi = top;
        }
        return Level{order_value(lo), bd.mass_above, bd.cnt_above};
    }

    // This CTA's candidates: up to SMP_LIST, in hist_mass()[0 .. n_local).
    __device__ __forceinline__ void collect(float l, int pos) {
        hist_mass()[atomicAdd(&sm.n_local, 1u)] = rank_key(l, token_at(pos));
    }
    // They go to the list of CTA `leader`, hist_mass() + SMP_LIST there, where n_list counts them; a barrier of the
    // cluster has to follow.
    __device__ __forceinline__ void send_candidates(int leader) {
        __syncthreads();
        const uint32_t n = sm.n_local;
        if (tid == 0 && n > 0) sm.base = atomicAdd(&cl.map_shared_rank(&sm, leader)->n_list, n);
        __syncthreads();
        u64* dst = cl.map_shared_rank(hist_mass() + SMP_LIST, leader) + sm.base;
        for (uint32_t i = tid; i < n; i += SMP_THREADS) dst[i] = hist_mass()[i];
    }
    // In the leader, after that barrier: sorts the list and returns its length.
    __device__ __forceinline__ int sort_candidates() {
        u64* list = hist_mass() + SMP_LIST;
        const int n = int(sm.n_list), m = sort_size(n);
        for (int i = n + tid; i < m; i += SMP_THREADS) list[i] = ~0ull;
        bitonic_sort(list, m);
        return n;
    }

    // ---- the whole rest on a list: every logit of bins 0..bin (at most SMP_LIST) goes to CTA `leader`, which sorts
    // them, applies the three prefixes and draws.  mass: of all weights (top-p without top-k).
    __device__ __forceinline__ void finish_on_list(int bin, int leader, u64 mass) {
        each_of_slice([&](float l, int pos) {
            if (l >= l_floor && bin0(l) <= bin) collect(l, pos);
        });
        send_candidates(leader);
        if (size > 1) cl.sync(); else __syncthreads();
        if (rank != leader) return;
        const int n = sort_candidates();
        draw_from_list(hist_mass() + SMP_LIST, n, hist_mass(), reinterpret_cast<u64*>(hist_cnt()), mass);
    }

    // ---- top-p alone: where the mass reaches the target, estimated from the counts (every weight of a bin as its
    // middle's, off by at most 0.7 %).  In every CTA: a window [lo, hi] of bins around the estimate, from the share of
    // CTA `owner`, with at most SMP_LIST logits.  all: the logits down to hi fit the list, and reach the target for certain.
    struct Window {
        int owner, lo, hi;
        bool all, none;  // none: the bin of the estimate (lo = hi) alone is too full
    };
    __device__ __forceinline__ Window p_window(u64& mass, u64& target, u64 sum) {
        u64 unused = 0;
        cta_sum(sum, unused);
        // the estimates, in place of the (unused) masses of the bins; all threads of one order: the same every run
        double* est = reinterpret_cast<double*>(own_mass());
        const double step = -2.0 / double(bin_scale) * weight.scale * (1.0 / SMP_TABLE);  // log2 of a weight per bin
        const double unit = exp2(double(p.frac_bits));
        double tm = 0.0;
        u64 tc = 0;
        const int per = max(1, lay.share / SMP_THREADS), b0 = tid * per;
        for (int i = 0; i < per && b0 + i < lay.share; ++i) {
            const int b = rank * lay.share + b0 + i;
            const uint32_t c = own_cnt()[b0 + i];
            const double e = c ? double(c) * unit * double(ex2f(float((double(b) + 0.5) * step))) : 0.0;
            est[b0 + i] = e;
            tm += e;
            tc += c;
        }
        // inclusive scans over the threads
        u64 em = u64(tm), ec = tc;
        const u64 em_own = em;
        cta_scan(em, ec);
        if (tid == SMP_THREADS - 1) {
            sm.r[0] = em;
            sm.r[1] = ec;
        }
        __syncthreads();
        exchange(sm.r[0], sm.r[1], sum);
        mass = 0;
        u64 est_all = 0;
        for (int r = 0; r < size; ++r) {
            mass += got(2, r);
            est_all += got(0, r);
        }
        target = p_target(mass);
        // Measured from the tail, whose many logits' estimates are good, not from the few largest: their error is the
        // difference of the sums.
        const u64 goal = est_all > mass - target ? est_all - (mass - target) : 1;
        int owner = 0;
        u64 am = 0, ac = 0, bm = 0, bc = 0;  // estimate and count above share r; those of the owner
        for (int r = 0, found = 0; r < size; ++r) {
            if (got(1, r) > 0 && !found) {  // never an empty share
                owner = r;
                bm = am;
                bc = ac;
                found = am + got(0, r) >= goal;
            }
            am += got(0, r);
            ac += got(1, r);
        }
        __syncthreads();
        if (tid == 0) {
            sm.lo = sm.all = lay.share;
            sm.hi = -1;
        }
        if (tid == SMP_THREADS - 1) sm.r[3] = ~0ull;  // the bin of the estimate and the count above it
        __syncthreads();
        if (rank == owner) {
            // the thread whose bins cross the target; the last one with a count if the estimate falls short
            const u64 begin = bm + em - em_own;
            const bool crosses = begin < goal && goal <= bm + em;
            if (crosses || (bm + sm.r[0] < goal && ec == sm.r[1] && tc > 0)) {
                double run = double(begin);
                u64 c = bc + ec - tc;
                int at = b0;
                for (int i = 0; i < per && b0 + i < lay.share; ++i) {
                    at = b0 + i;
                    run += est[at];
                    if (run >= double(goal) || (!crosses && c + own_cnt()[at] == bc + ec)) break;
                    if (i + 1 < per && b0 + i + 1 < lay.share) c += own_cnt()[at];
                }
                sm.r[3] = u64(at) << 40 | c;
            }
        }
        __syncthreads();
        if (rank == owner) {
            const int at = int(sm.r[3] >> 40);
            const u64 c_at = sm.r[3] & 0xffffffffffull;           // count above the bin
            const u64 n_at = sm.r[3] == ~0ull ? ~0ull : own_cnt()[at];
            const u64 room = n_at < SMP_LIST ? (SMP_LIST - n_at) / 2 : 0;
            if (n_at <= SMP_LIST) {
                u64 c = bc + ec - tc;
                double run = double(bm + em - em_own);
                for (int i = 0; i < per && b0 + i < lay.share; ++i) {  // (c, c + n]: the logits of this bin
                    const int b = b0 + i;
                    const u64 n = own_cnt()[b];
                    run += est[b];
                    if (b <= at && c_at - c <= room) atomicMin(&sm.lo, b);
                    if (b >= at && c + n - c_at - n_at <= room) {
                        atomicMax(&sm.hi, b);
                        if (c + n <= SMP_LIST && (c + n == ac || run * 0.98 >= double(target))) atomicMin(&sm.all, b);
                    }
                    c += n;
                }
            }
        }
        __syncthreads();
        // sm.all: a bin down to which everything fits the list and reaches the target
        exchange(u64(owner * lay.share + sm.lo), u64(sm.hi < 0 ? 0 : owner * lay.share + sm.hi + 1),
                 u64(sm.all == lay.share ? 0 : owner * lay.share + sm.all + 1),
                 u64(owner * lay.share + min(int(sm.r[3] >> 40), lay.share - 1)));
        const int hi = int(got(1, owner)) - 1, all = int(got(2, owner)) - 1;
        if (hi < 0) return Window{owner, int(got(3, owner)), int(got(3, owner)), false, true};
        return Window{owner, int(got(0, owner)), all >= 0 ? all : hi, all >= 0, false};
    }

    // The exact border of top-p in the window.  Leaves the kept weights by blocks in blk_mass; the key of the last
    // kept logit, or 0 when the window missed the border.
    __device__ __forceinline__ u64 cut_in_window(const Window& win, u64 target) {
        // the logits from `edge` on lie above the window, those from `last` on in it
        const float edge = win.lo == 0 ? INFINITY : lowest_of_bins(win.lo - 1), last = lowest_of_bins(win.hi);
        const float min_edge = fmaxf(edge, l_min);
        double above_d = 0.0;
        for (int b = warp; b < n_blk; b += SMP_WARPS) {
            double bm = 0.0, bw = 0.0;
            each_piece(b, [&](const float (&l)[VE], int pos) {
                weight.sum_weights(l, edge, bw);
                if (min_edge > edge) weight.sum_weights(l, min_edge, bm);
#pragma unroll
                for (int i = 0; i < VE; ++i)
                    if (l[i] < edge && l[i] >= last) collect(l[i], pos + i);
            });
            above_d += bw;
            const u64 kept = warp_sum_u64(u64(min_edge > edge ? bm : bw));
            if (lane == 0) blk_mass()[b] = kept;
        }
        u64 above = u64(above_d), unused = 0;
        cta_sum(above, unused);
        send_candidates(win.owner);
        exchange(above);
        above = 0;
        for (int r = 0; r < size; ++r) above += got(0, r);
        if (rank == win.owner) {
            const int n = sort_candidates();
            const u64* const list = hist_mass() + SMP_LIST;
            u64 w[2];
#pragma unroll
            for (int i = 0; i < 2; ++i) w[i] = 2 * tid + i < n ? weight(key_logit(list[2 * tid + i])) : 0;
            u64 cum = w[0] + w[1];
            cta_scan(cum, unused);
            if (tid == 0) sm.r[0] = 0;
            __syncthreads();
            const u64 end = above + cum, begin = end - w[0] - w[1];
            if (begin < target && target <= end)  // one thread, if the border is here
                sm.r[0] = list[2 * tid + (begin + w[0] >= target ? 0 : 1)];
            __syncthreads();
        }
        exchange(sm.r[0]);
        const u64 cut = got(0, win.owner);
        if (cut) {
            // this CTA's kept candidates join their blocks (its own list may have been sorted into the leader's: it is
            // still here, the leader's copy is the other half)
            for (uint32_t i = tid; i < sm.n_local; i += SMP_THREADS) {
                const u64 key = hist_mass()[i];
                const float l = key_logit(key);
                if (key <= cut && l >= l_min)
                    atomicAdd(&blk_mass()[int((long long)(key & 0xffffffffu) - start + phase) / SMP_BLK], weight(l));
            }
        }
        __syncthreads();
        return cut;
    }

    // The border of top-p by exact sums, in bins lo..hi or in those next to them, 1, 2, 4, .. at a time.  False: it is not
    // there.
    __device__ __forceinline__ bool search_near(int lo, int hi, u64 target, Level& found) {
        float edge = lo == 0 ? INFINITY : lowest_of_bins(lo - 1), last = lowest_of_bins(hi);
        for (int attempt = 0; attempt < 8; ++attempt) {
            double above_d = 0.0, with_d = 0.0;
            // keys: the next value below, the (inverted) next from the edge on; the largest and (inverted) smallest between
            uint32_t q[4] = {0, 0, 0, 0};
            for (int b = warp; b < n_blk; b += SMP_WARPS)
                each_piece(b, [&](const float (&l)[VE], int) {
                    weight.sum_weights(l, edge, above_d);
                    weight.sum_weights(l, last, with_d);
#pragma unroll
                    for (int i = 0; i < VE; ++i) {
                        const uint32_t key = order_key(l[i]);
                        if (l[i] >= edge) {
                            q[1] = max(q[1], ~key);
                        } else if (l[i] >= last) {
                            q[2] = max(q[2], key);
                            q[3] = max(q[3], ~key);
                        } else if (l[i] >= l_floor) {
                            q[0] = max(q[0], key);
                        }
                    }
                });
            u64 above = u64(above_d), with = u64(with_d);
            __syncthreads();
            if (tid < 4) sm.key[tid] = 0;
            cta_sum(above, with);  // its barriers stand between the clearing and the maxima
#pragma unroll
            for (int i = 0; i < 4; ++i) {
                const uint32_t m = __reduce_max_sync(0xffffffffu, q[i]);
                if (lane == 0) atomicMax(&sm.key[i], m);
            }
            __syncthreads();
            exchange(above, with, u64(sm.key[0]) << 32 | sm.key[1], u64(sm.key[2]) << 32 | sm.key[3]);
            above = with = 0;
            for (int i = 0; i < 4; ++i) q[i] = 0;
            for (int r = 0; r < size; ++r) {
                above += got(0, r);
                with += got(1, r);
                q[0] = max(q[0], uint32_t(got(2, r) >> 32));
                q[1] = max(q[1], uint32_t(got(2, r)));
                q[2] = max(q[2], uint32_t(got(3, r) >> 32));
                q[3] = max(q[3], uint32_t(got(3, r)));
            }
            if (above < target && target <= with) {
                found = descend_keys(~q[3], q[2], Border{0, 0, above, 0, 0}, true, target);
                return true;
            }
            if (target <= above) {
                if (!q[1]) return false;
                const int bin = bin0(order_value(~q[1])) - (1 << attempt);
                last = edge;
                edge = bin < 0 ? INFINITY : lowest_of_bins(bin);
            } else {
                if (!q[0]) return false;
                edge = last;
                last = lowest_of_bins(min(n_bins - 1, bin0(order_value(q[0])) + (1 << attempt) - 1));
            }
        }
        return false;
    }

    // ---- the key of the last kept logit by narrowing histograms, for borders that no list holds
    // For top-p alone: the mass of all weights, and the bins where the border is expected.
    __device__ __forceinline__ u64 cut_by_levels(bool top_k_cuts, const Border& k_border, u64 k_target, u64 mass, int hint_lo,
                                                 int hint_hi) {
        Level lv{-INFINITY, 0, 0};
        long long n_tie = 0;  // how many of the logits equal to lv.value are kept
        if (top_k_cuts) {
            lv = descend(k_border, false, k_target);
            n_tie = (long long)(k_target - lv.cnt_above);
        }
        if (top_p < 1.0) {
            if (k) {  // the mass of the top-k
                const float from = n_tie > 0 ? fmaxf(l_floor, order_value(order_key(lv.value) + 1)) : l_floor;
                double sum = 0.0;
                for (int b = warp; b < n_blk; b += SMP_WARPS)
                    each_piece(b, [&](const float (&l)[VE], int) { weight.sum_weights(l, from, sum); });
                u64 s = u64(sum), unused = 0;
                cta_sum(s, unused);
                exchange(s);
                mass = n_tie > 0 ? u64(n_tie) * weight(lv.value) : 0;
                for (int r = 0; r < size; ++r) mass += got(0, r);
            }
            const u64 target = p_target(mass);
            Level lp{0.0f, 0, 0};
            if (hint_lo < 0 || !search_near(hint_lo, hint_hi, target, lp)) {
                level0(true);
                exchange_totals();
                lp = descend(find_border(true, target, 0, 0), true, target);
            }
            const u64 w = weight(lp.value);
            long long need = (long long)((target - lp.mass_above + w - 1) / w);  // the mass above is short of the target
            if (n_tie > 0 && lp.value == lv.value) need = min(need, n_tie);
            lv = lp;
            n_tie = need;
        }
        if (n_tie == 0) return ~0ull;
        // the index of the n_tie-th of the equal logits
        u64 mine = 0, unused = 0;
        __syncthreads();
        for (int b = warp; b < n_blk; b += SMP_WARPS) {
            uint32_t t = 0;
            each(b, [&](float l, int) { t += l == lv.value; });
            t = __reduce_add_sync(0xffffffffu, t);
            if (lane == 0) {
                blk_tie()[b] = t;
                mine += t;
            }
        }
        cta_sum(mine, unused);
        exchange(mine);
        u64 before = 0;
        for (int r = 0; r < rank; ++r) before += got(0, r);
        u64 left = u64(n_tie) > before ? u64(n_tie) - before : 0;  // 1-based within this CTA
        if (tid == 0) sm.r[0] = 0;
        __syncthreads();
        if (warp == 0 && left > 0 && left <= mine) {
            for (int b0 = 0; b0 < n_blk; b0 += 32) {
                const u64 t = b0 + lane < n_blk ? blk_tie()[b0 + lane] : 0;
                const u64 incl = warp_scan_u64(t, lane);
                const unsigned hit = __ballot_sync(0xffffffffu, incl >= left);
                if (!hit) {
                    left -= __shfl_sync(0xffffffffu, incl, 31);
                    continue;
                }
                const int f = __ffs(hit) - 1;
                left -= __shfl_sync(0xffffffffu, incl - t, f);
                const int pos0 = (b0 + f) * SMP_BLK + lane * (SMP_BLK / 32);
                const T* x = reinterpret_cast<const T*>(data) + pos0;
                u64 n = 0;
                for (int i = 0; i < SMP_BLK / 32; ++i) n += float(x[i]) == lv.value;
                const u64 n_incl = warp_scan_u64(n, lane);
                if (n_incl >= left && n_incl - n < left) {
                    u64 seen = n_incl - n;
                    for (int i = 0; i < SMP_BLK / 32; ++i)
                        if (float(x[i]) == lv.value && ++seen == left) sm.r[0] = rank_key(lv.value, token_at(pos0 + i));
                }
                break;
            }
        }
        __syncthreads();
        exchange(sm.r[0]);
        u64 cut = 0;
        for (int r = 0; r < size; ++r) cut = max(cut, got(0, r));
        return cut;
    }

    // the kept weights by blocks
    __device__ __forceinline__ void sum_blocks(u64 cut) {
        const float cut_l = cut_logit(cut);
        __syncthreads();
        for (int b = warp; b < n_blk; b += SMP_WARPS) {
            u64 bm = 0;
            if (cut == ~0ull) {
                double sum = 0.0;
                each_piece(b, [&](const float (&l)[VE], int) { weight.sum_weights(l, l_min, sum); });
                bm = u64(sum);
            } else {
                each(b, [&](float l, int pos) {
                    if (is_kept(l, token_at(pos), cut, cut_l)) bm += weight(l);
                });
            }
            bm = warp_sum_u64(bm);
            if (lane == 0) blk_mass()[b] = bm;
        }
        __syncthreads();
    }

    // ---- the draw over the slices, from the kept weights by blocks: which CTA, which block, which position
    __device__ __forceinline__ void draw(u64 cut) {
        u64 mine = 0, unused = 0;
        for (int b = tid; b < n_blk; b += SMP_THREADS) mine += blk_mass()[b];
        cta_sum(mine, unused);
        exchange(mine);
        u64 total = 0, before = 0;
        for (int r = 0; r < size; ++r) {
            if (r < rank) before += got(0, r);
            total += got(0, r);
        }
        u64 target = draw_target(total);
        if (target < before || target >= before + mine || warp != 0) return;  // the owner's first warp goes on
        target -= before;
        const float cut_l = cut_logit(cut);
        for (int b0 = 0; b0 < n_blk; b0 += 32) {
            const u64 m = b0 + lane < n_blk ? blk_mass()[b0 + lane] : 0;
            const u64 m_incl = warp_scan_u64(m, lane);
            const unsigned hit = __ballot_sync(0xffffffffu, m_incl > target);
            if (!hit) {
                target -= __shfl_sync(0xffffffffu, m_incl, 31);
                continue;
            }
            const int f = __ffs(hit) - 1;
            target -= __shfl_sync(0xffffffffu, m_incl - m, f);
            // inside block b0 + f every lane takes 16 consecutive positions
            const int pos0 = (b0 + f) * SMP_BLK + lane * (SMP_BLK / 32);
            const T* x = reinterpret_cast<const T*>(data) + pos0;
            u64 lm = 0;
#pragma unroll 4
            for (int i = 0; i < SMP_BLK / 32; ++i) {
                const float l = float(x[i]);
                if (is_kept(l, token_at(pos0 + i), cut, cut_l)) lm += weight(l);
            }
            const u64 incl = warp_scan_u64(lm, lane);
            const unsigned lane_hit = __ballot_sync(0xffffffffu, incl > target);
            if (lane == __ffs(lane_hit) - 1) {
                u64 run = incl - lm;
                for (int i = 0; i < SMP_BLK / 32; ++i) {
                    const float l = float(x[i]);
                    if (is_kept(l, token_at(pos0 + i), cut, cut_l)) run += weight(l);
                    if (run > target) {
                        write(token_at(pos0 + i), log_share(l, total));
                        break;
                    }
                }
            }
            break;
        }
    }

    __device__ __forceinline__ void run() {
        make_table();
        if (tid == 0) sm.n_local = sm.n_list = sm.base = 0;
        __syncthreads();
        if (size > 1) cluster_arrive();
        load();
        if (!(mx > -INFINITY)) {  // nothing to draw from
            if (rank == 0 && tid == 0) write(-1, -INFINITY);
            return;
        }
        if (greedy_row()) {
            greedy();
            return;
        }
        prepare(mx);
        const bool want_p = top_p < 1.0;
        if (!k && !want_p) {
            sum_blocks(~0ull);
            draw(~0ull);
            return;
        }
        u64 cut;
        if (k) {  // top-k comes first, and is exact in the counts
            level0(false);
            exchange_totals();
            u64 cnt = 0;
            for (int r = 0; r < size; ++r) cnt += got(1, r);
            const u64 target = min(u64(k), cnt);
            const Border bd = find_border(false, target, 0, 0);
            if (bd.cnt_above + bd.cnt <= SMP_LIST) {
                finish_on_list(bd.bin, bd.owner, 0);
                return;
            }
            cut = cut_by_levels(u64(k) < cnt, bd, target, 0, -1, -1);
        } else {
            const u64 sum = level0_counts_and_sum();
            u64 mass, target;
            const Window win = p_window(mass, target, sum);
            if (win.all) {
                finish_on_list(win.hi, win.owner, mass);
                return;
            }
            cut = win.none ? 0 : cut_in_window(win, target);
            if (cut) {
                draw(cut);
                return;
            }
            cut = cut_by_levels(false, Border{}, 0, mass, win.lo, win.hi);
        }
        sum_blocks(cut);
        draw(cut);
    }
};

// The rows of a call, one per cluster; or (only: their states) those in ROW_BY_CLUSTER, dealt to the clusters of a small
// grid.
template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 2)
sample_kernel(const SampleParams p, const RowState* only, long long B) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ SmpShared sm;
    __shared__ uint32_t todo[SMP_WARPS];
    const cooperative_groups::cluster_group cl = cooperative_groups::this_cluster();
    const int cluster = int(cl.num_blocks());
    if (!only) {
        Sampler<T> s(p, sm, dyn, blockIdx.x / cluster, cluster);
        s.run();
        return;
    }
    pdl_wait();
    const long long n_cluster = gridDim.x / cluster, first = blockIdx.x / cluster;
    for (long long r0 = first; r0 < B; r0 += n_cluster * SMP_THREADS) {
        // bit t of the list: row r0 + t * n_cluster; the same in all CTAs of the cluster
        const long long mine = r0 + threadIdx.x * n_cluster;
        const unsigned bits = __ballot_sync(0xffffffffu, mine < B && only[mine].mode == ROW_BY_CLUSTER);
        __syncthreads();
        if ((threadIdx.x & 31) == 0) todo[threadIdx.x >> 5] = bits;
        __syncthreads();
        for (int t = 0; t < SMP_THREADS; ++t) {
            if (!todo[t >> 5]) t |= 31;
            if (!(todo[t >> 5] >> (t & 31) & 1)) continue;
            Sampler<T> s(p, sm, dyn, r0 + t * n_cluster, cluster);
            s.run();
            if (cluster > 1) cl.sync(); else __syncthreads();  // before the next row takes the shared memory
        }
    }
}

}  // namespace cce
