// Sampling of many long rows: the same steps as sample.cuh's, each as a kernel over (row, chunk of the row).
//
// In sample.cuh a row's passes are separated by cluster barriers, and an SM holds two CTAs at most: 512 rows x 152064
// fp32 logits took 640 us with top-p, 256 x 256000 without filters 268 us, mostly waiting.  Here every pass is a
// kernel with full occupancy that streams the logits from HBM (or L2), so that a pass costs what its bytes or its fp64
// weights cost (0.4 cycles per logit and SM), and what a barrier did is the end of a kernel: 366 and 141 us.  Of the 366:
// maximum 47 (6.6 TB/s), counts and sum 149, plan 14, pass 116, draw 40; of the 141: maximum 38, weights 95, draw 8.
// Below some tens of megabytes the launches cost more than the barriers, and rows that two CTAs of an SM can hold are
// faster there (api_serving.cuh has the rule).
//
//   row_max_kernel     the largest logit of every chunk
//   row_prepare_kernel per row (a warp): its maximum and thresholds, and whether there is anything to do (RowMode)
//   row_stats_kernel   counts by bin and, for top-p alone, the exact sum of the weights; without any filter: the
//                      weights by blocks of 512 positions, and the first of the largest logits of greedy rows
//   row_plan_kernel    per row with a filter: which logits are needed in order
//   row_pass_kernel    gathers them, and sums the kept weights by blocks where not everything is gathered
//   row_draw_kernel    per row: the border among the gathered, the draw
//   sample_kernel      the rows that no list holds (ROW_BY_CLUSTER)
// They are launched with leave to overlap the one before.  Every CTA waits for that one before it returns, even when
// it has nothing to do: a kernel that ended early would let its successor start before its predecessor has ended.
#pragma once
#include "sample.cuh"

namespace cce {

constexpr int STR_BLOCKS = 32;                       // blocks of SMP_BLK positions per chunk
constexpr int STR_CHUNK = STR_BLOCKS * SMP_BLK;
// Twice as many as a cluster's: a bin of a long row of 16-bit logits held up to 900 equal or nearly equal ones, so that
// one beside the estimate's did not fit the window's list and the row went to sample_kernel.
constexpr int STR_BINS = 2 * SMP_BINS;

// Workspace of a call; per row where not said otherwise.
struct StreamBuffers {
    RowState* state;
    float* chunk_max;   // [n_chunk]
    u64* chunk_sum;     // [n_chunk]
    u64* blk_mass;      // [n_chunk * STR_BLOCKS]
    uint32_t* hist;     // [STR_BINS]
    u64* list;          // [SMP_LIST]
    int n_chunk;
};

// The logits of a row by position: counted from the 16-byte boundary at or below the row's first logit; positions
// outside the row hold -inf.
template <typename T>
struct RowStream {
    static constexpr int VE = 16 / int(sizeof(T));
    static constexpr int CHUNKS = SMP_BLK / VE / 32;  // 16-byte pieces per lane and block
    const T* base;
    int phase;
    long long V;
    __device__ __forceinline__ RowStream(const SampleParams& p, long long row) {
        const T* src = reinterpret_cast<const T*>(p.logits) + row * p.ld;
        phase = int((reinterpret_cast<uintptr_t>(src) & 15) / sizeof(T));
        base = src - phase;
        V = p.V;
    }
    __device__ __forceinline__ uint4 piece(long long q) const {
        const long long first = q * VE;
        if (first >= phase && first + VE <= phase + V) return __ldg(reinterpret_cast<const uint4*>(base) + q);
        uint4 w;
        T* x = reinterpret_cast<T*>(&w);
#pragma unroll
        for (int i = 0; i < VE; ++i) x[i] = (first + i >= phase && first + i < phase + V) ? base[first + i] : T(-INFINITY);
        return w;
    }
    __device__ __forceinline__ float at(long long pos) const {
        return pos >= phase && pos < phase + V ? float(base[pos]) : -INFINITY;
    }
    __device__ __forceinline__ bool holds(long long block) const { return block * SMP_BLK < phase + V; }
    // f(logits of a 16-byte piece, first position) for the pieces of a block, a warp together
    template <typename F>
    __device__ __forceinline__ void each_piece(long long block, int lane, F f) const {
        uint4 w[CHUNKS];
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) w[c] = piece((block * CHUNKS + c) * 32 + lane);
#pragma unroll
        for (int c = 0; c < CHUNKS; ++c) {
            const T* x = reinterpret_cast<const T*>(&w[c]);
            float l[VE];
#pragma unroll
            for (int i = 0; i < VE; ++i) l[i] = float(x[i]);
            f(l, ((block * CHUNKS + c) * 32 + lane) * VE);
        }
    }
    // f(l, position) for every position of a block, likewise
    template <typename F>
    __device__ __forceinline__ void each(long long block, int lane, F f) const {
        each_piece(block, lane, [&](const float (&l)[VE], long long pos) {
#pragma unroll
            for (int i = 0; i < VE; ++i) f(l[i], pos + i);
        });
    }
};

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS)
row_max_kernel(const SampleParams p, const StreamBuffers b) {
    __shared__ float wf[SMP_WARPS];
    pdl_launch();
    const long long row = blockIdx.x / b.n_chunk;
    const int chunk = blockIdx.x % b.n_chunk, tid = threadIdx.x, warp = tid >> 5, lane = tid & 31;
    const RowStream<T> rs(p, row);
    float m = -INFINITY;
#pragma unroll
    for (int i = warp; i < STR_BLOCKS; i += SMP_WARPS) {
        const long long block = (long long)chunk * STR_BLOCKS + i;
        if (rs.holds(block)) rs.each(block, lane, [&](float l, long long) { m = fmaxf(m, l); });  // drops NaN
    }
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (lane == 0) wf[warp] = m;
    for (int i = chunk * SMP_THREADS + tid; b.hist && i < STR_BINS; i += b.n_chunk * SMP_THREADS)
        b.hist[row * STR_BINS + i] = 0;
    __syncthreads();
    if (tid == 0) {
#pragma unroll
        for (int w = 0; w < SMP_WARPS; ++w) m = fmaxf(m, wf[w]);
        b.chunk_max[row * b.n_chunk + chunk] = m;
    }
}

// A warp per row.
constexpr int PREP_WARPS = 4;
__global__ void __launch_bounds__(32 * PREP_WARPS)
row_prepare_kernel(const SampleParams p, const StreamBuffers b, long long B) {
    __shared__ CtaScratch sc;  // unused by what is called here
    pdl_launch();
    const long long row = (long long)blockIdx.x * PREP_WARPS + (threadIdx.x >> 5);
    pdl_wait();
    if (row >= B) return;
    RowBase r(p, sc, row);
    r.n_bins = STR_BINS;
    float m = -INFINITY;
    for (int i = r.lane; i < b.n_chunk; i += 32) m = fmaxf(m, b.chunk_max[row * b.n_chunk + i]);
#pragma unroll
    for (int o = 16; o > 0; o >>= 1) m = fmaxf(m, __shfl_xor_sync(0xffffffffu, m, o));
    if (r.lane != 0) return;
    RowState st = {};
    st.mode = !(m > -INFINITY) ? ROW_DONE : r.greedy_row() ? ROW_GREEDY : r.k || r.top_p < 1.0 ? ROW_LIST : ROW_SUM;
    st.first = 0xffffffffu;
    st.mx = m;
    if (st.mode == ROW_LIST || st.mode == ROW_SUM) {
        r.prepare(m);
        st.scale = r.weight.scale;
        st.mx = r.mx;
        st.l_floor = r.l_floor;
        st.l_min = r.l_min;
        st.bin_scale = r.bin_scale;
    }
    b.state[row] = st;
}

// ROW_GREEDY: the lowest index of the largest logits of a chunk joins the row's.
template <typename T>
__device__ __forceinline__ void first_of_largest(const RowBase& r, const RowStream<T>& rs, const StreamBuffers& b, int chunk,
                                                 float mx) {
    unsigned best = 0xffffffffu;
    for (int i = r.warp; i < STR_BLOCKS; i += SMP_WARPS) {
        const long long block = (long long)chunk * STR_BLOCKS + i;
        if (rs.holds(block))
            rs.each(block, r.lane, [&](float l, long long pos) {
                if (l == mx) best = min(best, unsigned(pos - rs.phase));
            });
    }
    best = __reduce_min_sync(0xffffffffu, best);
    if (r.lane == 0 && best != 0xffffffffu) atomicMin(&b.state[r.row].first, best);
}

// FILTERS: some row may have top-k or top-p
template <typename T, bool FILTERS>
__global__ void __launch_bounds__(SMP_THREADS, 3)
row_stats_kernel(const SampleParams p, const StreamBuffers b) {
    __shared__ CtaScratch sc;
    __shared__ uint32_t hist[FILTERS ? STR_BINS : 1];
    pdl_launch();
    const long long row = blockIdx.x / b.n_chunk;
    const int chunk = blockIdx.x % b.n_chunk;
    RowBase r(p, sc, row);
    r.n_bins = STR_BINS;
    r.make_table();
    if (FILTERS)
        for (int i = r.tid; i < STR_BINS; i += SMP_THREADS) hist[i] = 0;
    const RowStream<T> rs(p, row);
    pdl_wait();
    const RowState st = b.state[row];
    if (!FILTERS && st.mode == ROW_GREEDY) {  // with filters row_pass_kernel does it
        first_of_largest(r, rs, b, chunk, st.mx);
        return;
    }
    if (st.mode != (FILTERS ? ROW_LIST : ROW_SUM)) return;
    r.prepare(st);
    __syncthreads();
    double sum_d = 0.0;
    const bool want_sum = !r.k;
    for (int i = r.warp; i < STR_BLOCKS; i += SMP_WARPS) {
        const long long block = (long long)chunk * STR_BLOCKS + i;
        if (!rs.holds(block)) {
            if (!FILTERS && r.lane == 0) b.blk_mass[(row * b.n_chunk + chunk) * STR_BLOCKS + i] = 0;
            continue;
        }
        double bm = 0.0;
        rs.each_piece(block, r.lane, [&](const float (&l)[RowStream<T>::VE], long long) {
            if (FILTERS) {
#pragma unroll
                for (int j = 0; j < RowStream<T>::VE; ++j)
                    if (l[j] >= r.l_floor) atomicAdd(&hist[r.bin0(l[j])], 1u);
                if (want_sum) r.weight.sum_weights(l, r.l_floor, sum_d);
            } else {
                r.weight.sum_weights(l, r.l_min, bm);
            }
        });
        if (!FILTERS) {
            const u64 kept = warp_sum_u64(u64(bm));
            if (r.lane == 0) b.blk_mass[(row * b.n_chunk + chunk) * STR_BLOCKS + i] = kept;
        }
    }
    if (!FILTERS) return;
    u64 sum = u64(sum_d), unused = 0;
    r.cta_sum(sum, unused);  // a barrier: the counts are complete
    if (r.tid == 0) b.chunk_sum[row * b.n_chunk + chunk] = sum;
    for (int i = r.tid; i < STR_BINS; i += SMP_THREADS)
        if (hist[i]) atomicAdd(&b.hist[row * STR_BINS + i], hist[i]);
}

// One CTA per row: the border's bin (top-k) or the window around its estimate (top-p alone), as in sample.cuh.
__global__ void __launch_bounds__(SMP_THREADS, 2)
row_plan_kernel(const SampleParams p, const StreamBuffers b) {
    constexpr int PER = STR_BINS / SMP_THREADS;
    __shared__ CtaScratch sc;
    __shared__ int lo, hi, all, at_bin;
    __shared__ u64 at_above;
    pdl_launch();
    const long long row = blockIdx.x;
    RowBase r(p, sc, row);
    r.n_bins = STR_BINS;
    if (r.tid == 0) {
        lo = all = STR_BINS;
        hi = at_bin = -1;
    }
    pdl_wait();
    RowState st = b.state[row];
    if (st.mode == ROW_LIST) {
        r.prepare(st);
        uint32_t cnt[PER];
        double est[PER];
        const double step = -2.0 / double(r.bin_scale) * r.weight.scale * (1.0 / SMP_TABLE);  // log2 of a weight per bin
        const double unit = exp2(double(p.frac_bits));
        double tm = 0.0;
        u64 tc = 0;
#pragma unroll
        for (int i = 0; i < PER; ++i) {
            const int bin = r.tid * PER + i;
            cnt[i] = b.hist[row * STR_BINS + bin];
            est[i] = cnt[i] ? double(cnt[i]) * unit * double(ex2f(float((double(bin) + 0.5) * step))) : 0.0;
            tm += est[i];
            tc += cnt[i];
        }
        u64 mass = 0, unused = 0;
        if (!r.k)
            for (int i = r.tid; i < b.n_chunk; i += SMP_THREADS) mass += b.chunk_sum[row * b.n_chunk + i];
        r.cta_sum(mass, unused);
        u64 em = u64(tm), ec = tc;
        const u64 em_own = em;
        r.cta_scan(em, ec);
        if (r.tid == SMP_THREADS - 1) {
            sc.r[0] = em;
            sc.r[1] = ec;
        }
        __syncthreads();
        const u64 n_all = sc.r[1];
        st.mass = mass;
        st.target = r.k ? min(u64(r.k), n_all) : r.p_target(mass);
        // top-p alone: the estimates are measured from the tail, whose many logits make them good, not from the few largest
        const u64 rest = mass - st.target;
        const u64 goal = r.k ? st.target : sc.r[0] > rest ? sc.r[0] - rest : 1;
        // the thread whose bins hold the border; for an estimate that falls short, the last one with a count
        const u64 c0 = ec - tc, e0 = em - em_own;
        const bool mine = r.k ? c0 < goal && goal <= ec
                              : (e0 < goal && goal <= em) || (sc.r[0] < goal && ec == n_all && tc > 0);
        if (mine) {
            u64 c = c0;
            double run = double(e0);
            int bin = -1;
            u64 above = 0;
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                if (cnt[i] && (bin < 0 || !(r.k ? c >= goal : run >= double(goal)))) {
                    bin = r.tid * PER + i;  // the last bin with a count before the target is reached
                    above = c;
                }
                c += cnt[i];
                run += est[i];
            }
            at_bin = bin;
            at_above = above;
        }
        __syncthreads();
        const u64 n_at = at_bin < 0 ? ~0ull : u64(b.hist[row * STR_BINS + max(at_bin, 0)]);
        if (at_bin < 0 || n_at > SMP_LIST) {
            st.mode = ROW_BY_CLUSTER;
        } else if (r.k) {
            st.mode = at_above + n_at <= SMP_LIST ? ROW_LIST : ROW_BY_CLUSTER;
            hi = at_bin;
        } else {
            const u64 room = (SMP_LIST - n_at) / 2;
            u64 c = c0;
            double run = double(e0);
#pragma unroll
            for (int i = 0; i < PER; ++i) {
                const int bin = r.tid * PER + i;
                run += est[i];
                if (bin <= at_bin && at_above - c <= room) atomicMin(&lo, bin);
                if (bin >= at_bin && c + cnt[i] - at_above - n_at <= room) {
                    atomicMax(&hi, bin);
                    if (c + cnt[i] <= SMP_LIST && (c + cnt[i] == n_all || run * 0.98 >= double(st.target))) atomicMin(&all, bin);
                }
                c += cnt[i];
            }
            __syncthreads();
            st.mode = all < STR_BINS ? ROW_LIST : ROW_WINDOW;
            if (all < STR_BINS) hi = all;  // by every thread alike
        }
        __syncthreads();
        if (st.mode == ROW_LIST || st.mode == ROW_WINDOW) {
            st.last = r.lowest_of_bins(hi);
            // (a window that begins with bin 0 has nothing above it)
            st.edge = st.mode == ROW_LIST || lo == 0 ? INFINITY : r.lowest_of_bins(lo - 1);
        }
    }
    if (r.tid == 0) b.state[row] = st;
}

template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 3)
row_pass_kernel(const SampleParams p, const StreamBuffers b) {
    __shared__ CtaScratch sc;
    __shared__ u64 local[SMP_LIST];
    __shared__ uint32_t n_local, base;
    pdl_launch();
    const long long row = blockIdx.x / b.n_chunk;
    const int chunk = blockIdx.x % b.n_chunk;
    RowBase r(p, sc, row);
    r.n_bins = STR_BINS;
    const RowStream<T> rs(p, row);
    r.make_table();
    if (r.tid == 0) n_local = 0;
    pdl_wait();
    const RowState st = b.state[row];
    if (st.mode == ROW_DONE || st.mode == ROW_BY_CLUSTER) return;
    if (st.mode == ROW_GREEDY) {
        first_of_largest(r, rs, b, chunk, st.mx);
        return;
    }
    r.prepare(st);
    __syncthreads();
    double above_d = 0.0;
    for (int i = r.warp; i < STR_BLOCKS; i += SMP_WARPS) {
        const long long block = (long long)chunk * STR_BLOCKS + i;
        u64 kept = 0;
        if (rs.holds(block)) {
            // The plan counted at most SMP_LIST of them; the bound is for logits that are written while the kernels run.
            auto collect = [&](float l, long long pos) {
                const uint32_t at = atomicAdd(&n_local, 1u);
                if (at < SMP_LIST) local[at] = r.rank_key(l, pos - rs.phase);
            };
            if (st.mode == ROW_LIST) {
                rs.each(block, r.lane, [&](float l, long long pos) {
                    if (l >= st.last) collect(l, pos);
                });
            } else {
                const float edge = st.mode == ROW_WINDOW ? st.edge : r.l_floor;  // ROW_SUM: all is above
                const float last = st.mode == ROW_WINDOW ? st.last : INFINITY;
                const float min_edge = fmaxf(edge, r.l_min);
                double bm = 0.0, bw = 0.0;
                rs.each_piece(block, r.lane, [&](const float (&l)[RowStream<T>::VE], long long pos) {
                    r.weight.sum_weights(l, edge, bw);
                    if (min_edge > edge) r.weight.sum_weights(l, min_edge, bm);
#pragma unroll
                    for (int j = 0; j < RowStream<T>::VE; ++j)
                        if (l[j] < edge && l[j] >= last) collect(l[j], pos + j);
                });
                above_d += bw;
                kept = warp_sum_u64(u64(min_edge > edge ? bm : bw));
            }
        }
        if (r.lane == 0) b.blk_mass[(row * b.n_chunk + chunk) * STR_BLOCKS + i] = kept;
    }
    u64 above = u64(above_d), unused = 0;
    r.cta_sum(above, unused);
    if (r.tid == 0) {
        b.chunk_sum[row * b.n_chunk + chunk] = above;
        base = n_local ? atomicAdd(&b.state[row].n_list, n_local) : 0;
    }
    __syncthreads();
    for (uint32_t i = r.tid; i < n_local && base + i < SMP_LIST; i += SMP_THREADS) b.list[row * SMP_LIST + base + i] = local[i];
}

// One CTA per row.  Dynamic shared memory: three lists of SMP_LIST keys, then the blocks' masses.
template <typename T>
__global__ void __launch_bounds__(SMP_THREADS, 2)
row_draw_kernel(const SampleParams p, const StreamBuffers b) {
    extern __shared__ __align__(16) uint8_t dyn[];
    __shared__ CtaScratch sc;
    pdl_launch();
    u64* const list = reinterpret_cast<u64*>(dyn);
    u64* const blk = list + 3 * SMP_LIST;
    const long long row = blockIdx.x;
    RowBase r(p, sc, row);
    r.n_bins = STR_BINS;
    r.make_table();
    if (r.tid == 0) sc.r[0] = 0;
    pdl_wait();
    const RowState st = b.state[row];
    if (st.mode == ROW_BY_CLUSTER) return;
    if (st.mode == ROW_DONE) {
        if (r.tid == 0) r.write(-1, -INFINITY);
        return;
    }
    if (st.mode == ROW_GREEDY) {
        if (r.tid == 0) r.write((long long)st.first, 0.0f);
        return;
    }
    r.prepare(st);
    __syncthreads();
    const int n_blk = b.n_chunk * STR_BLOCKS;
    u64 cut = ~0ull;
    if (st.mode == ROW_LIST || st.mode == ROW_WINDOW) {
        const int n = int(min(st.n_list, unsigned(SMP_LIST))), size = sort_size(n);
        for (int i = r.tid; i < size; i += SMP_THREADS) list[i] = i < n ? b.list[row * SMP_LIST + i] : ~0ull;
        bitonic_sort(list, size);
        if (st.mode == ROW_LIST) {
            r.draw_from_list(list, n, list + SMP_LIST, list + 2 * SMP_LIST, st.mass);
            return;
        }
        for (int i = r.tid; i < n_blk; i += SMP_THREADS) blk[i] = b.blk_mass[row * n_blk + i];
        u64 above = 0, unused = 0;
        for (int i = r.tid; i < b.n_chunk; i += SMP_THREADS) above += b.chunk_sum[row * b.n_chunk + i];
        r.cta_sum(above, unused);
        u64 w[2];
#pragma unroll
        for (int i = 0; i < 2; ++i) w[i] = 2 * r.tid + i < n ? r.weight(RowBase::key_logit(list[2 * r.tid + i])) : 0;
        u64 cum = w[0] + w[1];
        r.cta_scan(cum, unused);
        const u64 end = above + cum, begin = end - w[0] - w[1];
        if (begin < st.target && st.target <= end)  // one thread, if the border is in the window
            sc.r[0] = list[2 * r.tid + (begin + w[0] >= st.target ? 0 : 1)];
        __syncthreads();
        cut = sc.r[0];
        if (!cut) {  // the estimate was off
            if (r.tid == 0) b.state[row].mode = ROW_BY_CLUSTER;
            return;
        }
        const RowStream<T> rs(p, row);
        for (int i = r.tid; i < n; i += SMP_THREADS) {
            const u64 key = list[i];
            const float l = RowBase::key_logit(key);
            if (key <= cut && l >= r.l_min) atomicAdd(&blk[((key & 0xffffffffu) + rs.phase) / SMP_BLK], r.weight(l));
        }
    } else {
        for (int i = r.tid; i < n_blk; i += SMP_THREADS) blk[i] = b.blk_mass[row * n_blk + i];
    }
    __syncthreads();
    // each thread takes a run of neighbouring blocks
    const int per = (n_blk + SMP_THREADS - 1) / SMP_THREADS, b0 = r.tid * per;
    u64 own = 0, unused = 0;
    for (int i = b0; i < min(n_blk, b0 + per); ++i) own += blk[i];
    u64 incl = own;
    r.cta_scan(incl, unused);
    if (r.tid == SMP_THREADS - 1) sc.r[1] = incl;
    __syncthreads();
    const u64 total = sc.r[1], target = r.draw_target(total);
    if (incl > target && incl - own <= target) {
        u64 run = incl - own;
        int i = b0;
        while (run + blk[i] <= target) run += blk[i++];
        sc.r[2] = u64(i);
        sc.r[3] = target - run;
    }
    __syncthreads();
    if (r.warp != 0) return;
    // inside the block every lane takes 16 consecutive positions
    const RowStream<T> rs(p, row);
    const long long pos0 = (long long)sc.r[2] * SMP_BLK + r.lane * (SMP_BLK / 32);
    const u64 rest = sc.r[3];
    const float cut_l = RowBase::cut_logit(cut);
    float l[SMP_BLK / 32];
    u64 lm = 0;
#pragma unroll
    for (int i = 0; i < SMP_BLK / 32; ++i) l[i] = rs.at(pos0 + i);
#pragma unroll
    for (int i = 0; i < SMP_BLK / 32; ++i)
        if (r.is_kept(l[i], pos0 + i - rs.phase, cut, cut_l)) lm += r.weight(l[i]);
    u64 run = warp_scan_u64(lm, r.lane) - lm;
    if (run <= rest && run + lm > rest) {  // one lane
        bool done = false;
#pragma unroll
        for (int i = 0; i < SMP_BLK / 32; ++i) {
            if (!done && r.is_kept(l[i], pos0 + i - rs.phase, cut, cut_l)) {
                run += r.weight(l[i]);
                if (run > rest) {
                    r.write(pos0 + i - rs.phase, r.log_share(l[i], total));
                    done = true;
                }
            }
        }
    }
}

}  // namespace cce
