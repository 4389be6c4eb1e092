// Logits of the head, with the low-rank adapters of many requests beside the shared classifier:
//
//   out[t][v] = cap( e_t . c_v + bias_v + s_a * sum_j B[a][v][j] (A[a][j] . e_t) ),  a = ids[t]
//
// (no adapter term where ids[t] lies outside [0, n); cap(x) = softcap * tanh(x / softcap)).
//
// adapter_shrink_kernel computes h[t][j] = s_a (A[a][j] . e_t), T x rank fp32 values.
// head_logits_kernel is the projection.  Its tiles are 128 classifier rows x up to 256 tokens, with
// the classifier on the M side of the tensor-core product and the tokens on the N side: a decode
// batch of 1..16 tokens then costs an N = 16 product instead of padding 128 rows, the token
// operand of a stage shrinks to 2 KB, and a thread of the epilogue (one TMEM lane) owns one
// vocabulary entry, so that a warp's store covers 32 neighbouring logits of one token and its
// row of B is read once for all tokens of an adapter.
//
//   warp 0      : TMA producer  (128-byte swizzled ring; as many stages as shared memory holds)
//   warp 1      : tcgen05.mma issuer, owns the TMEM allocation (2 accumulators of 128 x 256 fp32)
//   warps 2..9  : epilogue; warp w reads TMEM lanes 32*(w%4)..+31, two warps share a quarter
//
// The adapters' second product stays on the fp32 pipe of the epilogue: every token picks its own
// rows of B, h is kept in fp32, and an infinity in one request's adapter cannot reach another's row
// (a masked tensor-core product would multiply it by zero).
#pragma once
#include "engine.cuh"

namespace cce {

constexpr int HEAD_EPI_WARPS = 8;
constexpr int HEAD_THREADS = 64 + 32 * HEAD_EPI_WARPS;
constexpr int HEAD_MAX_STAGES = 12;
constexpr int HEAD_SMEM = 227 * 1024;          // everything: the ring decides how many bytes are in flight
constexpr int HEAD_RING_BYTES = HEAD_SMEM - 1024 /*align slack*/ - 512 /*barriers*/;
constexpr int ADAPTER_RANK_PAD = 16;           // h rows are padded to this many ranks with zeros

struct HeadParams {
    int T, V;          // tokens, classifier rows
    int n_kblk;        // ceil(K / 64)
    int n_tok;         // tokens per tile: a multiple of 16, at most 256
    int n_ntile;       // token tiles
    int n_vtile;       // classifier tiles of 128 rows
    int n_stage;
    uint32_t idesc;
    int* status;
    const float* bias;  // fp32 [V] or null
    int has_softcap;
    float softcap;
    void* out;          // [T][V]
    int out_dtype;      // CCE_DT_*
    // adapters (lora_b null: none)
    const void* lora_b;  // [n_adapters][V][rank], e's type
    const void* ids;     // [T] int32 / int64
    int ids_i64;
    int n_adapters;
    int rank;
    int b_vec;           // rows of B can be read 16 bytes at a time
    const float* h;      // [T][ldh] fp32, zero padded to ldh = rank rounded up to ADAPTER_RANK_PAD
    int ldh;
};

template <typename T>
__device__ __forceinline__ float to_float(T x) { return float(x); }

// 16 consecutive values of a row of B (ranks k0 .. k0+15 of `rank`; zeros past it) as fp32
template <typename T>
__device__ __forceinline__ void load_b16(const T* row, int k0, int rank, bool vec, float (&b)[ADAPTER_RANK_PAD]) {
    constexpr int VE = 16 / int(sizeof(T));
    if (vec) {  // rank is a multiple of VE
#pragma unroll
        for (int q = 0; q < ADAPTER_RANK_PAD / VE; ++q) {
            uint4 u = make_uint4(0u, 0u, 0u, 0u);
            if (k0 + q * VE < rank) u = __ldg(reinterpret_cast<const uint4*>(row + k0 + q * VE));
            const T* x = reinterpret_cast<const T*>(&u);
#pragma unroll
            for (int i = 0; i < VE; ++i) b[q * VE + i] = to_float(x[i]);
        }
    } else {
#pragma unroll
        for (int i = 0; i < ADAPTER_RANK_PAD; ++i) b[i] = (k0 + i < rank) ? to_float(row[k0 + i]) : 0.0f;
    }
}

__device__ __forceinline__ int adapter_of(const HeadParams& p, int t) {
    const long long a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[t]
                                  : (long long)reinterpret_cast<const int*>(p.ids)[t];
    return (a >= 0 && a < p.n_adapters) ? int(a) : -1;
}

// x[j] += sum_k B[a_j][v][k] h[t0 + j][k] for the 32 tokens of one chunk; lane j holds a_j
template <typename T>
__device__ __forceinline__ void add_adapters(const HeadParams& p, int v, bool v_ok, int t0, int ncol, int my_id,
                                             float (&x)[32]) {
    if (!__any_sync(0xffffffffu, my_id >= 0)) return;
    const T* B = reinterpret_cast<const T*>(p.lora_b);
#pragma unroll 1
    for (int k0 = 0; k0 < p.rank; k0 += ADAPTER_RANK_PAD) {
        int cur = -1;
        float b[ADAPTER_RANK_PAD];
#pragma unroll
        for (int i = 0; i < ADAPTER_RANK_PAD; ++i) b[i] = 0.0f;
#pragma unroll
        for (int j = 0; j < 32; ++j) {
            const int a = __shfl_sync(0xffffffffu, my_id, j);  // warp-uniform; -1 past the last token
            if (a >= 0) {
                if (a != cur) {
                    cur = a;
                    if (v_ok) load_b16(B + ((size_t)a * p.V + v) * p.rank, k0, p.rank, p.b_vec != 0, b);
                }
                const float4* hp = reinterpret_cast<const float4*>(p.h + (size_t)(t0 + j) * p.ldh + k0);
                float s = 0.0f;
#pragma unroll
                for (int q = 0; q < ADAPTER_RANK_PAD / 4; ++q) {
                    const float4 hv = hp[q];
                    s = fmaf(b[4 * q], hv.x, s);
                    s = fmaf(b[4 * q + 1], hv.y, s);
                    s = fmaf(b[4 * q + 2], hv.z, s);
                    s = fmaf(b[4 * q + 3], hv.w, s);
                }
                x[j] += s;
            }
        }
    }
}

template <typename O>
__device__ __forceinline__ O from_float(float x);
template <>
__device__ __forceinline__ float from_float<float>(float x) { return x; }
template <>
__device__ __forceinline__ __nv_bfloat16 from_float<__nv_bfloat16>(float x) { return __float2bfloat16_rn(x); }
template <>
__device__ __forceinline__ __half from_float<__half>(float x) { return __float2half_rn(x); }

template <typename O>
__device__ __forceinline__ void store_column_chunk(const HeadParams& p, int v, int t0, int ncol, const float (&x)[32]) {
    O* dst = reinterpret_cast<O*>(p.out) + (size_t)t0 * p.V + v;
#pragma unroll
    for (int j = 0; j < 32; ++j)
        if (j < ncol) dst[(size_t)j * p.V] = from_float<O>(x[j]);
}

struct HeadSmem {
    uint8_t* stages;
    uint64_t *full, *empty, *tfull, *tempty, *tdown;
    uint32_t* tmem_base;
    volatile int* abort_flag;
};

// BT: element type of the adapters (and of e)
template <typename BT>
__global__ void __launch_bounds__(HEAD_THREADS, 1)
head_logits_kernel(const __grid_constant__ CUtensorMap tmC, const __grid_constant__ CUtensorMap tmE,
                   const HeadParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    const uint32_t stage_bytes = A_BYTES + p.n_tok * BK * 2;
    HeadSmem s;
    s.stages = base;
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + HEAD_RING_BYTES);
    s.full = bars;
    s.empty = bars + HEAD_MAX_STAGES;
    s.tfull = bars + 2 * HEAD_MAX_STAGES;
    s.tempty = s.tfull + 2;
    s.tdown = s.tfull + 4;
    s.tmem_base = reinterpret_cast<uint32_t*>(s.tfull + 5);
    s.abort_flag = reinterpret_cast<int*>(s.tmem_base + 1);

    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int n_items = p.n_vtile * p.n_ntile;
    if (int(blockIdx.x) >= n_items) return;  // uniform over the CTA
    if (threadIdx.x == 0) {
        for (int i = 0; i < p.n_stage; ++i) {
            mbar_init(smem_u32(&s.full[i]), 1);
            mbar_init(smem_u32(&s.empty[i]), 1);
        }
        for (int i = 0; i < 2; ++i) {
            mbar_init(smem_u32(&s.tfull[i]), 1);
            mbar_init(smem_u32(&s.tempty[i]), HEAD_EPI_WARPS);
        }
        mbar_init(smem_u32(s.tdown), 1);
        *s.abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
        tma_prefetch_desc(&tmC);
        tma_prefetch_desc(&tmE);
    }
    if (warp == 1) {
        tmem_alloc(smem_u32(s.tmem_base), TMEM_COLS);
        tmem_relinquish();
    }
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(s.tmem_base);

    if (warp == 0) {
        if (lane == 0) {
            int stage = 0;
            uint32_t phase = 0;
            bool ok = true;
            for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
                const int row_c = (item / p.n_ntile) * BM, row_e = (item % p.n_ntile) * p.n_tok;
                for (int kb = 0; kb < p.n_kblk; ++kb) {
                    if (!mbar_wait(smem_u32(&s.empty[stage]), phase ^ 1u, s.abort_flag, p.status,
                                   ERR_WAIT_SMEM_EMPTY)) {
                        ok = false;
                        break;
                    }
                    const uint32_t bar = smem_u32(&s.full[stage]);
                    const uint32_t sa = smem_u32(s.stages) + stage * stage_bytes;
                    mbar_expect_tx(bar, stage_bytes);
                    tma_load_2d(sa, &tmC, bar, kb * BK, row_c);
                    tma_load_2d(sa + A_BYTES, &tmE, bar, kb * BK, row_e);
                    if (++stage == p.n_stage) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
            }
        }
    } else if (warp == 1) {
        if (lane == 0) {
            int stage = 0, acc = 0;
            uint32_t phase = 0, acc_phase = 0;
            bool ok = true;
            const uint64_t adesc0 = make_smem_desc(smem_u32(s.stages), 16, 1024);
            for (int item = blockIdx.x; ok && item < n_items; item += gridDim.x) {
                if (!mbar_wait(smem_u32(&s.tempty[acc]), acc_phase ^ 1u, s.abort_flag, p.status,
                               ERR_WAIT_TMEM_EMPTY))
                    break;
                tc_fence_after();
                const uint32_t d_tmem = tmem_base + acc * BN;
                for (int kb = 0; kb < p.n_kblk; ++kb) {
                    if (!mbar_wait(smem_u32(&s.full[stage]), phase, s.abort_flag, p.status, ERR_WAIT_SMEM_FULL)) {
                        ok = false;
                        break;
                    }
                    tc_fence_after();
                    // the address field of a descriptor counts 16-byte units
                    const uint64_t ad = adesc0 + ((stage * stage_bytes) >> 4);
                    const uint64_t bd = ad + (A_BYTES >> 4);
#pragma unroll
                    for (int k = 0; k < BK / UMMA_K; ++k)
                        tc_mma_f16(d_tmem, ad + k * (UMMA_K * 2 >> 4), bd + k * (UMMA_K * 2 >> 4), p.idesc,
                                   (kb | k) ? 1u : 0u);
                    tc_commit(smem_u32(&s.empty[stage]));
                    if (++stage == p.n_stage) {
                        stage = 0;
                        phase ^= 1u;
                    }
                }
                if (ok) tc_commit(smem_u32(&s.tfull[acc]));
                if (++acc == 2) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
        }
    } else {
        const int q = warp & 3;              // TMEM lane quarter this warp may read
        const int half = (warp - 2) >> 2;    // the quarter's two warps take alternate chunks of 32 tokens
        int acc = 0;
        uint32_t acc_phase = 0;
        int ok = 1;
        const float inv_softcap = p.has_softcap ? 1.0f / p.softcap : 0.0f;
        for (int item = blockIdx.x; item < n_items; item += gridDim.x) {
            const int v = (item / p.n_ntile) * BM + q * 32 + lane;
            const bool v_ok = v < p.V;
            const int tok0 = (item % p.n_ntile) * p.n_tok;
            const int tok_end = min(p.T, tok0 + p.n_tok);
            const float bias = (p.bias && v_ok) ? __ldg(p.bias + v) : 0.0f;
            // an abandoned wait: the rest of this CTA's tiles is written as NaN
            if (ok) ok = mbar_wait(smem_u32(&s.tfull[acc]), acc_phase, s.abort_flag, p.status, ERR_WAIT_TMEM_FULL);
            ok = __all_sync(0xffffffffu, ok);
            if (ok) tc_fence_after();
            const uint32_t taddr = tmem_base + acc * BN + (uint32_t(q * 32) << 16);
#pragma unroll 1
            for (int t0 = tok0 + half * 32; t0 < tok_end; t0 += 64) {
                const int ncol = min(32, tok_end - t0);
                float x[32];
                if (ok) {
                    uint32_t r[32];
                    tmem_ld32(taddr + (t0 - tok0), r);
                    tmem_ld_wait();
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = __uint_as_float(r[j]) + bias;
                } else {
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = __int_as_float(0x7fc00000);
                }
                if (p.lora_b) {
                    const int my_id = lane < ncol ? adapter_of(p, t0 + lane) : -1;
                    add_adapters<BT>(p, v, v_ok, t0, ncol, my_id, x);
                }
                if (p.has_softcap) {
#pragma unroll
                    for (int j = 0; j < 32; ++j) x[j] = apply_softcap(x[j], p.softcap, inv_softcap);
                }
                if (v_ok) {
                    if (p.out_dtype == 2)
                        store_column_chunk<float>(p, v, t0, ncol, x);
                    else if (p.out_dtype == 1)
                        store_column_chunk<__nv_bfloat16>(p, v, t0, ncol, x);
                    else
                        store_column_chunk<__half>(p, v, t0, ncol, x);
                }
            }
            tc_fence_before();
            __syncwarp();
            if (ok && lane == 0) mbar_arrive(smem_u32(&s.tempty[acc]));
            if (++acc == 2) {
                acc = 0;
                acc_phase ^= 1u;
            }
        }
    }

    // tear-down: wait (bounded) for every MMA this CTA issued, then release TMEM
    tc_fence_before();
    __syncthreads();
    if (warp == 1) {
        if (lane == 0) {
            tc_commit(smem_u32(s.tdown));
            mbar_wait(smem_u32(s.tdown), 0, s.abort_flag, p.status, ERR_WAIT_TEARDOWN);
        }
        __syncwarp();
        tc_fence_after();
        tmem_dealloc(tmem_base, TMEM_COLS);
    }
}

// h[t][j] = scale[a_t] * (A[a_t][j] . e_t), zero where a token has no adapter and for the padding ranks.
// One block per (8 consecutive tokens, 4 ranks): its 8 warps split D, each lane reads 16 bytes of the
// four rows of A and of every token of a run that shares an adapter, and the 32 sums are joined
// in shared memory in warp order (no atomics: the same bits every run).
constexpr int SHRINK_TOK = 8, SHRINK_RANK = 4, SHRINK_WARPS = 8;

struct ShrinkParams {
    const void* e;
    long long lde;
    const void* lora_a;  // [n_adapters][rank][D]
    const float* scale;  // [n_adapters] or null (1)
    const void* ids;
    int ids_i64;
    int n_adapters, rank, T;
    long long D;
    int vec;  // 16-byte loads are possible for every row
    float* h;
    int ldh;
};

// 16 bytes of a row, `left` of whose elements remain (zeros past them); vec: loaded at once
template <typename T>
__device__ __forceinline__ uint4 load_piece(const T* q, long long left, bool vec) {
    if (vec) return __ldg(reinterpret_cast<const uint4*>(q));
    uint4 u;
    T* x = reinterpret_cast<T*>(&u);
#pragma unroll
    for (int i = 0; i < 16 / int(sizeof(T)); ++i) x[i] = i < left ? q[i] : T(0.0f);
    return u;
}

template <typename T>
__global__ void __launch_bounds__(SHRINK_WARPS * 32)
adapter_shrink_kernel(const ShrinkParams p) {
    constexpr int VE = 16 / int(sizeof(T));
    __shared__ float part[SHRINK_WARPS][SHRINK_TOK * SHRINK_RANK];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tok0 = blockIdx.x * SHRINK_TOK, rank0 = blockIdx.y * SHRINK_RANK;
    const int ntok = min(SHRINK_TOK, p.T - tok0);
    int ids[SHRINK_TOK];
#pragma unroll
    for (int i = 0; i < SHRINK_TOK; ++i) {
        long long a = -1;
        if (i < ntok)
            a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[tok0 + i]
                          : (long long)reinterpret_cast<const int*>(p.ids)[tok0 + i];
        ids[i] = (a >= 0 && a < p.n_adapters) ? int(a) : -1;
    }
    float acc[SHRINK_TOK][SHRINK_RANK];
#pragma unroll
    for (int i = 0; i < SHRINK_TOK; ++i)
#pragma unroll
        for (int k = 0; k < SHRINK_RANK; ++k) acc[i][k] = 0.0f;

    const T* E = reinterpret_cast<const T*>(p.e);
    const T* A = reinterpret_cast<const T*>(p.lora_a);
    int done = 0;  // bit i: token i is accounted for
#pragma unroll 1
    for (int lead = 0; lead < ntok; ++lead) {
        if (done >> lead & 1) continue;
        int a = -1, members = 0;
#pragma unroll
        for (int i = 0; i < SHRINK_TOK; ++i)
            if (i == lead) a = ids[i];
#pragma unroll
        for (int i = 0; i < SHRINK_TOK; ++i)
            if (i < ntok && ids[i] == a) members |= 1 << i;
        done |= members;
        if (a < 0) continue;  // uniform over the block
        const T* arow[SHRINK_RANK];
#pragma unroll
        for (int k = 0; k < SHRINK_RANK; ++k)  // ranks past the end repeat the last row; their sums are dropped
            arow[k] = A + ((size_t)a * p.rank + min(rank0 + k, p.rank - 1)) * p.D;
        // the same lane takes the same VE elements whether or not they can be loaded together
        for (long long d = (long long)(warp * 32 + lane) * VE; d < p.D; d += SHRINK_WARPS * 32 * VE) {
            uint4 av[SHRINK_RANK];
#pragma unroll
            for (int k = 0; k < SHRINK_RANK; ++k) av[k] = load_piece(arow[k] + d, p.D - d, p.vec != 0);
#pragma unroll
            for (int i = 0; i < SHRINK_TOK; ++i) {
                if (members >> i & 1) {
                    const uint4 ev = load_piece(E + (size_t)(tok0 + i) * p.lde + d, p.D - d, p.vec != 0);
                    const T* ex = reinterpret_cast<const T*>(&ev);
#pragma unroll
                    for (int k = 0; k < SHRINK_RANK; ++k) {
                        const T* ax = reinterpret_cast<const T*>(&av[k]);
#pragma unroll
                        for (int c = 0; c < VE; ++c) acc[i][k] = fmaf(to_float(ax[c]), to_float(ex[c]), acc[i][k]);
                    }
                }
            }
        }
    }
    // sum over the lanes: a butterfly that halves the live values at every step; lane l ends up
    // with value l = token (l >> 2), rank (l & 3)
    float v[32];
#pragma unroll
    for (int i = 0; i < SHRINK_TOK; ++i)
#pragma unroll
        for (int k = 0; k < SHRINK_RANK; ++k) v[i * SHRINK_RANK + k] = acc[i][k];
#pragma unroll
    for (int o = 16; o >= 1; o >>= 1) {
        const bool up = (lane & o) != 0;
#pragma unroll
        for (int j = 0; j < o; ++j) {
            const float keep = up ? v[j + o] : v[j];
            const float send = up ? v[j] : v[j + o];
            v[j] = keep + __shfl_xor_sync(0xffffffffu, send, o);
        }
    }
    part[warp][lane] = v[0];
    __syncthreads();
    if (warp == 0) {
        const int i = lane / SHRINK_RANK, k = rank0 + lane % SHRINK_RANK;
        float sum = 0.0f;
#pragma unroll
        for (int w = 0; w < SHRINK_WARPS; ++w) sum += part[w][lane];
        int a = -1;
#pragma unroll
        for (int j = 0; j < SHRINK_TOK; ++j)
            if (j == i) a = ids[j];
        if (a >= 0 && p.scale) sum *= p.scale[a];
        if (i < ntok && k < p.ldh) p.h[(size_t)(tok0 + i) * p.ldh + k] = (a >= 0 && k < p.rank) ? sum : 0.0f;
    }
}

}  // namespace cce
