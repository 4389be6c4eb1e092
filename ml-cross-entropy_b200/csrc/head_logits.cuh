// Logits of the head, with the low-rank adapters of many requests beside the shared classifier:
//
//   out[t][v] = cap( e_t . c_v + bias_v + s_a * sum_j B[a][v][j] (A[a][j] . e_t) ),  a = ids[t]
//
// (no adapter term where ids[t] lies outside [0, n); cap(x) = softcap * tanh(x / softcap)).
//
// adapter_shrink_kernel computes h[t][j] = s_a (A[a][j] . e_t), T x rank values.
// head_logits_kernel is the projection, on CTA pairs (tcgen05 cta_group::2).  Its tiles are 256 classifier
// rows x up to 256 tokens, with the classifier on the M side of the tensor-core product and the tokens
// on the N side: a decode batch of 1..16 tokens then costs an N = 16 product instead of padding 128
// rows, the token operand shrinks to 1 KB per CTA and 64 reduction elements, and a thread of the epilogue
// (one TMEM lane) owns one vocabulary entry, so that a warp's store covers 32 neighbouring logits of one token.
//
//   warp 0      : TMA producer of both CTAs (128-byte swizzled ring; as many stages as shared memory holds)
//   warp 1      : tcgen05.mma issuer (leader CTA), owner of the TMEM (512 columns: 2 to 8 accumulators per CTA)
//   warps 4..11 : epilogue; warp w reads TMEM lanes 32*(w%4)..+31, two warps share a quarter
//
// The adapters' second product.  The accumulator's columns are looked at in groups of 16.  A group whose tokens
// all use one adapter (or none) takes it on the tensor cores, as further reduction blocks of the same columns: A
// operand = the tile's rows of B, B operand = the group's h, split into 16-bit terms of one sign: two in fp16
// (22 bits, down to 2^-25), three in bf16 (23).  A group of several adapters is added by the epilogue in fp32, every token with its own rows
// of B: a masked tensor-core product would multiply one request's adapter by another's zeros, and an infinity
// there would reach the wrong row.  The same is done for groups whose h does not fit the 16-bit type.
// Unless the adapters are many (api_serving.cuh has the rule) adapter_layout_kernel orders the columns by
// adapter, each adapter's run padded to whole groups, so that no group is mixed.
//
// Measured (bf16, 152064 x 3584, one box; others and other moments differ by 10 % from 256 tokens on): 1 token 170 us
// (6.4 TB/s; cuBLAS 177), 64 tokens 181 (188), 256 tokens 247 (287), 2048 tokens 1560 (1740); with 4 adapters of rank 16
// 174, 202, 325, 1940; fp32 logits 171, 184, 290, 1900.  Up to 128 columns HBM bounds it; then the loads from L2 (256 tokens: 2.1 GB of tiles, 9 TB/s), at 2048 the tensor pipe.
// One lane issues: an MMA of 144 columns then follows the last one after 78 cycles, which is what the tensor pipe takes, a
// TMA load after 120.  Few and large loads for that reason: the token loads have four sizes, the runs of h two.
#pragma once
#include "engine.cuh"
#include "ptx_pair.cuh"

namespace cce {

constexpr int HEAD_EPI_WARPS = 8;
constexpr int HEAD_EPI_FIRST = 4;              // the epilogue's first warp: registers are handed out by groups of 4
constexpr int HEAD_THREADS = 32 * (HEAD_EPI_FIRST + HEAD_EPI_WARPS);
constexpr int HEAD_REGS = 168;                 // per thread at launch: 65536 / 384, in steps of 8
// wide tiles of fp32 logits: of the others, and of the epilogue, whose running sums then do not spill
constexpr int HEAD_REGS_FEW = 72, HEAD_REGS_MANY = 216;
static_assert(HEAD_EPI_FIRST * HEAD_REGS_FEW + HEAD_EPI_WARPS * HEAD_REGS_MANY <= (HEAD_EPI_FIRST + HEAD_EPI_WARPS) * HEAD_REGS,
              "no more registers than the block was launched with");
constexpr int HEAD_SPLIT_ABOVE = 2;            // chunks of 32 columns per warp above which the registers are split
constexpr int HEAD_KSUB = 2;                   // 64-element K sub-blocks per ring stage
constexpr int HEAD_MAX_STAGES = 8;
constexpr int HEAD_SMEM = 227 * 1024;          // everything: the ring decides how many bytes are in flight
constexpr int HEAD_RING_BYTES = HEAD_SMEM - 1024 /*align slack*/ - 1024 /*barriers, runs*/;
constexpr int HEAD_GROUP = 16;                 // tokens that share one decision about their adapters
constexpr int ADAPTER_RANK_PAD = 16;           // fp32 rows of h are padded to this many ranks with zeros
constexpr int GROUP_NONE = -1, GROUP_MIXED = -2;
constexpr int HEAD_MAX_ACC = 8;
constexpr long long HEAD_DRAIN_CYCLES = 20000000;  // 10 ms, many times what a load takes
constexpr int HEAD_FORMS = 5;  // of head_logits_kernel: CHUNKS 0 to 4
// fp32 logits: the tensor core truncates every addition, so a sum over all of D drifts (2.4e-6 of the logits'
// norm at D = 2304).  The accumulator is therefore emptied every HEAD_SEGMENT stages (256 elements) into fp32 registers,
// which add with rounding.  Against twice as long segments, 2304 and 4096 elements: error 2.4e-7 (4.5e-7 and 4.8e-7), time
// 189 us (188) for 8 x 256000 x 2304, 305 (286) for 32 tokens of 8 adapters, whose 144 columns have two accumulators,
// 262 to 274 (257 to 260) for 256 x 128256 x 4096.
// 16-bit logits are rounded far above the drift and take the sum in one piece.
constexpr int HEAD_SEGMENT = 2;

struct HeadParams {
    int T, V;          // tokens, classifier rows
    int n_kblk;        // ceil(K / 64)
    int n_tok;         // columns (tokens) a tile has room for: a multiple of 16, at most 256
    int n_col;         // columns: T, or with col_token an upper bound of *n_col_dev
    int n_vtile;       // classifier tiles of 256 rows
    int e_step;        // the token maps' boxes have e_step, 2 e_step, .. rows; the smallest that holds half a tile is used
    int n_acc;         // accumulators in TMEM: 512 columns in n_acc parts of at least n_tok
    const int* col_token;  // null (column = token), or [n_col]: the token of every column, -1 for padding
    const int* n_col_dev;
    uint32_t idesc;    // without its N field
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
    const float* h;      // [column][ldh] fp32, zero padded to ldh = rank rounded up to ADAPTER_RANK_PAD
    int ldh;
    const int* group;    // [ceil(columns / 16)]: the adapter of a group, GROUP_NONE or GROUP_MIXED
    const int* group_bad;  // likewise; non-zero: h does not fit the 16-bit type, treat as mixed
    const unsigned* h_max;  // null, or [16 ceil(columns / 16)]: the bits of the largest |h| of every column
};

constexpr int HEAD_E_MAPS = 4;
struct HeadMaps {
    CUtensorMap c;               // classifier: 64 x 128 rows
    CUtensorMap e[HEAD_E_MAPS];  // tokens: 64 x (i + 1) e_step rows
    CUtensorMap b;               // adapters' B
    CUtensorMap h8, h32;         // 16-bit h: 64 x 8 and 64 x 32 rows
};

// The column tiles of a launch, from the number of columns that the device knows.
struct HeadTiles {
    int n_col, n_ntile, n_tok;
    __device__ __forceinline__ explicit HeadTiles(const HeadParams& p) {
        n_col = p.n_col_dev ? min(*p.n_col_dev, p.n_col) : p.n_col;
        n_ntile = (n_col + p.n_tok - 1) / p.n_tok;
        n_tok = ((n_col + n_ntile - 1) / n_ntile + HEAD_GROUP - 1) / HEAD_GROUP * HEAD_GROUP;  // even shares
    }
};

// The ring of a launch: as many stages as shared memory holds, of HEAD_KSUB sub-blocks of both operands.
struct HeadRing {
    int e_size;             // which token map: its boxes have e_size e_step rows
    uint32_t sub_e, bytes;  // of a sub-block's token operand (this CTA's half of the tile's columns), and of a stage
    int n_stage;
    static constexpr uint32_t off_e = HEAD_KSUB * A_BYTES;  // of a stage: the token operand
    __device__ __forceinline__ HeadRing(const HeadParams& p, const HeadTiles& tiles) {
        e_size = (tiles.n_tok / 2 + p.e_step - 1) / p.e_step;
        sub_e = e_size * p.e_step * BK * 2;
        bytes = off_e + HEAD_KSUB * sub_e;
        n_stage = min(HEAD_MAX_STAGES, int(HEAD_RING_BYTES / bytes));
    }
    // rows of h that a stage of adapters holds per term
    __device__ __forceinline__ int h_rows() const { return sub_e / (BK * 2); }
};
// Classifier stages of its first tile that a CTA brings into L2 while it waits for the kernels that order the columns (they
// take 15 us, in which HBM could deliver 90 MB: 16 stages are 78 MB)
constexpr int HEAD_L2_AHEAD = 16;

// The terms of h in its 16-bit type, see SplitH
template <typename T>
constexpr int H_TERMS = 2;
template <>
constexpr int H_TERMS<__nv_bfloat16> = 3;

// How h and B meet on the tensor cores: `width` ranks at a time.  The 16-bit rows of h consist of blocks of 64 elements
// (128 bytes, a swizzle row); `width` ranks take one or two of them.
//   two terms    rank <= 32: one block, 32 ranks of each term; above: 64 ranks, a block per term
//   three terms  rank <= 16: one block, 16 ranks of each; above: 32 ranks, a block with the first two and a block with the third
struct HPack {
    int width, blocks;
    int pitch, ranks;  // elements of a row of h, and the ranks it has room for
    __host__ __device__ HPack(int rank, int terms) {
        width = terms == 3 ? (rank <= 16 ? 16 : 32) : (rank <= 32 ? 32 : 64);
        blocks = rank <= (terms == 3 ? 16 : 32) ? 1 : 2;
        const int n = (rank + width - 1) / width;
        pitch = n * blocks * BK;
        ranks = n * width;
    }
    // where term t of rank k stands in the row
    __host__ __device__ int at(int k, int t) const { return k / width * blocks * BK + t * width + k % width; }
};

template <typename T>
__device__ __forceinline__ float to_float(T x) { return float(x); }

// fp16 ends at 2^-24, and so does what two terms keep of h: half a step, 2^-25, is lost of every value.  Columns whose
// largest |h| lies below this (but is not 0) would lose more than 2^-17 of it; their groups take the fp32 path.
constexpr float HEAD_H_MIN_FP16 = 0.00390625f;  // 2^-8

__device__ __forceinline__ int group_adapter(const HeadParams& p, int g) {
    const int a = p.group[g];
    if (a < 0) return a;
    bool bad = p.group_bad[g] != 0;
    if (p.h_max) {
        const uint4* m = reinterpret_cast<const uint4*>(p.h_max + (size_t)g * HEAD_GROUP);
#pragma unroll
        for (int i = 0; i < HEAD_GROUP / 4; ++i) {
            const uint4 w = m[i];
            for (const unsigned x : {w.x, w.y, w.z, w.w}) bad |= x != 0 && x < __float_as_uint(HEAD_H_MIN_FP16);
        }
    }
    return bad ? GROUP_MIXED : a;
}

// A run of neighbouring groups of a column tile that share an adapter.
struct Run {
    int adapter;
    short first, cols;  // within the tile
};
constexpr int HEAD_MAX_RUNS = BN / HEAD_GROUP;

// The runs of the tile that starts at column col0, found by a whole warp (one group per lane) and left in shared
// memory; returns their number.  The producers of both CTAs and the MMA issuer find the same.
__device__ __forceinline__ int find_runs(const HeadParams& p, const HeadTiles& tiles, int col0, Run* runs) {
    const int lane = threadIdx.x & 31;
    const int g0 = col0 / HEAD_GROUP;
    const int n = (min(tiles.n_col, col0 + tiles.n_tok) + HEAD_GROUP - 1) / HEAD_GROUP - g0;  // at most 16
    const int a = lane < n ? group_adapter(p, g0 + lane) : GROUP_NONE;
    const int before = __shfl_up_sync(0xffffffffu, a, 1);
    const bool change = lane == 0 || before != a || lane == n;
    const unsigned changes = __ballot_sync(0xffffffffu, change);
    const bool start = change && a >= 0;
    const unsigned starts = __ballot_sync(0xffffffffu, start);
    __syncwarp();
    if (start) {
        const int end = __ffs(changes & ~((2u << lane) - 1)) - 1;  // there is one: lane n
        runs[__popc(starts & ((1u << lane) - 1))] = Run{a, short(lane * HEAD_GROUP), short((end - lane) * HEAD_GROUP)};
    }
    __syncwarp();
    return __popc(starts);
}

// How the adapters' second product uses the ring: an entry is one run x up to h.width ranks; its rows of B take
// 128 x (32, 64 or 128) bytes, in the swizzle of that width, so that 8, 4 or 2 entries share a stage.
struct AdapterPack {
    HPack h;
    int width;  // ranks per entry as B's boxes have them: 16 where that is all
    int a_bytes, max_entries;
    uint32_t layout, sbo;  // of the descriptor: swizzle type, distance of 8-row groups
    __host__ __device__ AdapterPack(int rank, int terms) : h(rank, terms) {
        width = rank <= 16 ? 16 : h.width;
        a_bytes = BM * width * 2;
        max_entries = HEAD_KSUB * A_BYTES / a_bytes;
        layout = width == 16 ? 6 : width == 32 ? 4 : 2;
        sbo = 8 * width * 2;
    }
    // open() begins a stage, entry(i, row, run, r0) is its i-th entry with its columns' rows of h from `row` on (of this
    // CTA's half), close() ends it; open returns false to stop.
    template <typename Open, typename Entry, typename Close>
    __device__ __forceinline__ bool walk(const Run* runs, int n_runs, int rank, int rows, Open open, Entry entry,
                                         Close close) const {
        int i = 0, row = 0;
        for (int k = 0; k < n_runs; ++k) {
            const Run run = runs[k];
            const int half = run.cols / 2;
            for (int r0 = 0; r0 < rank; r0 += h.width) {
                if (i > 0 && (i == max_entries || row + half > rows)) {
                    close();
                    i = row = 0;
                }
                if (i == 0 && !open()) return false;
                entry(i, row, run, r0);
                ++i;
                row += half;
            }
        }
        if (i > 0) close();
        return true;
    }
};

// 16 consecutive values of a row of B (ranks k0 .. k0+15 of `rank`; zeros past it), as they are stored
template <typename T, bool VEC>
struct BRow {
    T x[ADAPTER_RANK_PAD];
    __device__ __forceinline__ void load(const T* row, int k0, int rank) {
        constexpr int VE = 16 / int(sizeof(T));
        if constexpr (VEC) {  // rank is a multiple of VE
#pragma unroll
            for (int q = 0; q < ADAPTER_RANK_PAD / VE; ++q) {
                uint4 u = make_uint4(0u, 0u, 0u, 0u);
                if (k0 + q * VE < rank) u = __ldg(reinterpret_cast<const uint4*>(row + k0 + q * VE));
                *reinterpret_cast<uint4*>(x + q * VE) = u;
            }
        } else {
#pragma unroll
            for (int i = 0; i < ADAPTER_RANK_PAD; ++i) x[i] = (k0 + i < rank) ? row[k0 + i] : T(0.0f);
        }
    }
};

__device__ __forceinline__ int adapter_of(const HeadParams& p, int t) {
    const long long a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[t]
                                  : (long long)reinterpret_cast<const int*>(p.ids)[t];
    return (a >= 0 && a < p.n_adapters) ? int(a) : -1;
}

// x[j] += sum_k B[a_j][v][k] h[col0 + j][k] for the 16 columns j of a mixed group; a_j comes from lane lane0 + j of my_id
// (-1: none).  No branch depends on the token, so that the loads of several tokens are in flight.  Not inlined:
// one copy serves every form of the kernel, and x (local memory) is touched by mixed groups only.
template <typename T, bool VEC>
__device__ __noinline__ void add_adapters(const HeadParams& p, int v, int col0, int n_col, int my_id, int lane0,
                                          float* x) {
    const T* B = reinterpret_cast<const T*>(p.lora_b);
    constexpr int U = 8;  // tokens at a time; their sums wait in registers, so that no store stands between the loads
    for (int j0 = 0; j0 < HEAD_GROUP; j0 += U) {
        int a[U];
        float s[U];
#pragma unroll
        for (int j = 0; j < U; ++j) {
            a[j] = __shfl_sync(0xffffffffu, my_id, lane0 + j0 + j);
            s[j] = 0.0f;
        }
        for (int k0 = 0; k0 < p.rank; k0 += ADAPTER_RANK_PAD) {
#pragma unroll
            for (int j = 0; j < U; ++j) {
                BRow<T, VEC> b;
                b.load(B + ((size_t)max(a[j], 0) * p.V + v) * p.rank, k0, p.rank);
                const float4* hp =
                    reinterpret_cast<const float4*>(p.h + (size_t)min(col0 + j0 + j, n_col - 1) * p.ldh + k0);
#pragma unroll
                for (int q = 0; q < ADAPTER_RANK_PAD / 4; ++q) {
                    const float4 hv = hp[q];
                    s[j] = fmaf(to_float(b.x[4 * q]), hv.x, s[j]);
                    s[j] = fmaf(to_float(b.x[4 * q + 1]), hv.y, s[j]);
                    s[j] = fmaf(to_float(b.x[4 * q + 2]), hv.z, s[j]);
                    s[j] = fmaf(to_float(b.x[4 * q + 3]), hv.w, s[j]);
                }
            }
        }
#pragma unroll
        for (int j = 0; j < U; ++j)
            if (a[j] >= 0) x[j0 + j] += s[j];
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

// A predicated store.  (Written as `if`, the 32 stores of a chunk become 32 branches: 180 cycles a store.)
__device__ __forceinline__ void store_if(float* q, float x, bool yes) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p st.global.f32 [%0], %1;\n\t}" ::"l"(q), "f"(x), "r"(int(yes))
                 : "memory");
}
__device__ __forceinline__ void store_if16(void* q, unsigned short x, bool yes) {
    asm volatile("{\n\t.reg .pred p;\n\tsetp.ne.s32 p, %2, 0;\n\t@p st.global.u16 [%0], %1;\n\t}" ::"l"(q), "h"(x), "r"(int(yes))
                 : "memory");
}
__device__ __forceinline__ void store_if(__nv_bfloat16* q, __nv_bfloat16 x, bool yes) {
    store_if16(q, __bfloat16_as_ushort(x), yes);
}
__device__ __forceinline__ void store_if(__half* q, __half x, bool yes) { store_if16(q, __half_as_ushort(x), yes); }

template <typename O>
__device__ __forceinline__ void store_chunk(const HeadParams& p, int v, int my_token, const float (&x)[32]) {
    O* dst = reinterpret_cast<O*>(p.out) + v;
    const bool v_ok = v < p.V;
    constexpr int U = 16;  // the shuffles of U columns before their stores, which keep their order
#pragma unroll
    for (int j0 = 0; j0 < 32; j0 += U) {
        int t[U];
#pragma unroll
        for (int j = 0; j < U; ++j) t[j] = __shfl_sync(0xffffffffu, my_token, j0 + j);
#pragma unroll
        for (int j = 0; j < U; ++j)
            store_if(dst + (long long)t[j] * p.V, from_float<O>(x[j0 + j]), t[j] >= 0 && v_ok);
    }
}

// bias, mixed groups (bits 0 and 1 of `mixed`: the chunk's two), soft-cap and store of one chunk of 32 columns; v is
// this lane's classifier row
template <typename BT, bool FP32_OUT>
__device__ __forceinline__ void finish_chunk(const HeadParams& p, const HeadTiles& tiles, int v, float bias, int c0,
                                             int col_end, unsigned mixed, float (&x)[32]) {
    const int lane = threadIdx.x & 31;
    const int ncol = min(32, col_end - c0);
    const int my_token = lane < ncol ? (p.col_token ? p.col_token[c0 + lane] : c0 + lane) : -1;
#pragma unroll
    for (int j = 0; j < 32; ++j) x[j] += bias;
    {
        const bool m0 = mixed & 1, m1 = mixed & 2;
        if (m0 || m1) {  // uniform over the warp
            const int my_id = my_token >= 0 ? adapter_of(p, my_token) : -1;
            const int row = min(v, p.V - 1);
            float y[32];
#pragma unroll
            for (int j = 0; j < 32; ++j) y[j] = x[j];
            for (int g = 0; g < 2; ++g) {
                if (!(g ? m1 : m0)) continue;
                const int j0 = g * HEAD_GROUP;
                if (p.b_vec)
                    add_adapters<BT, true>(p, row, c0 + j0, tiles.n_col, my_id, j0, y + j0);
                else
                    add_adapters<BT, false>(p, row, c0 + j0, tiles.n_col, my_id, j0, y + j0);
            }
#pragma unroll
            for (int j = 0; j < 32; ++j) x[j] = y[j];
        }
    }
    if (p.has_softcap) {
        const float inv = 1.0f / p.softcap;
        // fp32 logits: the special-function tanh (1e-7 of the cap) would be their largest error
#pragma unroll
        for (int j = 0; j < 32; ++j)
            x[j] = FP32_OUT ? p.softcap * tanhf(x[j] * inv) : apply_softcap(x[j], p.softcap, inv);
    }
    if (FP32_OUT)
        store_chunk<float>(p, v, my_token, x);
    else if (p.out_dtype == 1)
        store_chunk<__nv_bfloat16>(p, v, my_token, x);
    else
        store_chunk<__half>(p, v, my_token, x);
}

struct HeadSmem {
    uint8_t* stages;
    uint64_t *full, *empty, *tfull, *tempty, *tdown;
    uint32_t* tmem_base;
    volatile int* abort_flag;
    int* ring_end;  // where the producer's use of the ring ended: stage, phase, number of stages
    Run* runs;  // [2][HEAD_MAX_RUNS]: producer, MMA issuer
};

// BT: element type of the adapters (and of e).  CHUNKS > 0: fp32 logits; the accumulator is emptied every HEAD_SEGMENT
// stages into the epilogue's registers, CHUNKS chunks of 32 columns per warp (tiles of up to 64 CHUNKS columns).  0: 16-bit
// logits, the sum in one piece.
template <typename BT, int CHUNKS>
__global__ void __cluster_dims__(2, 1, 1) __launch_bounds__(HEAD_THREADS, 1)
head_logits_kernel(const __grid_constant__ HeadMaps maps, const __grid_constant__ HeadParams p) {
    extern __shared__ uint8_t smem_raw[];
    uint8_t* base = reinterpret_cast<uint8_t*>((reinterpret_cast<uintptr_t>(smem_raw) + 1023) & ~uintptr_t(1023));
    HeadSmem s;
    s.stages = base;
    uint64_t* bars = reinterpret_cast<uint64_t*>(base + HEAD_RING_BYTES);
    s.full = bars;                          // leader: both CTAs' bytes -> MMA
    s.empty = bars + HEAD_MAX_STAGES;       // per CTA: MMA -> producer
    s.tfull = bars + 2 * HEAD_MAX_STAGES;   // per CTA: MMA -> epilogue
    s.tempty = s.tfull + HEAD_MAX_ACC;      // leader: both CTAs' epilogues -> MMA
    s.tdown = s.tempty + HEAD_MAX_ACC;
    s.tmem_base = reinterpret_cast<uint32_t*>(s.tdown + 1);
    s.abort_flag = reinterpret_cast<int*>(s.tmem_base + 1);
    s.ring_end = reinterpret_cast<int*>(s.tmem_base + 2);
    s.runs = reinterpret_cast<Run*>(base + HEAD_RING_BYTES + 512);

    constexpr bool SEGMENTED = CHUNKS > 0;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int rank = int(cluster_ctarank());
    const uint32_t acc_cols = TMEM_COLS / p.n_acc;
    const int n_pairs = int(gridDim.x >> 1), pair = int(blockIdx.x >> 1);
    const int n_kstage = (p.n_kblk + HEAD_KSUB - 1) / HEAD_KSUB;
    if (threadIdx.x == 0) {
        for (int i = 0; i < HEAD_MAX_STAGES; ++i) {
            mbar_init(smem_u32(&s.full[i]), 1);
            mbar_init(smem_u32(&s.empty[i]), 1);
        }
        for (int i = 0; i < p.n_acc; ++i) {
            mbar_init(smem_u32(&s.tfull[i]), 1);
            mbar_init(smem_u32(&s.tempty[i]), 2 * HEAD_EPI_WARPS);
        }
        mbar_init(smem_u32(s.tdown), 1);
        *s.abort_flag = 0;
        fence_barrier_init();
        fence_proxy_async();
        tma_prefetch_desc(&maps.c);
    }
    if (warp == 1) {
        tmem_alloc_pair(smem_u32(s.tmem_base), TMEM_COLS);
        tmem_relinquish_pair();
    }
    tc_fence_before();
    __syncthreads();
    cluster_arrive();  // both CTAs' barriers exist before either one signals the other
    cluster_wait();
    tc_fence_after();
    const uint32_t tmem_base = *reinterpret_cast<volatile uint32_t*>(s.tmem_base);

    constexpr int TERMS = H_TERMS<BT>;
    const AdapterPack pack(p.rank, TERMS);
    const bool ordered = p.col_token != nullptr;  // the columns come from the kernels before this one
    if (warp < HEAD_EPI_FIRST) {
        if constexpr (CHUNKS > HEAD_SPLIT_ABOVE) set_max_regs_down<HEAD_REGS_FEW>();
        if (warp == 0) {
            if (ordered) {
                const int row = pair * 2 * BM + rank * BM;  // of the first tile, if there is one column tile
                if (p.n_col <= p.n_tok && row < p.V && elect_one())
                    for (int kb = 0; kb < min(HEAD_L2_AHEAD * HEAD_KSUB, p.n_kblk); ++kb) tma_prefetch_2d(&maps.c, kb * BK, row);
                pdl_wait();
            }
            const HeadTiles tiles(p);
            const HeadRing ring(p, tiles);
            const int n_items = p.n_vtile * tiles.n_ntile;
            const CUtensorMap* map_e = &maps.e[ring.e_size - 1];
            int stage = 0;
            uint32_t phase = 0;
            auto free_stage = [&]() -> bool {
                return mbar_wait(smem_u32(&s.empty[stage]), phase ^ 1u, s.abort_flag, p.status, ERR_WAIT_SMEM_EMPTY);
            };
            auto next_stage = [&]() {
                if (++stage == ring.n_stage) {
                    stage = 0;
                    phase ^= 1u;
                }
            };
            auto announce = [&](uint32_t bytes) {  // the bytes of both CTAs
                if (rank == 0) mbar_expect_tx(smem_u32(&s.full[stage]), 2 * bytes);
            };
            bool ok = true, waited = ordered;  // waited: for the kernel that makes h
            int n_runs = 0;
            for (int item = pair; item < n_items; item += n_pairs) {
                const int row_c = (item / tiles.n_ntile) * 2 * BM + rank * BM;
                const int col0 = (item % tiles.n_ntile) * tiles.n_tok;
                const int row_e = col0 + rank * (tiles.n_tok / 2);
                // (with one column tile they are the same in every item)
                if (p.lora_b && waited && (item == pair || tiles.n_ntile > 1)) n_runs = find_runs(p, tiles, col0, s.runs);
                if (elect_one()) {  // one lane runs the loop over the stages
                    for (int ks = 0; ok && ks < n_kstage; ++ks) {
                        ok = free_stage();
                        if (!ok) break;
                        const int n = min(HEAD_KSUB, p.n_kblk - ks * HEAD_KSUB);
                        announce(n * (A_BYTES + ring.sub_e));
                        const uint32_t bar = map_to_cta(smem_u32(&s.full[stage]), 0);
                        const uint32_t sa = smem_u32(s.stages) + stage * ring.bytes, sb = sa + ring.off_e;
                        for (int j = 0; j < n; ++j) {
                            const int x = (ks * HEAD_KSUB + j) * BK;
                            tma_load_2d_pair(sa + j * A_BYTES, &maps.c, bar, x, row_c);
                            tma_load_2d_pair(sb + j * ring.sub_e, map_e, bar, x, row_e);
                        }
                        next_stage();
                    }
                }
                if (!p.lora_b) continue;  // an abandoned wait ends every later one at once
                __syncwarp();
                if (!waited) {
                    pdl_wait();
                    waited = true;
                    n_runs = find_runs(p, tiles, col0, s.runs);
                }
                if (elect_one()) {
                    uint32_t bytes = 0;  // announced when the stage is complete: the loads may land before that
                    ok = ok && pack.walk(
                        s.runs, n_runs, p.rank, ring.h_rows(),
                        [&]() -> bool {
                            bytes = 0;
                            return free_stage();
                        },
                        [&](int i, int row, const Run& run, int r0) {
                            const uint32_t bar = map_to_cta(smem_u32(&s.full[stage]), 0);
                            const uint32_t sa = smem_u32(s.stages) + stage * ring.bytes, sb = sa + ring.off_e;
                            const int half = run.cols / 2;  // rows of h that this CTA supplies: a multiple of 8
                            const int blocks = pack.h.blocks;
                            tma_load_3d_pair(sa + i * pack.a_bytes, &maps.b, bar, r0, row_c, run.adapter);
                            for (int t = 0; t < blocks; ++t)
                                for (int y = 0; y < half;) {  // few and large loads: each costs its issue
                                    const bool large = half - y >= 32;
                                    tma_load_2d_pair(sb + t * ring.sub_e + (row + y) * BK * 2, large ? &maps.h32 : &maps.h8, bar,
                                                     pack.h.at(r0, 0) + t * BK, col0 + run.first + rank * half + y);
                                    y += large ? 32 : 8;
                                }
                            bytes += pack.a_bytes + blocks * half * BK * 2;
                        },
                        [&]() {
                            announce(bytes);
                            next_stage();
                        });
                }
            }
            if (elect_one()) {
                s.ring_end[0] = stage;
                s.ring_end[1] = int(phase);
                s.ring_end[2] = ring.n_stage;
            }
        } else if (warp == 1) {
            if (rank == 0) {
                if (ordered) pdl_wait();
                const HeadTiles tiles(p);
                const HeadRing ring(p, tiles);
                const int n_items = p.n_vtile * tiles.n_ntile;
                const uint32_t idesc = p.idesc | (uint32_t(tiles.n_tok >> 3) << 17);
                int stage = 0, acc = 0;
                uint32_t phase = 0, acc_phase = 0;
                const uint64_t adesc0 = make_smem_desc(smem_u32(s.stages), 16, 1024);
                const uint32_t empty0 = smem_u32(s.empty), empty1 = map_to_cta(empty0, 1);
                const uint32_t tfull0 = smem_u32(s.tfull), tfull1 = map_to_cta(tfull0, 1);
                auto filled_stage = [&]() -> bool {
                    if (!mbar_wait(smem_u32(&s.full[stage]), phase, s.abort_flag, p.status, ERR_WAIT_SMEM_FULL)) return false;
                    tc_fence_after();
                    return true;
                };
                auto release_stage = [&]() {  // in both CTAs, once the MMAs issued so far have read it
                    tc_commit_pair(empty0 + 8 * stage);
                    tc_commit_pair(empty1 + 8 * stage);
                    if (++stage == ring.n_stage) {
                        stage = 0;
                        phase ^= 1u;
                    }
                };
                auto publish = [&]() {  // the accumulator, to both CTAs' epilogues
                    tc_commit_pair(tfull0 + 8 * acc);
                    tc_commit_pair(tfull1 + 8 * acc);
                    if (++acc == p.n_acc) {
                        acc = 0;
                        acc_phase ^= 1u;
                    }
                };
                constexpr int STEP = UMMA_K * 2 >> 4;  // descriptor units (16 bytes) per MMA step
                Run* runs = s.runs + HEAD_MAX_RUNS;
                bool ok = true, waited = ordered;
                int n_runs = 0;
                for (int item = pair; item < n_items; item += n_pairs) {
                    const int col0 = (item % tiles.n_ntile) * tiles.n_tok;
                    // (with one column tile they are the same in every item)
                    if (p.lora_b && waited && (item == pair || tiles.n_ntile > 1)) n_runs = find_runs(p, tiles, col0, runs);
                    uint32_t d_tmem = 0;
                    if (elect_one()) {  // one lane issues
                        for (int ks = 0; ok && ks < n_kstage; ++ks) {
                            const bool opens = SEGMENTED ? ks % HEAD_SEGMENT == 0 : ks == 0;
                            if (opens) {
                                if (SEGMENTED && ks > 0) publish();
                                ok = mbar_wait(smem_u32(&s.tempty[acc]), acc_phase ^ 1u, s.abort_flag, p.status,
                                               ERR_WAIT_TMEM_EMPTY);
                                if (!ok) break;
                                tc_fence_after();
                                d_tmem = tmem_base + acc * acc_cols;
                            }
                            ok = filled_stage();
                            if (!ok) break;
                            // the address field of a descriptor counts 16-byte units
                            const uint64_t ad = adesc0 + ((stage * ring.bytes) >> 4), bd = ad + (ring.off_e >> 4);
                            const int n = min(HEAD_KSUB, p.n_kblk - ks * HEAD_KSUB);
                            for (int j = 0; j < n; ++j)
    #pragma unroll
                                for (int k = 0; k < BK / UMMA_K; ++k)
                                    tc_mma_f16_pair(d_tmem, ad + j * (A_BYTES >> 4) + k * STEP,
                                                    bd + j * (ring.sub_e >> 4) + k * STEP, idesc, (!opens || j || k) ? 1u : 0u);
                            release_stage();
                        }
                    }
                    __syncwarp();
                    if (p.lora_b && !waited) {
                        pdl_wait();
                        waited = true;
                        n_runs = find_runs(p, tiles, col0, runs);
                    }
                    if (elect_one() && ok) {
                        ok = pack.walk(
                            runs, n_runs, p.rank, ring.h_rows(), filled_stage,
                            [&](int i, int row, const Run& run, int r0) {
                                const uint32_t run_idesc = p.idesc | (uint32_t(run.cols >> 3) << 17);
                                // from the first term to the second and the third (two blocks are sub_e apart)
                                const uint32_t half_row = pack.h.width / UMMA_K * STEP, block = ring.sub_e >> 4;
                                const uint32_t term2 = TERMS == 2 && pack.h.blocks == 2 ? block : half_row;
                                const uint32_t term3 = pack.h.blocks == 2 ? block : 2 * half_row;
                                const uint32_t sa = smem_u32(s.stages) + stage * ring.bytes;
                                const uint64_t rad = (make_smem_desc(sa + i * pack.a_bytes, 16, pack.sbo) & ~(uint64_t(7) << 61)) |
                                                     uint64_t(pack.layout) << 61;
                                const uint64_t rbd = make_smem_desc(sa + ring.off_e + row * BK * 2, 16, 1024);
                                const int steps = (min(pack.h.width, p.rank - r0) + UMMA_K - 1) / UMMA_K;
                                for (int k = 0; k < steps; ++k) {
                                    tc_mma_f16_pair(d_tmem + run.first, rad + k * STEP, rbd + k * STEP, run_idesc, 1u);
                                    tc_mma_f16_pair(d_tmem + run.first, rad + k * STEP, rbd + term2 + k * STEP, run_idesc, 1u);
                                    if constexpr (TERMS == 3)
                                        tc_mma_f16_pair(d_tmem + run.first, rad + k * STEP, rbd + term3 + k * STEP, run_idesc, 1u);
                                }
                            },
                            release_stage);
                        if (ok) publish();
                    }
                    if (!__all_sync(0xffffffffu, ok)) break;
                }
            }
        }
    } else {
        if constexpr (CHUNKS > HEAD_SPLIT_ABOVE) set_max_regs_up<HEAD_REGS_MANY>();
        const int q = warp & 3;              // TMEM lane quarter this warp may read
        const int half = (warp - HEAD_EPI_FIRST) >> 2;    // the quarter's two warps take alternate chunks of 32 columns
        const uint32_t tempty0 = map_to_cta(smem_u32(s.tempty), 0);
        int acc = 0;
        uint32_t acc_phase = 0;
        int ok = 1;
        if (p.lora_b) pdl_wait();
        const HeadTiles tiles(p);
        const int n_items = p.n_vtile * tiles.n_ntile;
        unsigned mixed = 0;  // bit g: group g of the tile is mixed
        const int n_seg = SEGMENTED ? (n_kstage + HEAD_SEGMENT - 1) / HEAD_SEGMENT : 1;
        for (int item = pair; item < n_items; item += n_pairs) {
            const int v = (item / tiles.n_ntile) * 2 * BM + rank * BM + q * 32 + lane;
            const int col0 = (item % tiles.n_ntile) * tiles.n_tok;
            const int col_end = min(tiles.n_col, col0 + tiles.n_tok);
            const float bias = (p.bias && v < p.V) ? __ldg(p.bias + v) : 0.0f;
            if (p.lora_b && (item == pair || tiles.n_ntile > 1))
                mixed = __ballot_sync(0xffffffffu, lane < HEAD_MAX_RUNS && col0 + lane * HEAD_GROUP < col_end &&
                                                       group_adapter(p, col0 / HEAD_GROUP + lane) == GROUP_MIXED);
            float sum[SEGMENTED ? CHUNKS : 1][32];
#pragma unroll
            for (int c = 0; c < CHUNKS; ++c)
#pragma unroll
                for (int j = 0; j < 32; ++j) sum[c][j] = 0.0f;
            for (int seg = 0; seg < n_seg; ++seg) {
                // an abandoned wait: the rest of this CTA's tiles is written as NaN
                if (ok) ok = mbar_wait(smem_u32(&s.tfull[acc]), acc_phase, s.abort_flag, p.status, ERR_WAIT_TMEM_FULL);
                ok = __all_sync(0xffffffffu, ok);
                if (ok) tc_fence_after();
                const uint32_t taddr = tmem_base + acc * acc_cols + (uint32_t(q * 32) << 16);
                if constexpr (SEGMENTED) {
#pragma unroll
                    for (int c = 0; c < CHUNKS; ++c) {
                        const int col = half * 32 + c * 64;
                        if (col0 + col < col_end && ok) {  // uniform over the warp
                            constexpr int W = CHUNKS > 3 ? 16 : 32;  // the sums leave few registers
#pragma unroll
                            for (int j0 = 0; j0 < 32; j0 += W) {
                                uint32_t r[W];
                                if constexpr (W == 16) tmem_ld16(taddr + col + j0, r); else tmem_ld32(taddr + col + j0, r);
                                tmem_ld_wait();
#pragma unroll
                                for (int j = 0; j < W; ++j) sum[c][j0 + j] += __uint_as_float(r[j]);
                            }
                        }
                    }
                } else {
#pragma unroll 1
                    for (int c0 = col0 + half * 32; c0 < col_end; c0 += 64) {
                        float x[32];
                        uint32_t r[32];
                        if (ok) {
                            tmem_ld32(taddr + (c0 - col0), r);
                            tmem_ld_wait();
                        }
#pragma unroll
                        for (int j = 0; j < 32; ++j) x[j] = ok ? __uint_as_float(r[j]) : __int_as_float(0x7fc00000);
                        finish_chunk<BT, false>(p, tiles, v, bias, c0, col_end, mixed >> ((c0 - col0) / HEAD_GROUP), x);
                    }
                }
                tc_fence_before();
                __syncwarp();
                if (ok && lane == 0) mbar_arrive_cluster_relaxed(tempty0 + 8 * acc);
                if (++acc == p.n_acc) {
                    acc = 0;
                    acc_phase ^= 1u;
                }
            }
            if constexpr (SEGMENTED) {
#pragma unroll
                for (int c = 0; c < CHUNKS; ++c) {  // in place: the sums fill the registers
                    const int c0 = col0 + half * 32 + c * 64;
                    if (c0 < col_end) {
                        if (!ok)
#pragma unroll
                            for (int j = 0; j < 32; ++j) sum[c][j] = __int_as_float(0x7fc00000);
                        finish_chunk<BT, true>(p, tiles, v, bias, c0, col_end, mixed >> ((c0 - col0) / HEAD_GROUP), sum[c]);
                    }
                }
            }
        }
    }

    // tear-down: the leader waits (bounded, whether or not a wait was abandoned before) for its MMAs, and after an abandoned
    // wait for the loads of both CTAs that it announced; neither CTA leaves, or frees TMEM, while the other may still read
    // its shared memory or signal its barriers
    tc_fence_before();
    __syncthreads();
    if (rank == 0) {
        int unset = 0;
        if (warp == 1 && elect_one()) {  // the lane that issued them: a commit covers its own thread's MMAs
            tc_commit_pair(smem_u32(s.tdown));
            mbar_wait(smem_u32(s.tdown), 0, &unset, p.status, ERR_WAIT_TEARDOWN);
        }
        if (warp == 0 && *s.abort_flag && elect_one()) {
            const int stage = s.ring_end[0], phase = s.ring_end[1], n_stage = s.ring_end[2];
            for (int i = 0; i < n_stage && !unset; ++i)  // stages from `stage` on were last filled a round earlier, if ever
                mbar_wait(smem_u32(&s.full[i]), uint32_t(i < stage ? phase : phase ^ 1), &unset, p.status, ERR_WAIT_TEARDOWN,
                          HEAD_DRAIN_CYCLES);
        }
    }
    __syncwarp();
    cluster_arrive();
    cluster_wait();
    if (warp == 1) {
        tc_fence_after();
        tmem_dealloc_pair(tmem_base, TMEM_COLS);
    }
}

// The columns in order of their adapter: column runs of one adapter each, padded to whole groups of 16, tokens
// without an adapter last; within a run in order of the tokens.  One block: counts, starts, and then the tokens
// 1024 at a time, the warps one after the other, so that a token's place is the number of those before it.
constexpr int LAYOUT_THREADS = 1024;
constexpr int LAYOUT_MAX_ADAPTERS = 8192;  // their places are in shared memory

struct LayoutParams {
    const void* ids;
    int ids_i64;
    int n_adapters, T, n_col;  // n_col: room in col_token
    int* col_token;
    int* n_col_dev;
    int* group;
};

__global__ void __launch_bounds__(LAYOUT_THREADS)
adapter_layout_kernel(const LayoutParams p) {
    extern __shared__ int place[];  // [n_adapters + 1]: counts, then the next free column of every run
    __shared__ int warp_sum[32];
    __shared__ int base;
    pdl_launch();
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5;
    const int n = p.n_adapters + 1;
    auto id_of = [&](int t) -> int {
        const long long a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[t]
                                      : (long long)reinterpret_cast<const int*>(p.ids)[t];
        return (a >= 0 && a < p.n_adapters) ? int(a) : p.n_adapters;
    };
    for (int a = tid; a < n; a += LAYOUT_THREADS) place[a] = 0;
    if (tid == 0) base = 0;
    __syncthreads();
    const int first_id = tid < p.T ? id_of(tid) : 0;
    for (int t = tid; t < p.T; t += LAYOUT_THREADS) atomicAdd(&place[t == tid ? first_id : id_of(t)], 1);
    __syncthreads();
    for (int a0 = 0; a0 < n; a0 += LAYOUT_THREADS) {  // starts, and the padding behind every run
        const int a = a0 + tid;
        const int count = a < n ? place[a] : 0;
        const int padded = (count + HEAD_GROUP - 1) / HEAD_GROUP * HEAD_GROUP;
        int incl = padded;
#pragma unroll
        for (int o = 1; o < 32; o <<= 1) {
            const int v = __shfl_up_sync(0xffffffffu, incl, o);
            if (lane >= o) incl += v;
        }
        if (lane == 31) warp_sum[warp] = incl;
        __syncthreads();
        int first = base + incl - padded;
        for (int w = 0; w < warp; ++w) first += warp_sum[w];
        if (a < n) {
            place[a] = first;
            for (int at = first + count; at < min(first + padded, p.n_col); ++at) p.col_token[at] = -1;
            for (int at = first; at < min(first + padded, p.n_col); at += HEAD_GROUP)
                p.group[at / HEAD_GROUP] = a < p.n_adapters ? a : GROUP_NONE;
        }
        __syncthreads();
        if (tid == LAYOUT_THREADS - 1) base = first + padded;
        __syncthreads();
    }
    if (tid == 0) *p.n_col_dev = base;
    for (int t0 = 0; t0 < p.T; t0 += LAYOUT_THREADS) {
        const int t = t0 + tid;
        const int id = t >= p.T ? -1 : t0 == 0 ? first_id : id_of(t);
        const unsigned peers = __match_any_sync(0xffffffffu, id);
        const int leader = __ffs(peers) - 1;
        const int n_warp = min(32, (p.T - t0 + 31) / 32);
        for (int w = 0; w < n_warp; ++w) {
            if (warp == w) {
                int at = 0;
                if (lane == leader && id >= 0) {
                    at = place[id];
                    place[id] = at + __popc(peers);
                }
                at = __shfl_sync(0xffffffffu, at, leader) + __popc(peers & ((1u << lane) - 1));
                if (id >= 0 && at < p.n_col) p.col_token[at] = t;
            }
            __syncthreads();
        }
    }
}

// h[column][j] = scale[a] * (A[a][j] . e_t), t and a the column's token and its adapter; zero without an adapter and
// for the padding ranks; in fp32 and in the 16-bit terms.  Without a column order the blocks of rank 0 also
// write the groups' adapters; with one, the blocks of the last eight y gather the columns' rows of e, a column each.
// One block per (8 consecutive columns, 4 ranks): its 8 warps split D, each lane reads 16 bytes of the
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
    const int* col_token;  // null: column = token
    const int* n_col_dev;
    void* e_cols;          // with col_token: [column][ld_cols], the rows of e in column order, zero padded
    long long ld_cols;
    int rank_blocks;       // blocks in y that compute; with col_token eight more copy
    long long D;
    int vec;  // 16-byte loads are possible for every row
    float* h;
    int ldh;
    void* h16;          // [T][HPack::pitch] in the 16-bit type of e, or null: every group is mixed
    int* group;         // [ceil(T / 16)]
    int* group_bad;     // [ceil(T / 16)], zero before the launch
    unsigned* h_max;    // fp16: [16 ceil(T / 16)], zero before the launch; else null
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

__device__ __forceinline__ __nv_bfloat16 cut_off(float x, __nv_bfloat16) { return __float2bfloat16_rz(x); }
__device__ __forceinline__ __half cut_off(float x, __half) { return __float2half_rz(x); }
__device__ __forceinline__ __nv_bfloat16 next_to_zero(__nv_bfloat16 x) { return __ushort_as_bfloat16(__bfloat16_as_ushort(x) - 1); }
__device__ __forceinline__ __half next_to_zero(__half x) { return __ushort_as_half(__half_as_ushort(x) - 1); }

// x as the sum of H_TERMS 16-bit numbers of its sign, none of them zero: an infinite entry of B then gives an infinity,
// where terms of two signs would give inf - inf and a zero term inf x 0.  Every term but the last is what it has to
// represent cut off, one step less where nothing would be left.  What is lost is half a step of the last term: 2^-22 of x, but
// at least 2^-25, in fp16 with two terms, 2^-23 of x in bf16 with three (with two it would be 2^-16, and show in fp32 logits).
template <typename T>
struct SplitH {
    T term[H_TERMS<T>];
    __device__ __forceinline__ explicit SplitH(float x) {
#pragma unroll
        for (int t = 0; t < H_TERMS<T>; ++t) {
            if (t == H_TERMS<T> - 1) {
                term[t] = T(x);
            } else {
                term[t] = cut_off(x, T());
                if (float(T(x - float(term[t]))) == 0.0f && float(term[t]) != 0.0f) term[t] = next_to_zero(term[t]);
                x -= float(term[t]);
            }
        }
    }
};

template <typename T>
__global__ void __launch_bounds__(SHRINK_WARPS * 32)
adapter_shrink_kernel(const ShrinkParams p) {
    constexpr int VE = 16 / int(sizeof(T));
    __shared__ float part[SHRINK_WARPS][SHRINK_TOK * SHRINK_RANK];
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int tok0 = blockIdx.x * SHRINK_TOK, rank0 = blockIdx.y * SHRINK_RANK;  // tok0: a column
    pdl_launch();
    const T* E = reinterpret_cast<const T*>(p.e);
    int ids[SHRINK_TOK], tok[SHRINK_TOK];
    int ntok;
    if (p.col_token) {
        pdl_wait();
        ntok = min(SHRINK_TOK, *p.n_col_dev - tok0);
        if (ntok <= 0) return;
        const int a = p.group[tok0 / HEAD_GROUP];
#pragma unroll
        for (int i = 0; i < SHRINK_TOK; ++i) {
            tok[i] = i < ntok ? p.col_token[tok0 + i] : -1;
            ids[i] = tok[i] >= 0 ? a : -1;
        }
        if (int(blockIdx.y) >= p.rank_blocks) {
            const int col = tok0 + blockIdx.y - p.rank_blocks;
            const int t = col < *p.n_col_dev ? p.col_token[col] : -1;
            if (t < 0) return;  // padding columns are never stored: whatever is there may be multiplied
            T* dst = reinterpret_cast<T*>(p.e_cols) + (size_t)col * p.ld_cols;
            for (long long d = threadIdx.x * VE; d < p.ld_cols; d += SHRINK_WARPS * 32 * VE)
                *reinterpret_cast<uint4*>(dst + d) = load_piece(E + (size_t)t * p.lde + d, p.D - d, p.vec != 0);
            return;
        }
    } else {
        ntok = min(SHRINK_TOK, p.T - tok0);
        if (blockIdx.y == 0 && tok0 % HEAD_GROUP == 0 && warp == 0) {
            const int n = min(HEAD_GROUP, p.T - tok0);
            long long a = -1;
            if (lane < n)
                a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[tok0 + lane]
                              : (long long)reinterpret_cast<const int*>(p.ids)[tok0 + lane];
            const int id = (a >= 0 && a < p.n_adapters) ? int(a) : -1;
            const int first = __shfl_sync(0xffffffffu, id, 0);
            const bool same = __all_sync(0xffffffffu, lane >= n || id == first);
            if (lane == 0) p.group[tok0 / HEAD_GROUP] = same && (first < 0 || p.h16) ? first : GROUP_MIXED;
        }
#pragma unroll
        for (int i = 0; i < SHRINK_TOK; ++i) {
            long long a = -1;
            if (i < ntok)
                a = p.ids_i64 ? reinterpret_cast<const long long*>(p.ids)[tok0 + i]
                              : (long long)reinterpret_cast<const int*>(p.ids)[tok0 + i];
            ids[i] = (a >= 0 && a < p.n_adapters) ? int(a) : -1;
            tok[i] = tok0 + i;
        }
    }
    float acc[SHRINK_TOK][SHRINK_RANK];
#pragma unroll
    for (int i = 0; i < SHRINK_TOK; ++i)
#pragma unroll
        for (int k = 0; k < SHRINK_RANK; ++k) acc[i][k] = 0.0f;

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
        if (a < 0 || rank0 >= p.rank) continue;  // uniform over the block; padding ranks are zeros
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
                    const uint4 ev = load_piece(E + (size_t)tok[i] * p.lde + d, p.D - d, p.vec != 0);
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
        sum = (a >= 0 && k < p.rank) ? sum : 0.0f;
        if (i < ntok) {
            if (k < p.ldh) p.h[(size_t)(tok0 + i) * p.ldh + k] = sum;
            if constexpr (sizeof(T) == 2) {
                if (p.h16) {
                    // |x| up to 2^15: above it, or not finite, and the group goes to the fp32 path; so it does for x too
                    // small for terms that are not zero (2^-23 is two steps of fp16; bf16 reaches as far as fp32)
                    const float x = fabsf(sum), least = H_TERMS<T> == 2 ? 0x1p-23f : 0x1p-100f;
                    if (!(x <= 32768.0f) || (x < least && x > 0.0f)) {
                        p.group_bad[(tok0 + i) / HEAD_GROUP] = 1;
                        sum = 0.0f;
                    }
                    // the order of the bits is the order of the numbers
                    if (p.h_max && x > 0.0f && k < p.rank) atomicMax(&p.h_max[tok0 + i], __float_as_uint(x));
                    const HPack pack(p.rank, H_TERMS<T>);
                    T* row = reinterpret_cast<T*>(p.h16) + (size_t)(tok0 + i) * pack.pitch;
                    const SplitH<T> h(sum);
#pragma unroll
                    for (int t = 0; t < H_TERMS<T>; ++t)
                        if (k < pack.ranks) row[pack.at(k, t)] = h.term[t];
                }
            }
        }
    }
}

}  // namespace cce
