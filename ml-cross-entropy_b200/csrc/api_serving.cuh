// Host side of the head's serving entry points (cce_b200_logits, cce_b200_sample); included by api.cu.
#pragma once

namespace {

int check_logits_args(const cce_b200_logits_args* a) {
    if (!a) return CCE_ERR_ARG;
    int rc = check_operands(&a->op);
    if (rc) return rc;
    const cce_b200_operands& op = a->op;
    if (op.valids || op.n_rows_dev || op.n_rows != op.n_total) return CCE_ERR_ARG;  // every token gets its logits
    if (a->out_dtype < 0 || a->out_dtype > 2) return CCE_ERR_ARG;
    if (a->lora_a || a->lora_b || a->adapter_ids) {
        if (!a->lora_a || !a->lora_b || !a->adapter_ids) return CCE_ERR_ARG;
        if (a->n_adapters <= 0 || a->n_adapters >= (1LL << 31)) return CCE_ERR_ARG;
        if (a->rank <= 0 || a->rank > CCE_B200_MAX_RANK) return CCE_ERR_ARG;
        if (a->ids_dtype != CCE_IDX_I32 && a->ids_dtype != CCE_IDX_I64) return CCE_ERR_ARG;
    }
    return CCE_OK;
}

inline int h_terms(int dtype) { return dtype == CCE_DT_BF16 ? H_TERMS<__nv_bfloat16> : H_TERMS<__half>; }

struct LogitsPlan {
    OperandPlan ops;
    long long ldh, n_col, n_group;
    bool sorted;         // the columns are ordered by adapter
    int pitch16;         // row length of the 16-bit h; 0: every group of columns is mixed
    int shrink_ranks;    // ranks that the shrink kernel writes: whole padding blocks of both forms of h
    long long ld_cols;
    size_t off_bad, off_h_max, cleared, off_group, off_cols, off_ncol, off_e_cols, off_h, off_h16, total;
};

LogitsPlan plan_logits(const cce_b200_logits_args* a) {
    LogitsPlan pl = {};
    const long long T = a->op.n_total;
    pl.n_col = T;
    bool mma = false;
    if (a->lora_b) {
        // TMA reads the adapters' rows: 16-byte pitch and base
        mma = a->op.dtype != CCE_DT_F32 && a->rank % 8 == 0 && (reinterpret_cast<uintptr_t>(a->lora_b) & 15) == 0;
        // Columns ordered by adapter: each run is padded by 0 to 15 columns, about half a group.  They are free while
        // the product is bound by reading the classifier (up to 256 columns) and cheaper than mixed groups up to
        // twice the tokens.
        const long long runs = std::min<long long>(T, a->n_adapters + 1);
        pl.sorted = mma && T > 1 && a->n_adapters < LAYOUT_MAX_ADAPTERS && T + HEAD_GROUP / 2 * runs <= std::max<long long>(BN, 2 * T);
        if (pl.sorted) pl.n_col = cdiv(T + (HEAD_GROUP - 1) * runs, HEAD_GROUP) * HEAD_GROUP;  // at most
        pl.n_group = cdiv(pl.n_col, HEAD_GROUP);
    }
    // the status word and, behind it, the flags that are cleared with it
    size_t off = 256;
    auto take = [&](size_t bytes) {
        const size_t at = off;
        off = align_up(off + bytes, 256);
        return at;
    };
    pl.off_bad = take((size_t)pl.n_group * 4);
    pl.off_h_max = take(mma && a->op.dtype == CCE_DT_F16 ? (size_t)pl.n_group * HEAD_GROUP * 4 : 0);
    pl.cleared = off;
    pl.off_group = take((size_t)pl.n_group * 4);
    if (pl.sorted) {
        pl.off_cols = take((size_t)pl.n_col * 4);
        pl.off_ncol = take(4);
    }
    pl.ops = plan_operands(&a->op, off, pl.sorted);  // ordered columns bring their own copy of e
    off = pl.ops.end;
    if (pl.sorted) {
        pl.ld_cols = cdiv(a->op.D, 8) * 8;
        pl.off_e_cols = take((size_t)pl.n_col * pl.ld_cols * 2);
    }
    if (a->lora_b) {
        pl.ldh = cdiv(a->rank, ADAPTER_RANK_PAD) * ADAPTER_RANK_PAD;
        const HPack pack((int)a->rank, h_terms(a->op.dtype));
        pl.pitch16 = mma ? pack.pitch : 0;
        pl.shrink_ranks = mma ? pack.ranks : (int)pl.ldh;
        pl.off_h = take((size_t)pl.n_col * pl.ldh * 4);
        pl.off_h16 = take((size_t)pl.n_col * pl.pitch16 * 2);
    }
    pl.total = off;
    return pl;
}

// Launches with the leave to start while the kernel before it in the stream still runs (a kernel that waits for it
// itself before it reads what that one wrote).
template <typename K, typename... Args>
int launch_behind(K* kernel, dim3 grid, int threads, int smem, cudaStream_t st, bool overlap, const Args&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = grid;
    cfg.blockDim = dim3(threads);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = overlap ? 1 : 0;
    cudaLaunchKernelEx(&cfg, kernel, args...);
    CCE_LAUNCH_CHECK();
    return CCE_OK;
}

template <typename T>
int launch_shrink(const ShrinkParams& sp, long long n_col, cudaStream_t st) {
    const dim3 grid((unsigned)cdiv(n_col, SHRINK_TOK), (unsigned)(sp.rank_blocks + (sp.col_token ? SHRINK_TOK : 0)));
    return launch_behind(adapter_shrink_kernel<T>, grid, SHRINK_WARPS * 32, 0, st, sp.col_token != nullptr, sp);
}

// What a form of the kernel needs before its first launch on a device.
template <typename T, int CHUNKS>
int setup_head() {
    CCE_CUDA(cudaFuncSetAttribute(head_logits_kernel<T, CHUNKS>, cudaFuncAttributeMaxDynamicSharedMemorySize, HEAD_SMEM));
    if (CHUNKS > HEAD_SPLIT_ABOVE) {
        // the split hands out what the block was launched with: with fewer it would wait for good
        cudaFuncAttributes attr;
        CCE_CUDA(cudaFuncGetAttributes(&attr, head_logits_kernel<T, CHUNKS>));
        if (attr.numRegs != HEAD_REGS) return CCE_ERR_UNSUPPORTED;
    }
    return CCE_OK;
}

// With adapters the projection may start while the shrink kernel, launched just before it, still runs.
template <typename T, int CHUNKS>
int launch_head_form(DeviceInfo* dev, int dtype, const HeadMaps& maps, const HeadParams& hp, int grid, cudaStream_t st) {
    std::atomic<bool>& set = dev->head_set[dtype][CHUNKS];
    if (!set) {
        const int rc = setup_head<T, CHUNKS>();
        if (rc) return rc;
        set = true;
    }
    return launch_behind(head_logits_kernel<T, CHUNKS>, dim3(grid), HEAD_THREADS, HEAD_SMEM, st, hp.lora_b != nullptr, maps, hp);
}

template <typename T>
int launch_head(DeviceInfo* dev, int dtype, const HeadMaps& maps, const HeadParams& hp, int grid, cudaStream_t st) {
    if (hp.out_dtype != CCE_DT_F32) return launch_head_form<T, 0>(dev, dtype, maps, hp, grid, st);
    if (hp.n_tok <= 64) return launch_head_form<T, 1>(dev, dtype, maps, hp, grid, st);
    if (hp.n_tok <= 128) return launch_head_form<T, 2>(dev, dtype, maps, hp, grid, st);
    if (hp.n_tok <= 192) return launch_head_form<T, 3>(dev, dtype, maps, hp, grid, st);
    return launch_head_form<T, 4>(dev, dtype, maps, hp, grid, st);
}

// The adapters' rows of B, [n][V][rank], as a 3-D map: a box of 16, 32 or 64 ranks x 128 classifier rows of one
// adapter, in the swizzle of its width.
int make_tmap_adapters(CUtensorMap* m, const void* base, int dtype, long long rank, long long V, long long n) {
    EncodeTiledFn enc = get_encode();
    if (!enc) {
        g_last_cuda = -1;
        return CCE_ERR_CUDA;
    }
    cuuint64_t dims[3] = {(cuuint64_t)rank, (cuuint64_t)V, (cuuint64_t)n};
    cuuint64_t strides[2] = {(cuuint64_t)rank * 2, (cuuint64_t)(rank * V) * 2};
    const int width = AdapterPack((int)rank, h_terms(dtype)).width;
    cuuint32_t box[3] = {(cuuint32_t)width, (cuuint32_t)BM, 1};
    cuuint32_t estr[3] = {1, 1, 1};
    CUresult r = enc(m, dtype == CCE_DT_BF16 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16,
                     3, const_cast<void*>(base), dims, strides, box, estr, CU_TENSOR_MAP_INTERLEAVE_NONE,
                     width == 16   ? CU_TENSOR_MAP_SWIZZLE_32B
                     : width == 32 ? CU_TENSOR_MAP_SWIZZLE_64B
                                   : CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                     CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) {
        g_last_cuda = int(r);
        return CCE_ERR_CUDA;
    }
    return CCE_OK;
}

// Positions per CTA for a row of V logits over `cluster` CTAs: whole blocks.
inline int sample_slice(long long V, int cluster) { return int(cdiv(cdiv(V, cluster), SMP_BLK) * SMP_BLK); }

struct SamplePlan {
    int cluster, slice, smem;  // of sample_kernel
    bool stream, filters;      // sample_stream.cuh's kernels; with top-k or top-p
    int n_chunk;
    size_t off_max, off_sum, off_blk, off_hist, off_list, total;
};

int plan_sample(const cce_b200_sample_args* a, SamplePlan* out) {
    if (!a || a->B < 0 || a->V <= 0 || a->ld < a->V) return CCE_ERR_ARG;
    if (a->dtype != CCE_DT_F16 && a->dtype != CCE_DT_BF16 && a->dtype != CCE_DT_F32) return CCE_ERR_ARG;
    SamplePlan pl = {};
    const int elem = a->dtype == CCE_DT_F32 ? 4 : 2;
    if (a->V > (1 << 20)) return CCE_ERR_TOO_LARGE;  // the weights keep at least 42 bits
    // CTAs per row.  Few rows: short slices (fp32, 1 x 256000: 20 us with 16384 positions, 24 with 32768; 16 x 256000,
    // top-p: 81 and 88; 31 x 128256: 53 and 51); many rows: fewer, longer ones, whose fixed cost is paid less often
    // (bf16, 64 x 128256, top-k and top-p: 41 and 29; top-p: 97 and 66; 100 x 152064: 287 and 164).
    const int longest = a->B >= 32 ? 32768 : 16384;
    pl.cluster = 1;
    while (pl.cluster < SMP_MAX_CLUSTER && sample_slice(a->V, pl.cluster) > longest) pl.cluster *= 2;
    pl.slice = sample_slice(a->V, pl.cluster);
    pl.smem = SampleLayout(pl.cluster, pl.slice, elem).bytes;
    if (pl.smem > SMP_SMEM) return CCE_ERR_TOO_LARGE;
    if (a->B * pl.cluster >= (1LL << 31)) return CCE_ERR_ARG;
    pl.filters = a->top_k || a->top_p || a->top_k_all > 0 || a->top_p_all < 1.0;
    // From 32 MB of logits on the streaming kernels win: fp32, no filters / top-p / top-k and top-p, 64 x 128000: 41 / 84 /
    // 55 us against one cluster per row's 41 / 109 / 55, 128 x 256000: 92 / 182 / 121 against 133 / 334 / 162; bf16,
    // 64 x 128000: 37 / 80 / 53 against 31 / 72 / 39, 128 x 128000: 51 / 109 / 72 against 51 / 127 / 64.
    // But only with long rows: while a row's logits leave room for a second CTA on the SM the clusters win.  64 MB,
    // streaming against clusters: fp32, rows of 15000: 67 / 182 / 121 against 60 / 157 / 95, 16000: 66 / 176 / 118 against
    // 85 / 200 / 120; bf16, 31000: 91 / 230 / 146 against 79 / 204 / 114, 33000: 95 / 242 / 157 against 104 / 283 / 167.
    // (Their workspace, 24 KB for a row with a filter, would be many times the logits of short rows.)
    const long long row_bytes = a->V * elem;
    pl.stream = row_bytes >= (62LL << 10) && a->B * row_bytes >= (32LL << 20);
    pl.total = 256;
    if (pl.stream) {
        pl.n_chunk = (int)cdiv(a->V + 16 / elem - 1, STR_CHUNK);
        if (a->B * pl.n_chunk >= (1LL << 31)) return CCE_ERR_ARG;
        size_t off = align_up((size_t)a->B * sizeof(RowState), 256);
        auto take = [&](size_t bytes) {
            const size_t at = off;
            off = align_up(off + bytes, 256);
            return at;
        };
        const size_t chunks = (size_t)a->B * pl.n_chunk;
        pl.off_max = take(chunks * sizeof(float));
        pl.off_sum = take(chunks * sizeof(u64));
        pl.off_blk = take(chunks * STR_BLOCKS * sizeof(u64));
        pl.off_hist = take(pl.filters ? (size_t)a->B * STR_BINS * sizeof(uint32_t) : 0);
        pl.off_list = take(pl.filters ? (size_t)a->B * SMP_LIST * sizeof(u64) : 0);
        pl.total = off;
    }
    *out = pl;
    return CCE_OK;
}

template <typename T>
int launch_sample(DeviceInfo* dev, int dtype, const SampleParams& sp, const SamplePlan& pl, long long B, char* ws,
                  cudaStream_t st) {
    std::atomic<bool>& set = dev->sample_set[dtype];
    if (!set) {
        CCE_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeMaxDynamicSharedMemorySize, SMP_SMEM));
        CCE_CUDA(cudaFuncSetAttribute(sample_kernel<T>, cudaFuncAttributeNonPortableClusterSizeAllowed, 1));
        set = true;
    }
    RowState* only = nullptr;
    if (pl.stream) {
        StreamBuffers b = {};
        b.state = reinterpret_cast<RowState*>(ws);
        b.chunk_max = reinterpret_cast<float*>(ws + pl.off_max);
        b.chunk_sum = reinterpret_cast<u64*>(ws + pl.off_sum);
        b.blk_mass = reinterpret_cast<u64*>(ws + pl.off_blk);
        b.hist = pl.filters ? reinterpret_cast<uint32_t*>(ws + pl.off_hist) : nullptr;
        b.list = reinterpret_cast<u64*>(ws + pl.off_list);
        b.n_chunk = pl.n_chunk;
        const dim3 chunks((unsigned)(B * pl.n_chunk)), rows((unsigned)B);
        const int draw_smem = (3 * SMP_LIST + pl.n_chunk * STR_BLOCKS) * (int)sizeof(u64);
        int rc = launch_behind(row_max_kernel<T>, chunks, SMP_THREADS, 0, st, false, sp, b);
        if (!rc)
            rc = launch_behind(row_prepare_kernel, dim3((unsigned)cdiv(B, PREP_WARPS)), 32 * PREP_WARPS, 0, st, true, sp, b, B);
        if (!rc && !pl.filters) rc = launch_behind(row_stats_kernel<T, false>, chunks, SMP_THREADS, 0, st, true, sp, b);
        if (!rc && pl.filters) rc = launch_behind(row_stats_kernel<T, true>, chunks, SMP_THREADS, 0, st, true, sp, b);
        if (!rc && pl.filters) rc = launch_behind(row_plan_kernel, rows, SMP_THREADS, 0, st, true, sp, b);
        if (!rc && pl.filters) rc = launch_behind(row_pass_kernel<T>, chunks, SMP_THREADS, 0, st, true, sp, b);
        if (!rc) rc = launch_behind(row_draw_kernel<T>, rows, SMP_THREADS, draw_smem, st, true, sp, b);
        if (rc || !pl.filters) return rc;
        only = b.state;
    }
    cudaLaunchConfig_t cfg = {};
    // behind the streaming kernels few rows are left, if any: what the GPU holds at a time
    cfg.gridDim = dim3((unsigned)((only ? std::min<long long>(B, 256 / pl.cluster) : B) * pl.cluster));
    cfg.blockDim = dim3(SMP_THREADS);
    cfg.dynamicSmemBytes = pl.smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[2];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = pl.cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    attr[1].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    attr[1].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = attr;
    cfg.numAttrs = only ? 2 : 1;
    cudaLaunchKernelEx(&cfg, sample_kernel<T>, sp, (const RowState*)only, B);
    CCE_LAUNCH_CHECK();
    return CCE_OK;
}

}  // namespace

extern "C" {

size_t cce_b200_logits_workspace_bytes(const cce_b200_logits_args* a) {
    if (check_logits_args(a)) return 0;
    return plan_logits(a).total;
}

int cce_b200_logits(const cce_b200_logits_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    int rc = check_logits_args(a);
    if (rc) return rc;
    const cce_b200_operands& op = a->op;
    if (op.n_total == 0) return CCE_OK;
    if (!a->out || !workspace) return CCE_ERR_ARG;
    const LogitsPlan pl = plan_logits(a);
    if (workspace_bytes < pl.total) return CCE_ERR_WORKSPACE;
    if (reinterpret_cast<uintptr_t>(workspace) & 255) return CCE_ERR_ALIGN;
    if (pl.n_col >= (1LL << 31) - BN) return CCE_ERR_ARG;
    DeviceInfo* dev;
    rc = device_info(&dev);
    if (rc) return rc;
    char* ws = reinterpret_cast<char*>(workspace);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    CCE_CUDA(cudaMemsetAsync(ws, 0, pl.cleared, st));
    Staged sg;
    rc = stage_operands(&op, pl.ops, ws, st, &sg, pl.sorted ? ws + pl.off_e_cols : nullptr);
    if (rc) return rc;

    const int elem = op.dtype == CCE_DT_F32 ? 4 : 2;
    auto aligned16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
    unsigned* const h_max = pl.pitch16 && op.dtype == CCE_DT_F16 ? reinterpret_cast<unsigned*>(ws + pl.off_h_max) : nullptr;
    const int* col_token = pl.sorted ? reinterpret_cast<const int*>(ws + pl.off_cols) : nullptr;
    const int* n_col_dev = pl.sorted ? reinterpret_cast<const int*>(ws + pl.off_ncol) : nullptr;
    if (pl.sorted) {
        LayoutParams lp = {};
        lp.ids = a->adapter_ids;
        lp.ids_i64 = a->ids_dtype == CCE_IDX_I64;
        lp.n_adapters = (int)a->n_adapters;
        lp.T = (int)op.n_total;
        lp.n_col = (int)pl.n_col;
        lp.col_token = reinterpret_cast<int*>(ws + pl.off_cols);
        lp.n_col_dev = reinterpret_cast<int*>(ws + pl.off_ncol);
        lp.group = reinterpret_cast<int*>(ws + pl.off_group);
        adapter_layout_kernel<<<1, LAYOUT_THREADS, (a->n_adapters + 1) * sizeof(int), st>>>(lp);
        CCE_LAUNCH_CHECK();
        sg.e = ws + pl.off_e_cols;
        sg.lde = pl.ld_cols;
    }
    if (a->lora_b) {
        ShrinkParams sp = {};
        sp.e = op.e;
        sp.lde = op.lde;
        sp.lora_a = a->lora_a;
        sp.scale = a->lora_scale;
        sp.ids = a->adapter_ids;
        sp.ids_i64 = a->ids_dtype == CCE_IDX_I64;
        sp.n_adapters = (int)a->n_adapters;
        sp.rank = (int)a->rank;
        sp.T = (int)op.n_total;
        sp.col_token = col_token;
        sp.n_col_dev = n_col_dev;
        sp.e_cols = ws + pl.off_e_cols;
        sp.ld_cols = pl.ld_cols;
        sp.rank_blocks = pl.shrink_ranks / SHRINK_RANK;
        sp.D = op.D;
        sp.vec = aligned16(op.e) && aligned16(a->lora_a) && (op.D * elem) % 16 == 0 && (op.lde * elem) % 16 == 0;
        sp.h = reinterpret_cast<float*>(ws + pl.off_h);
        sp.ldh = (int)pl.ldh;
        sp.h16 = pl.pitch16 ? ws + pl.off_h16 : nullptr;
        sp.group = reinterpret_cast<int*>(ws + pl.off_group);
        sp.group_bad = reinterpret_cast<int*>(ws + pl.off_bad);
        sp.h_max = h_max;
        if (op.dtype == CCE_DT_F32)
            rc = launch_shrink<float>(sp, pl.n_col, st);
        else if (op.dtype == CCE_DT_BF16)
            rc = launch_shrink<__nv_bfloat16>(sp, pl.n_col, st);
        else
            rc = launch_shrink<__half>(sp, pl.n_col, st);
        if (rc) return rc;
    }

    HeadParams hp = {};
    hp.T = (int)op.n_total;
    hp.V = (int)op.V;
    hp.n_kblk = (int)cdiv(sg.Dk, BK);
    hp.n_col = (int)pl.n_col;
    hp.col_token = col_token;
    hp.n_col_dev = n_col_dev;
    hp.out_dtype = a->out_dtype;
    // Columns that only the device can count may be far fewer than the bound: there a tile has room for as many as
    // possible.
    const long long n_ntile = cdiv(pl.n_col, BN);
    hp.n_tok = n_ntile > 1 && pl.sorted ? BN : (int)(cdiv(cdiv(pl.n_col, n_ntile), HEAD_GROUP) * HEAD_GROUP);
    // where the device counts the columns, four sizes of token loads, in whole groups of 8 rows
    hp.e_step = pl.sorted ? (int)(cdiv(cdiv(hp.n_tok / 2, HEAD_E_MAPS), 8) * 8) : hp.n_tok / 2;
    hp.n_acc = hp.n_tok <= 64 ? HEAD_MAX_ACC : hp.n_tok <= 128 ? HEAD_MAX_ACC / 2 : 2;
    hp.n_vtile = (int)cdiv(op.V, 2 * BM);
    const int cdt = compute_dtype(&op);
    hp.idesc = make_idesc(cdt == CCE_DT_BF16 ? 1 : 0, 0, 0, 2 * BM, 0);
    hp.status = reinterpret_cast<int*>(ws);
    hp.bias = sg.bias;
    hp.has_softcap = op.has_softcap;
    hp.softcap = op.softcap;
    hp.out = a->out;
    if (a->lora_b) {
        hp.lora_b = a->lora_b;
        hp.ids = a->adapter_ids;
        hp.ids_i64 = a->ids_dtype == CCE_IDX_I64;
        hp.n_adapters = (int)a->n_adapters;
        hp.rank = (int)a->rank;
        hp.b_vec = aligned16(a->lora_b) && (a->rank * elem) % 16 == 0;
        hp.h = reinterpret_cast<const float*>(ws + pl.off_h);
        hp.ldh = (int)pl.ldh;
        hp.group = reinterpret_cast<const int*>(ws + pl.off_group);
        hp.group_bad = reinterpret_cast<const int*>(ws + pl.off_bad);
        hp.h_max = h_max;
    }
    HeadMaps maps;
    rc = make_tmap(&maps.c, sg.c, cdt, sg.Dk, op.V, sg.ldc, BK, BM);
    if (rc) return rc;
    for (int i = 0; i < HEAD_E_MAPS; ++i) {
        if (i > 0 && !pl.sorted) {
            maps.e[i] = maps.e[0];
            continue;
        }
        rc = make_tmap(&maps.e[i], sg.e, cdt, sg.Dk, pl.n_col, sg.lde, BK, (i + 1) * hp.e_step);
        if (rc) return rc;
    }
    maps.b = maps.h8 = maps.h32 = maps.c;
    if (pl.pitch16) {
        rc = make_tmap_adapters(&maps.b, a->lora_b, cdt, a->rank, op.V, a->n_adapters);
        if (rc) return rc;
        rc = make_tmap(&maps.h8, ws + pl.off_h16, cdt, pl.pitch16, pl.n_col, pl.pitch16, BK, 8);
        if (rc) return rc;
        rc = make_tmap(&maps.h32, ws + pl.off_h16, cdt, pl.pitch16, pl.n_col, pl.pitch16, BK, 32);
        if (rc) return rc;
    }
    const long long n_items = (long long)hp.n_vtile * n_ntile;
    if (n_items >= (1LL << 30)) return CCE_ERR_ARG;
    const int grid = 2 * (int)std::min<long long>(dev->sms / 2, n_items);
    if (op.dtype == CCE_DT_F32) return launch_head<float>(dev, op.dtype, maps, hp, grid, st);
    if (op.dtype == CCE_DT_BF16) return launch_head<__nv_bfloat16>(dev, op.dtype, maps, hp, grid, st);
    return launch_head<__half>(dev, op.dtype, maps, hp, grid, st);
}

size_t cce_b200_sample_workspace_bytes(const cce_b200_sample_args* a) {
    SamplePlan pl;
    return plan_sample(a, &pl) ? 0 : pl.total;
}

int cce_b200_sample(const cce_b200_sample_args* a, void* workspace, size_t workspace_bytes, void* stream) {
    SamplePlan pl;
    int rc = plan_sample(a, &pl);
    if (rc) return rc;
    if (a->B == 0) return CCE_OK;
    if (!a->logits || !a->u || !a->tokens || !workspace) return CCE_ERR_ARG;
    if (workspace_bytes < pl.total) return CCE_ERR_WORKSPACE;
    if ((reinterpret_cast<uintptr_t>(workspace) & 255) ||
        reinterpret_cast<uintptr_t>(a->logits) % (a->dtype == CCE_DT_F32 ? 4 : 2))
        return CCE_ERR_ALIGN;
    DeviceInfo* dev;
    rc = device_info(&dev);
    if (rc) return rc;
    SampleParams sp = {};
    sp.logits = a->logits;
    sp.ld = a->ld;
    sp.V = a->V;
    sp.u = a->u;
    sp.temperature = a->temperature;
    sp.top_k = reinterpret_cast<const long long*>(a->top_k);
    sp.top_p = a->top_p;
    sp.min_p = a->min_p;
    sp.temperature_all = a->temperature_all;
    sp.top_k_all = a->top_k_all;
    sp.top_p_all = a->top_p_all;
    sp.min_p_all = a->min_p_all;
    sp.tokens = reinterpret_cast<long long*>(a->tokens);
    sp.logprobs = a->logprobs;
    sp.slice = pl.slice;
    int log2v = 0;
    while ((1LL << log2v) < a->V) ++log2v;
    // V weights of at most 1 << frac_bits stay below 2^63
    sp.frac_bits = std::min(SMP_MAX_FRAC, 62 - log2v);
    for (int j = 0; j < SMP_TABLE; ++j) sp.table[j] = WeightFn::entry(j, sp.frac_bits);
    char* ws = reinterpret_cast<char*>(workspace);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == CCE_DT_F32) return launch_sample<float>(dev, a->dtype, sp, pl, a->B, ws, st);
    if (a->dtype == CCE_DT_BF16) return launch_sample<__nv_bfloat16>(dev, a->dtype, sp, pl, a->B, ws, st);
    return launch_sample<__half>(dev, a->dtype, sp, pl, a->B, ws, st);
}

}  // extern "C"
