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

struct LogitsPlan {
    OperandPlan ops;
    long long ldh;
    size_t off_h, total;
};

LogitsPlan plan_logits(const cce_b200_logits_args* a) {
    LogitsPlan pl;
    pl.ops = plan_operands(&a->op, 256);
    pl.ldh = a->lora_b ? cdiv(a->rank, ADAPTER_RANK_PAD) * ADAPTER_RANK_PAD : 0;
    pl.off_h = pl.ops.end;
    pl.total = align_up(pl.off_h + (size_t)a->op.n_total * pl.ldh * 4, 256);
    return pl;
}

template <typename T>
int launch_shrink(const ShrinkParams& sp, cudaStream_t st) {
    const dim3 grid((unsigned)cdiv(sp.T, SHRINK_TOK), (unsigned)(sp.ldh / SHRINK_RANK));
    adapter_shrink_kernel<T><<<grid, SHRINK_WARPS * 32, 0, st>>>(sp);
    CCE_LAUNCH_CHECK();
    return CCE_OK;
}

template <typename T>
int launch_head(const CUtensorMap& tc, const CUtensorMap& te, const HeadParams& hp, int grid, cudaStream_t st) {
    head_logits_kernel<T><<<grid, HEAD_THREADS, HEAD_SMEM, st>>>(tc, te, hp);
    CCE_LAUNCH_CHECK();
    return CCE_OK;
}

template <typename T>
int launch_sample(const SampleParams& sp, int cluster, int smem, long long B, cudaStream_t st) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)(B * cluster));
    cfg.blockDim = dim3(SMP_THREADS);
    cfg.dynamicSmemBytes = smem;
    cfg.stream = st;
    cudaLaunchAttribute attr[1];
    attr[0].id = cudaLaunchAttributeClusterDimension;
    attr[0].val.clusterDim.x = cluster;
    attr[0].val.clusterDim.y = attr[0].val.clusterDim.z = 1;
    cfg.attrs = attr;
    cfg.numAttrs = 1;
    cudaLaunchKernelEx(&cfg, sample_kernel<T>, sp);
    CCE_LAUNCH_CHECK();
    return CCE_OK;
}

// Positions per CTA for a row of V logits over `cluster` CTAs: whole blocks.
inline int sample_slice(long long V, int cluster) { return int(cdiv(cdiv(V, cluster), SMP_BLK) * SMP_BLK); }

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
    DeviceInfo* dev;
    rc = device_info(&dev);
    if (rc) return rc;
    char* ws = reinterpret_cast<char*>(workspace);
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    CCE_CUDA(cudaMemsetAsync(ws, 0, 256, st));
    Staged sg;
    rc = stage_operands(&op, pl.ops, ws, st, &sg);
    if (rc) return rc;

    const int elem = op.dtype == CCE_DT_F32 ? 4 : 2;
    auto aligned16 = [](const void* q) { return (reinterpret_cast<uintptr_t>(q) & 15) == 0; };
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
        sp.D = op.D;
        sp.vec = aligned16(op.e) && aligned16(a->lora_a) && (op.D * elem) % 16 == 0 && (op.lde * elem) % 16 == 0;
        sp.h = reinterpret_cast<float*>(ws + pl.off_h);
        sp.ldh = (int)pl.ldh;
        if (op.dtype == CCE_DT_F32)
            rc = launch_shrink<float>(sp, st);
        else if (op.dtype == CCE_DT_BF16)
            rc = launch_shrink<__nv_bfloat16>(sp, st);
        else
            rc = launch_shrink<__half>(sp, st);
        if (rc) return rc;
    }

    HeadParams hp = {};
    hp.T = (int)op.n_total;
    hp.V = (int)op.V;
    hp.n_kblk = (int)cdiv(sg.Dk, BK);
    hp.n_ntile = (int)cdiv(op.n_total, BN);
    hp.n_tok = (int)(cdiv(cdiv(op.n_total, hp.n_ntile), 16) * 16);  // even shares of the tokens
    hp.n_vtile = (int)cdiv(op.V, BM);
    hp.n_stage = std::min(HEAD_MAX_STAGES, HEAD_RING_BYTES / (A_BYTES + hp.n_tok * BK * 2));
    const int cdt = compute_dtype(&op);
    hp.idesc = make_idesc(cdt == CCE_DT_BF16 ? 1 : 0, 0, 0, BM, hp.n_tok);
    hp.status = reinterpret_cast<int*>(ws);
    hp.bias = sg.bias;
    hp.has_softcap = op.has_softcap;
    hp.softcap = op.softcap;
    hp.out = a->out;
    hp.out_dtype = a->out_dtype;
    if (a->lora_b) {
        hp.lora_b = a->lora_b;
        hp.ids = a->adapter_ids;
        hp.ids_i64 = a->ids_dtype == CCE_IDX_I64;
        hp.n_adapters = (int)a->n_adapters;
        hp.rank = (int)a->rank;
        hp.b_vec = aligned16(a->lora_b) && (a->rank * elem) % 16 == 0;
        hp.h = reinterpret_cast<const float*>(ws + pl.off_h);
        hp.ldh = (int)pl.ldh;
    }
    CUtensorMap tc, te;
    rc = make_tmap(&tc, sg.c, cdt, sg.Dk, op.V, sg.ldc, BK, BM);
    if (rc) return rc;
    rc = make_tmap(&te, sg.e, cdt, sg.Dk, op.n_total, sg.lde, BK, hp.n_tok);
    if (rc) return rc;
    const long long n_items = (long long)hp.n_vtile * hp.n_ntile;
    if (n_items >= (1LL << 31)) return CCE_ERR_ARG;
    const int grid = (int)std::min<long long>(dev->sms, n_items);
    if (op.dtype == CCE_DT_F32) return launch_head<float>(tc, te, hp, grid, st);
    if (op.dtype == CCE_DT_BF16) return launch_head<__nv_bfloat16>(tc, te, hp, grid, st);
    return launch_head<__half>(tc, te, hp, grid, st);
}

int cce_b200_sample(const cce_b200_sample_args* a, void* stream) {
    if (!a || a->B < 0 || a->V <= 0 || a->ld < a->V) return CCE_ERR_ARG;
    if (a->dtype != CCE_DT_F16 && a->dtype != CCE_DT_BF16 && a->dtype != CCE_DT_F32) return CCE_ERR_ARG;
    if (a->B == 0) return CCE_OK;
    if (!a->logits || !a->u || !a->tokens) return CCE_ERR_ARG;
    const int elem = a->dtype == CCE_DT_F32 ? 4 : 2;
    if (reinterpret_cast<uintptr_t>(a->logits) % elem) return CCE_ERR_ALIGN;
    DeviceInfo* dev;
    int rc = device_info(&dev);
    if (rc) return rc;
    // CTAs per row.  Few rows: short slices (1 x 256000 fp32: 22.5 us with 16384 positions, 24.6 with 32768);
    // many rows: fewer, longer ones, whose fixed cost is paid less often (512 x 152064: 803 us against 1360).
    int cluster = 1;
    const int longest = a->B >= 32 ? 32768 : 16384;
    if (a->V > (1 << 20)) return CCE_ERR_TOO_LARGE;  // the weights keep at least 42 bits
    while (cluster < SMP_MAX_CLUSTER && sample_slice(a->V, cluster) > longest) cluster *= 2;
    const int slice = sample_slice(a->V, cluster);
    const SampleLayout lay(cluster, slice, elem);
    if (lay.bytes > SMP_SMEM) return CCE_ERR_TOO_LARGE;
    if (a->B * cluster >= (1LL << 31)) return CCE_ERR_ARG;
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
    sp.slice = slice;
    int log2v = 0;
    while ((1LL << log2v) < a->V) ++log2v;
    sp.frac_bits = std::min(50, 62 - log2v);  // V weights of at most 1 << frac_bits stay below 2^63
    cudaStream_t st = reinterpret_cast<cudaStream_t>(stream);
    if (a->dtype == CCE_DT_F32) return launch_sample<float>(sp, cluster, lay.bytes, a->B, st);
    if (a->dtype == CCE_DT_BF16) return launch_sample<__nv_bfloat16>(sp, cluster, lay.bytes, a->B, st);
    return launch_sample<__half>(sp, cluster, lay.bytes, a->B, st);
}

}  // extern "C"
