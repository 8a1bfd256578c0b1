// The calls of a speculative step (the end of pam_cabi.cu): argument checks, the
// placement of the buffers, the launch with the library's retry loop, statistics.

namespace {

// Rows of `width` bytes that start `pitch` bytes apart.
struct StepRows {
    size_t count, width, pitch;
};

// One buffer of a call: what it must hold, which way it goes, the address the kernels use, and for rows that
// may be strided (count > 0) what of it is the call's.
struct StepArg {
    const char* name;
    const PamBuffer* buffer;
    size_t need;
    bool output, optional;
    bool onDevice;
    void* device;
    StepRows rows;
};

bool stepSizes(Context* c, StepArg* args, int n) {
    for (int i = 0; i < n; ++i)
        if (!(args[i].optional && !args[i].buffer->ptr) && !requireBuffer(c, *args[i].buffer, args[i].name, args[i].need)) return false;
    return true;
}

// Where every buffer lives.  Memory of another GPU is refused (the kernels would fault on it, or
// read it over the link without being asked to); a host buffer cannot be staged in a capture.
bool stepPlaces(Context* c, StepArg* args, int n, bool capturing) {
    for (int i = 0; i < n; ++i) {
        StepArg& a = args[i];
        a.onDevice = false;
        a.device = nullptr;
        if (!a.buffer->ptr) continue;
        cudaPointerAttributes at{};
        if (cudaPointerGetAttributes(&at, a.buffer->ptr) != cudaSuccess) { cudaGetLastError(); at.type = cudaMemoryTypeUnregistered; }
        a.onDevice = at.type == cudaMemoryTypeDevice || at.type == cudaMemoryTypeManaged;
        if (at.type == cudaMemoryTypeDevice && at.device != c->device) {
            c->fail(PAM_ERR_INVALID_CONFIGURATION, invalidConfiguration(std::string(a.name) + " buffer lives on GPU " + std::to_string(at.device) +
                                                                        ", the context on GPU " + std::to_string(c->device) + "."));
            return false;
        }
        if (a.onDevice) a.device = a.buffer->ptr;
        else if (capturing) {
            c->fail(PAM_ERR_INVALID_CONFIGURATION, invalidConfiguration(std::string(a.name) + " buffer is host memory: it cannot be staged while the stream is being captured."));
            return false;
        }
    }
    return true;
}

// What lies between strided rows belongs to somebody else (often another output of the same call), so that
// only the rows themselves are copied.
cudaError_t stepCopy(Context* c, const StepArg& a, void* to, const void* from, cudaMemcpyKind kind) {
    const StepRows& r = a.rows;
    if (r.count < 2 || r.width == r.pitch) return cudaMemcpyAsync(to, from, a.need, kind, c->stream);
    return cudaMemcpy2DAsync(to, r.pitch, from, r.pitch, r.width, r.count, kind, c->stream);
}

// Host buffers go through the arena.  A host output goes up as well: the kernels leave parts of
// it as they were.
cudaError_t stepStage(Context* c, StepArg* args, int n) {
    for (int i = 0; i < n; ++i) {
        StepArg& a = args[i];
        if (a.onDevice || !a.buffer->ptr || a.need == 0) continue;
        a.device = c->arena.take(a.need);
        if (!a.device) return cudaErrorMemoryAllocation;
        cudaError_t e = stepCopy(c, a, a.device, a.buffer->ptr, cudaMemcpyHostToDevice);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}
cudaError_t stepBack(Context* c, StepArg* args, int n) {
    for (int i = 0; i < n; ++i) {
        StepArg& a = args[i];
        if (a.onDevice || !a.buffer->ptr || !a.output || a.need == 0) continue;
        cudaError_t e = stepCopy(c, a, a.buffer->ptr, a.device, cudaMemcpyDeviceToHost);
        if (e != cudaSuccess) return e;
    }
    return cudaSuccess;
}

// Workspace of a call: the caller's, else the context's arena.  Returns false after c->fail.
bool stepWorkspace(Context* c, const PamBuffer& given, size_t need, bool capturing, const char* call) {
    if (need == 0) return true;
    if (given.ptr) {
        if (!requireBuffer(c, given, "workspace", need)) return false;
        if (reinterpret_cast<uintptr_t>(given.ptr) & 255) {
            c->fail(PAM_ERR_INVALID_CONFIGURATION, invalidConfiguration("workspace must start on a 256-byte boundary."));
            return false;
        }
        return true;
    }
    if (capturing) {
        c->fail(PAM_ERR_INVALID_CONFIGURATION, invalidConfiguration(std::string(call) + " needs a workspace of " + std::to_string(need) + " bytes while the stream is being captured."));
        return false;
    }
    return true;
}

// Stages, launches (with the retry loop, unless the stream is being captured) and copies host
// outputs back.  `launch(launches)` enqueues the kernels.
template <class F>
int32_t stepRun(Context* c, const char* name, StepArg* args, int n, bool capturing, F launch) {
    bool hostSide = false;
    for (int i = 0; i < n; ++i) hostSide = hostSide || (args[i].buffer->ptr && !args[i].onDevice);
    auto attempt = [&]() -> cudaError_t {
        cudaError_t e = stepStage(c, args, n);
        if (e != cudaSuccess) return e;
        int launches = 0;
        e = launch(&launches);
        c->launches += launches;
        return e == cudaSuccess ? stepBack(c, args, n) : e;
    };
    if (capturing) {
        cudaError_t e = attempt();
        if (e == cudaSuccess) return 0;
        cudaGetLastError();
        return c->fail(PAM_ERR_COMMAND_EXECUTION, commandExecutionFailed(cudaGetErrorString(e)));
    }
    const int32_t rc = withRetry(c, name, attempt);
    // the caller's host memory must be settled when the call returns
    if (hostSide && (c->async || rc != 0)) cudaStreamSynchronize(c->stream);
    return rc;
}

int32_t badStep(Context* c, const std::string& m) { return c->fail(PAM_ERR_INVALID_CONFIGURATION, invalidConfiguration(m)); }

// Bytes from the first element of a strided array of rows to its last; more than any buffer has where they pass
// 64 bits.
size_t rowSpan(int64_t rows, int64_t stride, int64_t width, int elem) {
    const unsigned __int128 bytes = (static_cast<unsigned __int128>(rows - 1) * stride + width) * elem;
    return bytes < kUnknownBytes ? static_cast<size_t>(bytes) : kUnknownBytes - 1;
}
StepRows stridedRows(int64_t rows, int64_t stride, int64_t width, int elem) {
    return {static_cast<size_t>(rows), static_cast<size_t>(width) * elem, static_cast<size_t>(stride) * elem};
}
bool rowStride(Context* c, int64_t given, int64_t width, const char* name, int64_t* out) {
    *out = given == 0 ? width : given;
    if (given != 0 && given < width) {
        badStep(c, std::string(name) + " must be 0 or at least the " + std::to_string(width) + " elements of a row.");
        return false;
    }
    if (*out > (int64_t(1) << 40)) {
        badStep(c, std::string(name) + " is out of range.");
        return false;
    }
    return true;
}

}  // namespace

extern "C" {

int32_t pamc_plan_step(void* ctx, const PamStepPlanRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    const PamStepPlanRequest& rq = *request;
    if (rq.batch_size <= 0 || rq.batch_size > 65536) return badStep(c, "batchSize must be in 1 ... 65536.");
    if (rq.block_size <= 0) return badStep(c, "blockSize must be positive.");
    if (rq.num_rows <= 0) return badStep(c, "numRows must be positive.");
    if (rq.max_new_tokens <= 0) return badStep(c, "maxNewTokens must be positive.");
    if (rq.num_lists <= 0 || rq.list_stride <= 0) return badStep(c, "numLists and listStride must be positive.");
    if (rq.tables.ptr && (rq.max_num_blocks <= 0 || rq.max_num_blocks > (1 << 26))) return badStep(c, "maxNumBlocks must be in 1 ... 2^26.");
    if (rq.max_new_tokens > (1 << 26)) return badStep(c, "maxNewTokens must be at most 2^26.");
    if (rq.parents.ptr && rq.max_new_tokens > pam::kMaxTreeNodes) return badStep(c, "a tree has at most " + std::to_string(pam::kMaxTreeNodes) + " nodes: maxNewTokens is too large.");
    if (rq.total_lengths.ptr && rq.total_lengths.ptr == rq.lengths.ptr)
        return badStep(c, "totalLengths must not lie over lengths (every block of the plan reads them).");
    if (rq.parents.ptr && rq.slots.ptr) return badStep(c, "the nodes of a tree have no slots before they are accepted (see pamc_accept_tree).");
    if (rq.masks.ptr && (rq.mask_words <= 0 || rq.mask_words > (1 << 20) || rq.max_new_tokens > 32ll * rq.mask_words))
        return badStep(c, "maskWords must hold one bit for each of maxNewTokens rows.");
    const size_t B = static_cast<size_t>(rq.batch_size), R = static_cast<size_t>(rq.num_rows);
    StepArg args[] = {
        {"blockLists", &rq.block_lists, static_cast<size_t>(rq.num_lists) * rq.list_stride * 4, false, false, false, nullptr},
        {"listIndex", &rq.list_index, B * 4, false, true, false, nullptr},
        {"lengths", &rq.lengths, B * 4, false, false, false, nullptr},
        {"newTokens", &rq.new_tokens, B * 4, false, false, false, nullptr},
        {"parents", &rq.parents, R * 4, false, true, false, nullptr},
        {"tables", &rq.tables, B * static_cast<size_t>(std::max(rq.max_num_blocks, 0)) * 4, true, true, false, nullptr},
        {"totalLengths", &rq.total_lengths, B * 4, true, true, false, nullptr},
        {"rowStarts", &rq.row_starts, (B + 1) * 4, true, true, false, nullptr},
        {"positions", &rq.positions, R * 4, true, true, false, nullptr},
        {"slots", &rq.slots, R * 8, true, true, false, nullptr},
        {"masks", &rq.masks, R * static_cast<size_t>(std::max(rq.mask_words, 0)) * 4, true, true, false, nullptr},
    };
    constexpr int n = sizeof(args) / sizeof(args[0]);
    if (!stepSizes(c, args, n)) return -1;
    if (c->device < 0) return noGpu(c);
    DeviceGuard dg(c->device);
    const bool capturing = isCapturing(c);
    if (!stepPlaces(c, args, n, capturing)) return -1;
    const double t0 = nowMs();
    if (!capturing) c->arena.reset(c->stream);
    const int32_t rc = stepRun(c, "planStep", args, n, capturing, [&](int* launches) -> cudaError_t {
        pam::StepPlanParams p{};
        p.lists = static_cast<const int32_t*>(args[0].device);
        p.listIndex = static_cast<const int32_t*>(args[1].device);
        p.lengths = static_cast<const int32_t*>(args[2].device);
        p.newTokens = static_cast<const int32_t*>(args[3].device);
        p.parents = static_cast<const int32_t*>(args[4].device);
        p.tables = static_cast<int32_t*>(args[5].device);
        p.totalLengths = static_cast<uint32_t*>(args[6].device);
        p.rowStarts = static_cast<int32_t*>(args[7].device);
        p.positions = static_cast<int32_t*>(args[8].device);
        p.slots = static_cast<int64_t*>(args[9].device);
        p.masks = static_cast<uint32_t*>(args[10].device);
        p.batch = rq.batch_size; p.numLists = rq.num_lists; p.listStride = rq.list_stride;
        p.maxNumBlocks = rq.max_num_blocks; p.numRows = rq.num_rows; p.maxNew = rq.max_new_tokens;
        p.maskWords = rq.mask_words; p.blockSize = rq.block_size;
        return pam::launchPlanStep(p, c->stream, launches);
    });
    if (rc != 0) return rc;
    c->stats = PamStats{PAM_OP_PLAN_STEP, rq.batch_size, rq.num_rows, rq.max_num_blocks, 0, 0, nowMs() - t0};
    c->clearError();
    return 0;
}

int32_t pamc_accept_tree(void* ctx, const PamAcceptRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    const PamAcceptRequest& rq = *request;
    if (rq.batch_size <= 0 || rq.batch_size > 65536) return badStep(c, "batchSize must be in 1 ... 65536.");
    if (rq.num_rows <= 0) return badStep(c, "numRows must be positive.");
    if (rq.max_tree <= 0 || rq.max_tree > pam::kMaxTreeNodes) return badStep(c, "maxTree must be in 1 ... " + std::to_string(pam::kMaxTreeNodes) + ".");
    if (rq.accepted_rows.ptr && rq.max_path <= 0) return badStep(c, "maxPath must be positive.");
    if (rq.slots.ptr && (!rq.block_tables.ptr || rq.max_num_blocks <= 0 || rq.block_size <= 0))
        return badStep(c, "slots need blockTables, maxNumBlocks and blockSize.");
    const size_t B = static_cast<size_t>(rq.batch_size), R = static_cast<size_t>(rq.num_rows);
    StepArg args[] = {
        {"rowStarts", &rq.row_starts, (B + 1) * 4, false, false, false, nullptr},
        {"parents", &rq.parents, R * 4, false, false, false, nullptr},
        {"draftTokens", &rq.draft_tokens, R * 4, false, false, false, nullptr},
        {"targetTokens", &rq.target_tokens, R * 4, false, false, false, nullptr},
        {"lengths", &rq.lengths, B * 4, false, false, false, nullptr},
        {"blockTables", &rq.block_tables, B * static_cast<size_t>(std::max(rq.max_num_blocks, 0)) * 4, false, true, false, nullptr},
        {"slots", &rq.slots, R * 8, true, true, false, nullptr},
        {"acceptedCounts", &rq.accepted_counts, B * 4, true, true, false, nullptr},
        {"acceptedRows", &rq.accepted_rows, B * static_cast<size_t>(std::max(rq.max_path, 0)) * 4, true, true, false, nullptr},
        {"nextTokens", &rq.next_tokens, B * 4, true, true, false, nullptr},
        {"newLengths", &rq.new_lengths, B * 4, true, true, false, nullptr},
    };
    constexpr int n = sizeof(args) / sizeof(args[0]);
    if (!stepSizes(c, args, n)) return -1;
    if (c->device < 0) return noGpu(c);
    DeviceGuard dg(c->device);
    const bool capturing = isCapturing(c);
    if (!stepPlaces(c, args, n, capturing)) return -1;
    const double t0 = nowMs();
    if (!capturing) c->arena.reset(c->stream);
    const int32_t rc = stepRun(c, "acceptTree", args, n, capturing, [&](int* launches) -> cudaError_t {
        pam::AcceptParams p{};
        p.rowStarts = static_cast<const int32_t*>(args[0].device);
        p.parents = static_cast<const int32_t*>(args[1].device);
        p.draft = static_cast<const int32_t*>(args[2].device);
        p.target = static_cast<const int32_t*>(args[3].device);
        p.lengths = static_cast<const int32_t*>(args[4].device);
        p.tables = static_cast<const int32_t*>(args[5].device);
        p.slots = static_cast<int64_t*>(args[6].device);
        p.counts = static_cast<int32_t*>(args[7].device);
        p.path = static_cast<int32_t*>(args[8].device);
        p.next = static_cast<int32_t*>(args[9].device);
        p.newLengths = static_cast<uint32_t*>(args[10].device);
        p.batch = rq.batch_size; p.numRows = rq.num_rows; p.maxTree = rq.max_tree; p.maxPath = rq.max_path;
        p.maxNumBlocks = rq.max_num_blocks; p.blockSize = std::max(rq.block_size, 1);
        return pam::launchAcceptTree(p, c->stream, launches);
    });
    if (rc != 0) return rc;
    c->stats = PamStats{PAM_OP_ACCEPT_TREE, rq.batch_size, rq.num_rows, rq.max_num_blocks, 0, 0, nowMs() - t0};
    c->clearError();
    return 0;
}

// Checks that the norm and its gradient share.
static bool normShape(Context* c, const PamLayerSpec& l, int32_t numRows, int32_t rotaryDim, float eps) {
    if (!validateLayer(c, l)) return false;
    if (l.head_dim > 256) { c->fail(PAM_ERR_UNSUPPORTED, "Unsupported paged attention path: headDim above 256."); return false; }
    if (numRows <= 0) { badStep(c, "numRows must be positive."); return false; }
    if (rotaryDim < 0 || rotaryDim > l.head_dim || rotaryDim % 2 != 0) { badStep(c, "rotaryDim must be even and in 0 ... headDim."); return false; }
    if (!(eps >= 0.f) || eps > 1e30f) { badStep(c, "epsilon must be non-negative and finite."); return false; }
    return true;
}

int32_t pamc_norm_rotate(void* ctx, const PamNormRotateRequest* request, void* cache) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    Cache* k = asCache(cache);
    std::lock_guard<std::mutex> g(c->mu);
    const PamNormRotateRequest& rq = *request;
    const PamLayerSpec& l = rq.layer;
    if (!normShape(c, l, rq.num_rows, rq.rotary_dim, rq.epsilon)) return -1;
    const bool fp8 = l.data_type == PAM_DTYPE_FP8;
    if (k) {
        if (k->bookkeeping) return c->fail(PAM_ERR_INVALID_STATE, "Invalid engine state: cache has no pools");
        if (k->dtype != l.data_type || k->headDim != l.head_dim || k->kvHeads != l.num_kv_heads || k->blockSize != l.block_size)
            return badStep(c, "the layer does not describe the cache (type, headDim, numKVHeads or blockSize).");
    } else if (fp8 && (rq.k_pool.ptr || rq.v_pool.ptr)) {
        return badStep(c, "FP8 append needs the cache handle that owns the scale buffers.");
    }
    PamBuffer kPool = k ? buf(k->kPool, k->poolBytes) : rq.k_pool, vPool = k ? buf(k->vPool, k->poolBytes) : rq.v_pool;
    const bool pages = kPool.ptr || vPool.ptr;
    if (!pages && !rq.k_out.ptr) return badStep(c, "the keys need kOut or pages to go to.");
    if (pages && (!kPool.ptr || !vPool.ptr)) return badStep(c, "pages need both kPool and vPool.");
    const int io = pam::ioBytes(l.data_type);
    const int64_t R = rq.num_rows, qWide = static_cast<int64_t>(l.num_heads) * l.head_dim, kWide = static_cast<int64_t>(l.num_kv_heads) * l.head_dim;
    int64_t qs, ks, vs, qo, ko;
    if (!rowStride(c, rq.q_stride, qWide, "qStride", &qs) || !rowStride(c, rq.k_stride, kWide, "kStride", &ks) ||
        !rowStride(c, rq.v_stride, kWide, "vStride", &vs) || !rowStride(c, rq.q_out_stride, qWide, "qOutStride", &qo) ||
        !rowStride(c, rq.k_out_stride, kWide, "kOutStride", &ko)) return -1;
    const size_t poolNeed = pages ? static_cast<size_t>(l.block_size) * kvBytesPerToken(l) : 0;
    static const PamBuffer none{nullptr, 0};
    StepArg args[] = {
        {"Q", &rq.q, rowSpan(R, qs, qWide, io), false, false, false, nullptr, stridedRows(R, qs, qWide, io)},
        {"K", &rq.k, rowSpan(R, ks, kWide, io), false, false, false, nullptr, stridedRows(R, ks, kWide, io)},
        {"V", pages ? &rq.v : &none, rowSpan(R, vs, kWide, io), false, !pages, false, nullptr, stridedRows(R, vs, kWide, io)},
        {"qWeight", &rq.q_weight, static_cast<size_t>(l.head_dim) * io, false, false, false, nullptr},
        {"kWeight", &rq.k_weight, static_cast<size_t>(l.head_dim) * io, false, false, false, nullptr},
        {"invFreq", &rq.inv_freq, static_cast<size_t>(rq.rotary_dim / 2) * 4, false, rq.rotary_dim == 0, false, nullptr},
        {"positions", &rq.positions, static_cast<size_t>(R) * 4, false, false, false, nullptr},
        {"qOut", &rq.q_out, rowSpan(R, qo, qWide, io), true, false, false, nullptr, stridedRows(R, qo, qWide, io)},
        {"kOut", &rq.k_out, rowSpan(R, ko, kWide, io), true, true, false, nullptr, stridedRows(R, ko, kWide, io)},
        {"K pool", &kPool, poolNeed, true, true, false, nullptr},
        {"V pool", &vPool, poolNeed, true, true, false, nullptr},
        {"slots", pages ? &rq.slots : &none, static_cast<size_t>(R) * 8, false, !pages, false, nullptr},
    };
    constexpr int n = sizeof(args) / sizeof(args[0]);
    if (!stepSizes(c, args, n)) return -1;
    if (c->device < 0) return noGpu(c);
    DeviceGuard dg(c->device);
    const bool capturing = isCapturing(c);
    if (!stepPlaces(c, args, n, capturing)) return -1;
    if (pages && (!args[9].onDevice || !args[10].onDevice)) return badStep(c, "KV pools must be device memory.");
    if (fp8 && pages && capturing)
        return c->fail(PAM_ERR_UNSUPPORTED, "Unsupported paged attention path: an FP8 append cannot be captured (its scales go by the call).");
    const double t0 = nowMs();
    if (!capturing) c->arena.reset(c->stream);
    const int32_t rc = stepRun(c, "normRotate", args, n, capturing, [&](int* launches) -> cudaError_t {
        pam::NormRotateParams p{};
        p.q = args[0].device; p.k = args[1].device; p.v = args[2].device;
        p.qWeight = args[3].device; p.kWeight = args[4].device;
        p.invFreq = static_cast<const float*>(args[5].device);
        p.positions = static_cast<const int32_t*>(args[6].device);
        p.qOut = args[7].device; p.kOut = args[8].device;
        p.slots = static_cast<const int64_t*>(args[11].device);
        p.qStride = qs; p.kStride = ks; p.vStride = vs; p.qOutStride = qo; p.kOutStride = ko;
        p.numRows = rq.num_rows; p.heads = l.num_heads; p.kvHeads = l.num_kv_heads; p.headDim = l.head_dim;
        p.blockSize = l.block_size; p.rotaryDim = rq.rotary_dim; p.interleaved = rq.interleaved != 0;
        p.ioType = fp8 ? PAM_DTYPE_F16 : l.data_type;
        p.eps = rq.epsilon;
        p.numSlots = static_cast<int64_t>(poolBlocksOf(kPool, vPool, l)) * l.block_size;
        if (!fp8 || !pages) {
            p.kPool = args[9].device; p.vPool = args[10].device;
            return pam::launchNormRotate(p, c->smCount, c->stream, launches);
        }
        // FP8: the scale of a block needs every new row of it first, so the rows go through the append
        // kernels, which take them back to back from a 16-byte boundary on: kOut and V where they are that,
        // else scratch that the same launch writes beside kOut (one launch, since the outputs may lie over the
        // inputs).  Skipped rows lose their slot.  32 + 8 + 8 heads of 128: 64 rows 12.7 us, 8192 rows 84 us, 32768
        // rows 234 us (float16 pages 4.8, 45, 138 us): three launches, and keys and values are read twice more.
        const size_t bytes = static_cast<size_t>(R) * kWide * io;
        const void *keys = p.kOut, *values = p.v;
        auto aligned = [](const void* a) { return (reinterpret_cast<uintptr_t>(a) & 15) == 0; };
        if (!p.kOut || ko != kWide || !aligned(keys)) keys = p.kPool = c->arena.take(bytes);
        if (vs != kWide || !aligned(values)) values = p.vPool = c->arena.take(bytes);
        p.slotsOut = static_cast<int64_t*>(c->arena.take(static_cast<size_t>(R) * 8));
        if (!keys || !values || !p.slotsOut) return cudaErrorMemoryAllocation;
        cudaError_t e = nextAbsmaxEpoch(k, c->stream);
        if (e == cudaSuccess) e = pam::launchNormRotate(p, c->smCount, c->stream, launches);
        if (e != cudaSuccess) return e;
        pam::SlotSource src;
        src.slots = p.slotsOut;
        src.numSlots = static_cast<int64_t>(k->maxBlocks) * k->blockSize;
        return pam::launchReshapeAndCacheFp8(keys, values, k->kPool, k->vPool, k->kScale, k->vScale, src, rq.num_rows, l.num_kv_heads,
                                             l.block_size, l.head_dim, k->amax, k->epoch, c->stream, launches);
    });
    if (rc != 0) return rc;
    c->stats = PamStats{PAM_OP_NORM_ROTATE, 1, rq.num_rows, 0, 0, 0, nowMs() - t0};
    c->clearError();
    return 0;
}

static void normBackwardSizes(const PamNormRotateBackwardRequest& rq, pam::NormRotateBackwardParams* p) {
    p->numRows = rq.num_rows; p->heads = rq.layer.num_heads; p->kvHeads = rq.layer.num_kv_heads; p->headDim = rq.layer.head_dim;
    p->blockSize = rq.layer.block_size; p->rotaryDim = rq.rotary_dim; p->interleaved = rq.interleaved != 0; p->ioType = rq.layer.data_type;
    p->eps = rq.epsilon;
    p->dV = rq.d_v.ptr;
    p->dQWeight = static_cast<float*>(rq.d_q_weight.ptr);
    p->dKWeight = static_cast<float*>(rq.d_k_weight.ptr);
}

int64_t pamc_norm_rotate_backward_workspace(void* ctx, const PamNormRotateBackwardRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    if (!normShape(c, request->layer, request->num_rows, request->rotary_dim, request->epsilon)) return -1;
    pam::NormRotateBackwardParams p{};
    normBackwardSizes(*request, &p);
    return static_cast<int64_t>(pam::normRotateBackwardWorkspaceBytes(p, c->smCount));
}

int32_t pamc_norm_rotate_backward(void* ctx, const PamNormRotateBackwardRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    const PamNormRotateBackwardRequest& rq = *request;
    const PamLayerSpec& l = rq.layer;
    if (!normShape(c, l, rq.num_rows, rq.rotary_dim, rq.epsilon)) return -1;
    if (l.data_type == PAM_DTYPE_FP8) return c->fail(PAM_ERR_UNSUPPORTED, "Unsupported paged attention path: backward over an FP8 cache.");
    const bool pages = rq.d_k_pool.ptr != nullptr;
    if (pages && rq.d_k_out.ptr) return badStep(c, "the keys' gradient comes from dKOut or from dKPool, not from both.");
    if (rq.d_v.ptr && !pages) return badStep(c, "dV is gathered from pages: it needs dKPool, dVPool and slots.");
    const int io = pam::ioBytes(l.data_type);
    const int64_t R = rq.num_rows, qWide = static_cast<int64_t>(l.num_heads) * l.head_dim, kWide = static_cast<int64_t>(l.num_kv_heads) * l.head_dim;
    int64_t qs, ks, dq, dk, dv;
    if (!rowStride(c, rq.q_stride, qWide, "qStride", &qs) || !rowStride(c, rq.k_stride, kWide, "kStride", &ks) ||
        !rowStride(c, rq.d_q_stride, qWide, "dQStride", &dq) || !rowStride(c, rq.d_k_stride, kWide, "dKStride", &dk) ||
        !rowStride(c, rq.d_v_stride, kWide, "dVStride", &dv)) return -1;
    const size_t poolNeed = static_cast<size_t>(l.block_size) * kvBytesPerToken(l), weight = static_cast<size_t>(l.head_dim) * io;
    static const PamBuffer none{nullptr, 0};
    const bool wantV = rq.d_v.ptr != nullptr;
    StepArg args[] = {
        {"Q", &rq.q, rowSpan(R, qs, qWide, io), false, false, false, nullptr, stridedRows(R, qs, qWide, io)},
        {"K", &rq.k, rowSpan(R, ks, kWide, io), false, false, false, nullptr, stridedRows(R, ks, kWide, io)},
        {"qWeight", &rq.q_weight, weight, false, false, false, nullptr},
        {"kWeight", &rq.k_weight, weight, false, false, false, nullptr},
        {"invFreq", &rq.inv_freq, static_cast<size_t>(rq.rotary_dim / 2) * 4, false, rq.rotary_dim == 0, false, nullptr},
        {"positions", &rq.positions, static_cast<size_t>(R) * 4, false, false, false, nullptr},
        {"dQOut", &rq.d_q_out, static_cast<size_t>(R) * qWide * io, false, false, false, nullptr},
        {"dKOut", &rq.d_k_out, static_cast<size_t>(R) * kWide * io, false, pages, false, nullptr},
        {"dK pool", &rq.d_k_pool, poolNeed, false, true, false, nullptr},
        {"dV pool", wantV ? &rq.d_v_pool : &none, poolNeed, false, !wantV, false, nullptr},
        {"slots", pages ? &rq.slots : &none, static_cast<size_t>(R) * 8, false, !pages, false, nullptr},
        {"dQ", &rq.d_q, rowSpan(R, dq, qWide, io), true, false, false, nullptr, stridedRows(R, dq, qWide, io)},
        {"dK", &rq.d_k, rowSpan(R, dk, kWide, io), true, false, false, nullptr, stridedRows(R, dk, kWide, io)},
        {"dV", &rq.d_v, rowSpan(R, dv, kWide, io), true, true, false, nullptr, stridedRows(R, dv, kWide, io)},
        {"dQWeight", &rq.d_q_weight, static_cast<size_t>(l.head_dim) * 4, true, true, false, nullptr},
        {"dKWeight", &rq.d_k_weight, static_cast<size_t>(l.head_dim) * 4, true, true, false, nullptr},
        {"workspace", &rq.workspace, 0, true, true, false, nullptr},
    };
    constexpr int n = sizeof(args) / sizeof(args[0]);
    if (!stepSizes(c, args, n)) return -1;
    pam::NormRotateBackwardParams p{};
    normBackwardSizes(rq, &p);
    const size_t need = pam::normRotateBackwardWorkspaceBytes(p, c->smCount);
    if (!stepWorkspace(c, rq.workspace, need, false, "normRotateBackward")) return -1;
    if (c->device < 0) return noGpu(c);
    DeviceGuard dg(c->device);
    const bool capturing = isCapturing(c);
    if (!stepPlaces(c, args, n, capturing)) return -1;
    if ((pages && !args[8].onDevice) || (wantV && !args[9].onDevice)) return badStep(c, "the gradient pools must be device memory.");
    if (rq.workspace.ptr && !args[16].onDevice) return badStep(c, "workspace must be device memory.");
    if (!stepWorkspace(c, rq.workspace, need, capturing, "normRotateBackward")) return -1;
    const double t0 = nowMs();
    if (!capturing) c->arena.reset(c->stream);
    const int32_t rc = stepRun(c, "normRotateBackward", args, n, capturing, [&](int* launches) -> cudaError_t {
        p.q = args[0].device; p.k = args[1].device; p.qWeight = args[2].device; p.kWeight = args[3].device;
        p.invFreq = static_cast<const float*>(args[4].device);
        p.positions = static_cast<const int32_t*>(args[5].device);
        p.dQOut = args[6].device; p.dKOut = args[7].device; p.dKPool = args[8].device; p.dVPool = args[9].device;
        p.slots = static_cast<const int64_t*>(args[10].device);
        p.dQ = args[11].device; p.dK = args[12].device; p.dV = args[13].device;
        p.dQWeight = static_cast<float*>(args[14].device);
        p.dKWeight = static_cast<float*>(args[15].device);
        p.qStride = qs; p.kStride = ks; p.dQStride = dq; p.dKStride = dk; p.dVStride = dv;
        if (pages) p.numSlots = static_cast<int64_t>(poolBlocksOf(rq.d_k_pool, wantV ? rq.d_v_pool : rq.d_k_pool, l)) * l.block_size;
        p.partials = nullptr;
        if (need) {
            p.partials = static_cast<float*>(rq.workspace.ptr ? rq.workspace.ptr : c->arena.take(need));
            if (!p.partials) return cudaErrorMemoryAllocation;
        }
        return pam::launchNormRotateBackward(p, c->smCount, c->stream, launches);
    });
    if (rc != 0) return rc;
    c->stats = PamStats{PAM_OP_NORM_ROTATE_BACKWARD, 1, rq.num_rows, 0, static_cast<int64_t>(need), 0, nowMs() - t0};
    c->clearError();
    return 0;
}

// Sizes of a tree attention request, checked; fills what does not need the buffers' places.
static bool treeShape(Context* c, const PamTreeAttentionRequest& rq, pam::TreeParams* p) {
    const PamLayerSpec& l = rq.layer;
    if (!validateLayer(c, l)) return false;
    auto bad = [&](const std::string& m) { badStep(c, m); return false; };
    if (l.head_dim > 256) { c->fail(PAM_ERR_UNSUPPORTED, "Unsupported paged attention path: headDim above 256."); return false; }
    if (rq.batch_size <= 0 || rq.batch_size > pam::kTreeMaxBatch) return bad("batchSize must be in 1 ... " + std::to_string(pam::kTreeMaxBatch) + ".");
    if (static_cast<int64_t>(l.num_kv_heads) * l.block_size > INT32_MAX) return bad("numKVHeads times blockSize is out of range.");
    if (rq.max_num_blocks <= 0) return bad("maxNumBlocks must be positive.");
    if (rq.num_rows <= 0) return bad("numRows must be positive.");
    if (rq.max_new_tokens <= 0) return bad("maxNewTokens must be positive.");
    if (rq.masks.ptr && (rq.mask_words <= 0 || rq.mask_words > (1 << 20) || rq.max_new_tokens > 32ll * rq.mask_words))
        return bad("maskWords must hold one bit for each of maxNewTokens rows.");
    const int window = l.window_size > 0 ? l.window_size : c->defaultWindow;
    if (window > 0 && rq.masks.ptr && !rq.positions.ptr) return bad("a window over a tree needs positions.");
    const int64_t qWide = static_cast<int64_t>(l.num_heads) * l.head_dim, kWide = static_cast<int64_t>(l.num_kv_heads) * l.head_dim;
    if (!rowStride(c, rq.q_stride, qWide, "qStride", &p->qStride) || !rowStride(c, rq.k_stride, kWide, "kStride", &p->kStride) ||
        !rowStride(c, rq.v_stride, kWide, "vStride", &p->vStride)) return false;
    p->q = rq.q.ptr; p->kNew = rq.k.ptr; p->vNew = rq.v.ptr; p->kPool = rq.k_pool.ptr; p->vPool = rq.v_pool.ptr; p->out = rq.output.ptr;
    p->batch = rq.batch_size; p->heads = l.num_heads; p->kvHeads = l.num_kv_heads; p->headDim = l.head_dim; p->blockSize = l.block_size;
    p->maxNumBlocks = rq.max_num_blocks; p->numRows = rq.num_rows; p->maxNew = std::min(rq.max_new_tokens, rq.num_rows);
    p->maskWords = rq.mask_words; p->window = window; p->dtype = l.data_type; p->exactWeights = c->exactWeights;
    // (tiles are counted in 32 bits up to a block's begin plus its share, of which there is at least one for each SM)
    if (pam::treeTileBound(*p) >= INT32_MAX - INT32_MAX / std::max(c->smCount, 1) - 1)
        return bad("batchSize, maxNumBlocks and maxNewTokens span more work than one call takes; split the batch.");
    return true;
}

int64_t pamc_tree_attention_workspace(void* ctx, const PamTreeAttentionRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    pam::TreeParams p{};
    if (!treeShape(c, *request, &p)) return -1;
    return static_cast<int64_t>(pam::treeWorkspaceBytes(p, c->smCount));
}

int32_t pamc_tree_attention(void* ctx, const PamTreeAttentionRequest* request) {
    if (!ctx || !request) return -1;
    Context* c = asCtx(ctx);
    std::lock_guard<std::mutex> g(c->mu);
    const PamTreeAttentionRequest& rq = *request;
    const PamLayerSpec& l = rq.layer;
    pam::TreeParams p{};
    if (!treeShape(c, rq, &p)) return -1;
    const bool fp8 = l.data_type == PAM_DTYPE_FP8;
    if (fp8 && (!rq.k_scale.ptr || !rq.v_scale.ptr)) return badStep(c, "FP8 attention needs kScaleBuffer and vScaleBuffer.");
    const int io = pam::ioBytes(l.data_type);
    const int64_t R = rq.num_rows, qWide = static_cast<int64_t>(l.num_heads) * l.head_dim, kWide = static_cast<int64_t>(l.num_kv_heads) * l.head_dim;
    const size_t B = static_cast<size_t>(rq.batch_size), poolNeed = static_cast<size_t>(l.block_size) * kvBytesPerToken(l);
    const size_t outBytes = static_cast<size_t>(R) * qWide * io, scaleNeed = static_cast<size_t>(l.num_kv_heads) * 2;
    static const PamBuffer none{nullptr, 0};
    StepArg args[] = {
        {"Q", &rq.q, rowSpan(R, p.qStride, qWide, io), false, false, false, nullptr, stridedRows(R, p.qStride, qWide, io)},
        {"K", &rq.k, rowSpan(R, p.kStride, kWide, io), false, false, false, nullptr, stridedRows(R, p.kStride, kWide, io)},
        {"V", &rq.v, rowSpan(R, p.vStride, kWide, io), false, false, false, nullptr, stridedRows(R, p.vStride, kWide, io)},
        {"K pool", &rq.k_pool, poolNeed, false, false, false, nullptr},
        {"V pool", &rq.v_pool, poolNeed, false, false, false, nullptr},
        {"blockTables", &rq.block_tables, B * rq.max_num_blocks * 4, false, false, false, nullptr},
        {"cacheLengths", &rq.cache_lengths, B * 4, false, false, false, nullptr},
        {"rowStarts", &rq.row_starts, (B + 1) * 4, false, false, false, nullptr},
        {"masks", &rq.masks, static_cast<size_t>(R) * std::max(rq.mask_words, 0) * 4, false, true, false, nullptr},
        {"positions", &rq.positions, static_cast<size_t>(R) * 4, false, true, false, nullptr},
        {"output", &rq.output, outBytes, true, false, false, nullptr},
        {"K scale", fp8 ? &rq.k_scale : &none, scaleNeed, false, !fp8, false, nullptr},
        {"V scale", fp8 ? &rq.v_scale : &none, scaleNeed, false, !fp8, false, nullptr},
        {"workspace", &rq.workspace, 0, true, true, false, nullptr},
    };
    constexpr int n = sizeof(args) / sizeof(args[0]);
    if (!stepSizes(c, args, n)) return -1;
    if (rq.workspace.ptr && !stepWorkspace(c, rq.workspace, pam::treeWorkspaceBytes(p, c->smCount), false, "treeAttention")) return -1;
    if (c->device < 0) return noGpu(c);
    DeviceGuard dg(c->device);
    const bool capturing = isCapturing(c);
    if (!stepPlaces(c, args, n, capturing)) return -1;
    if (!args[3].onDevice || !args[4].onDevice || (fp8 && (!args[11].onDevice || !args[12].onDevice)))
        return badStep(c, "KV pools must be device memory.");
    if (rq.workspace.ptr && !args[13].onDevice) return badStep(c, "workspace must be device memory.");
    if (!rq.workspace.ptr && capturing && !stepWorkspace(c, rq.workspace, pam::treeWorkspaceBytes(p, c->smCount), true, "treeAttention")) return -1;
    p.poolBlocks = poolBlocksOf(rq.k_pool, rq.v_pool, l);
    if (fp8)
        for (const PamBuffer* s : {&rq.k_scale, &rq.v_scale})
            if (s->bytes != kUnknownBytes) p.poolBlocks = static_cast<int>(std::min<size_t>(static_cast<size_t>(p.poolBlocks), s->bytes / scaleNeed));
    const double t0 = nowMs();
    if (!capturing) c->arena.reset(c->stream);
    p.errFlag = c->devErr;
    p.waitCycles = c->waitLimitCycles;
    const size_t need = pam::treeWorkspaceBytes(p, c->smCount);
    int32_t rc = stepRun(c, "treeAttention", args, n, capturing, [&](int* launches) -> cudaError_t {
        p.q = args[0].device; p.kNew = args[1].device; p.vNew = args[2].device; p.kPool = args[3].device; p.vPool = args[4].device;
        p.tables = static_cast<const int32_t*>(args[5].device);
        p.lens = static_cast<const uint32_t*>(args[6].device);
        p.rowStarts = static_cast<const int32_t*>(args[7].device);
        p.masks = static_cast<const uint32_t*>(args[8].device);
        p.positions = static_cast<const int32_t*>(args[9].device);
        p.out = args[10].device;
        p.kScale = args[11].device; p.vScale = args[12].device;
        p.workspace = static_cast<float*>(rq.workspace.ptr ? rq.workspace.ptr : c->arena.take(need));
        if (!p.workspace) return cudaErrorMemoryAllocation;
        bool bounded = false;
        cudaError_t e = beforeBounded(c, capturing);
        if (e == cudaSuccess) e = pam::launchTreeAttention(p, c->smCount, c->stream, launches, &bounded);
        return e == cudaSuccess && bounded ? afterBounded(c, capturing) : e;
    });
    if (rc != 0) {
        if (!c->graceful || capturing) return rc;
        // as a failed decode: zeros instead of an error
        if (args[10].onDevice) cudaMemsetAsync(rq.output.ptr, 0, outBytes, c->stream);
        else std::memset(rq.output.ptr, 0, outBytes);
    }
    c->stats = PamStats{PAM_OP_TREE_ATTENTION, rq.batch_size, rq.num_rows, rq.max_num_blocks, static_cast<int64_t>(need), 0, nowMs() - t0};
    c->clearError();
    return 0;
}

}  // extern "C"
