// fxr_q8_api.cuh — extern "C" entry points of the 8-bit spatial cache (include/fxr.h): argument
// checks and launches. Part of fxr_capi.cu's translation unit, whose helpers it uses.
#pragma once

namespace {

int32_t check_q8_cache(const fxr_frame_desc* d, const fxr_q8_cache* c, int32_t rows, const char* what) {
    if (!c) return fail(FXR_ERR_INVALID, "%s: null cache", what);
    if (c->format != FXR_Q8_INT8 && c->format != FXR_Q8_E4M3)
        return fail(FXR_ERR_INVALID, "%s: format %d is neither FXR_Q8_INT8 nor FXR_Q8_E4M3", what, c->format);
    if (c->n_rows < rows) return fail(FXR_ERR_INVALID, "%s: %d rows, %d needed", what, c->n_rows, rows);
    const int64_t C = (int64_t)d->n_heads * d->head_dim;
    if (c->ld < C || (c->ld % 16)) return fail(FXR_ERR_INVALID, "%s: ld must be a multiple of 16, >= %lld", what, (long long)C);
    if (c->ld_scale < c->n_rows || (c->ld_scale % 8))
        return fail(FXR_ERR_INVALID, "%s: ld_scale must be a multiple of 8, >= n_rows", what);
    if (c->n_rows == 0) return FXR_OK;
    if (!c->k || !c->v || !c->k_scale || !c->v_scale) return fail(FXR_ERR_INVALID, "%s: null pointer", what);
    if (!aligned16(c->k) || !aligned16(c->v) || !aligned16(c->k_scale) || !aligned16(c->v_scale))
        return fail(FXR_ERR_INVALID, "%s: codes and scales must be 16-byte aligned", what);
    return FXR_OK;
}

fxr::q8::Cache q8_arg(const fxr_q8_cache* c) {
    return fxr::q8::Cache{static_cast<uint8_t*>(c->k), static_cast<uint8_t*>(c->v), c->k_scale, c->v_scale, c->ld, c->ld_scale};
}

// f(T, F) for the frame's type and the cache's format.
template <typename Fn>
int32_t q8_dispatch(int32_t dtype, int32_t format, Fn&& f) {
    using I8 = std::integral_constant<int, fxr::q8::kInt8>;
    using E4 = std::integral_constant<int, fxr::q8::kE4m3>;
    if (dtype == FXR_BF16) return format == FXR_Q8_INT8 ? f(__nv_bfloat16{}, I8{}) : f(__nv_bfloat16{}, E4{});
    return format == FXR_Q8_INT8 ? f(__half{}, I8{}) : f(__half{}, E4{});
}

int64_t q8_save_bytes(const fxr_frame_desc* d) {
    return (int64_t)align_up((size_t)d->n_heads * ((size_t)d->head_dim * 2 + 4), 16);
}

// Revolutions per position of each rotary pair. 64 powers cost as much as a launch, so a thread keeps
// the table of the last axes and theta it was asked for.
void fill_turns(const fxr_frame_desc* d, fxr::q8::WriteArgs* a) {
    struct Table {
        int32_t n_axes = -1;
        int32_t dims[4];
        float theta;
        float2 turns[fxr::kPairs];
        int8_t axis[fxr::kPairs];
    };
    static thread_local Table t;
    bool same = t.n_axes == d->rope_n_axes && t.theta == d->rope_theta;
    for (int x = 0; same && x < d->rope_n_axes; ++x) same = t.dims[x] == d->rope_axes_dim[x];
    if (!same) {
        std::memset(t.turns, 0, sizeof(t.turns));
        std::memset(t.axis, 0, sizeof(t.axis));
        for (int x = 0, j = 0; x < d->rope_n_axes; ++x) {
            t.dims[x] = d->rope_axes_dim[x];
            for (int jj = 0; jj < d->rope_axes_dim[x] / 2; ++jj, ++j) {
                const double w = std::pow((double)d->rope_theta, -2.0 * jj / d->rope_axes_dim[x]) / 6.283185307179586;
                const float hi = (float)w;
                t.turns[j] = make_float2(hi, (float)(w - (double)hi));
                t.axis[j] = (int8_t)x;
            }
        }
        t.n_axes = d->rope_n_axes;
        t.theta = d->rope_theta;
    }
    std::memcpy(a->turns, t.turns, sizeof(t.turns));
    std::memcpy(a->axis, t.axis, sizeof(t.axis));
}

int32_t launch_q8_write(const fxr_frame_desc* d, const fxr_q8_cache* cache, fxr::q8::WriteArgs a, bool raw, int64_t max_rows,
                        cudaStream_t s) {
    NvtxRange nvtx_("fxr:q8_write");
    a.c = q8_arg(cache);
    a.n_tokens = d->n_tokens;
    a.n_heads = d->n_heads;
    a.n_axes = d->rope_n_axes;
    a.eps = d->eps;
    a.ld_save = q8_save_bytes(d);
    fill_turns(d, &a);
    const int64_t units = max_rows * ((d->n_heads + fxr::q8::kVecHeads - 1) / fxr::q8::kVecHeads);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((units + fxr::q8::kWriteWarps - 1) / fxr::q8::kWriteWarps,
                                                                (int64_t)sm_count() * 2));
    return q8_dispatch(d->dtype, cache->format, [&](auto t, auto f) -> int32_t {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        const cudaError_t e = raw ? launch_pdl(fxr::q8::q8_write_kernel<T, F, true>, dim3(grid), dim3(fxr::q8::kWriteThreads), 0, s, a)
                                  : launch_pdl(fxr::q8::q8_write_kernel<T, F, false>, dim3(grid), dim3(fxr::q8::kWriteThreads), 0, s, a);
        return cuda_status(e, "q8_write_kernel launch");
    });
}

// The kernel for few rows serves streams of up to 32 rows: with more, a second group of rows reads the
// cache again (24 heads over 4608 keys: 32 rows 27 us, and 34 with the other kernel; 64 rows 35.5, and
// 35; 100 rows of 8 heads 30, and 27).
constexpr int32_t kQ8FewRows = fxr::attn8::kMaxRowsPerStream;

// A call without groups and prefix turns its caches into 16 bits and runs the 16-bit kernel on them, where
// a stream has at least this many 256-row units and the SMs this many steps (256 rows x 128 keys) each: a
// step takes 2.0 us there, and 2.6 where converters work along; the rows cost 3.4 ns each (24 heads) and a
// launch. 24 heads: 2304 rows over 4608 keys 142 us, and 156 with the converters; 4224 over 16896 905, and
// 1010; the frame of 16896 tokens 586 to 662, and 826. Below: 1536 rows over 4608 keys 94.5, and 93; 6 heads with 2304
// rows 67, and 60. A call without a bound is taken to run a quarter of the tokens.
constexpr int32_t kQ8WideUnits = 8, kQ8WideSteps = 32;

// Workspace of the attention: arrivals (zero before and after a call), then partial results, then the
// visible steps of the kernel for many rows.
struct Q8Work {
    int32_t* cnt;
    float* part;
    fxr::attn8::CutUnit* cuts;
    int32_t* steps;
    uint16_t* list;
    uint32_t* groups;
    int32_t rows;         // bound of a stream's rows
    bool bounded;         // by the caller
    bool few;             // the kernel for few rows
    int32_t tiles;        // it takes groups of 8 * tiles rows
    int64_t line;         // bound of its work line
    int32_t slots;        // its partial results: one per column and CTA boundary
    int32_t units;        // 256-row units of a stream, key tiles: the kernel for many
    int32_t n_pre, n_own;
    bool wide;            // without groups: the 16-bit kernel, in the same place of the workspace
    char* wide_k;
    char* wide_v;
    char* split;
    int32_t* wide_rows;
    size_t zero_bytes;    // from the start: what has to be zero before a launch, and is after it
    size_t total;
};

Q8Work carve_q8(const fxr_frame_desc* d, int32_t n_streams, int32_t n_prefix, int32_t max_rows, void* ws) {
    Q8Work w{};
    w.bounded = max_rows > 0;
    w.rows = w.bounded ? std::min(max_rows, d->n_tokens) : d->n_tokens;
    w.few = w.rows <= kQ8FewRows;
    const int64_t S = std::min<int32_t>(n_streams, FXR_MAX_BATCH), R = w.rows;
    size_t off = 0;
    char* b = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* p = b ? b + off : nullptr;
        off = align_up(off + bytes, 256);
        return p;
    };
    // one place and size for the arrivals, whichever kernel a call takes and however many heads it has (up
    // to 256): calls of other bounds and head counts may share a workspace, and none writes anything else
    // where another has its arrivals
    const size_t ctas = (size_t)sm_count(), per_head = (size_t)FXR_MAX_BATCH * fxr::attn8::kGroupsPerStream * sizeof(int32_t);
    w.cnt = reinterpret_cast<int32_t*>(take((size_t)std::max(d->n_heads, 256) * per_head));
    w.zero_bytes = align_up((size_t)d->n_heads * per_head, 16);
    const size_t body = off;
    if (w.few) {
        // groups as large as a stream's rows need; the packed rows of a prefix fill groups of 16 at most
        // otherwise (8 streams, 4608 + 2304 keys, 24 heads, in a graph: 6 rows each 75.9 us, and 81.6 in groups
        // of 32 with 8 warps; 10 rows 81.3, and 109; 15 rows 102.6, and 117; 3 streams of 15 rows 45.7, and 74.6)
        const int64_t packed = n_prefix > 0 ? std::max(R, std::min<int64_t>(S * R, 16)) : R;
        w.tiles = packed <= 8 ? 1 : packed <= 16 ? 2 : 4;
        const int64_t tile = 8 * w.tiles;
        const int64_t groups = (n_prefix > 0 ? (S * R + tile - 1) / tile : 0) + S * ((R + tile - 1) / tile);
        w.slots = (int32_t)std::min<int64_t>(INT32_MAX, sm_count() + groups * d->n_heads);
        w.line = groups * d->n_heads * ((std::max(n_prefix, d->n_tokens) + fxr::attn8::kUnitKeys - 1) / fxr::attn8::kUnitKeys);
        w.part = reinterpret_cast<float*>(take((size_t)w.slots * fxr::attn8::kRowsSlotFloats * sizeof(float)));
    } else {
        w.units = (w.rows + fxr::attn8::kUnitRows - 1) / fxr::attn8::kUnitRows;
        w.n_pre = (n_prefix + fxr::attn8::kBN - 1) / fxr::attn8::kBN;
        w.n_own = (d->n_tokens + fxr::attn8::kBN - 1) / fxr::attn8::kBN;
        w.part = reinterpret_cast<float*>(take(ctas * fxr::attn8::kPartSlots * fxr::attn8::kPartFloats * sizeof(float)));
        w.cuts = reinterpret_cast<fxr::attn8::CutUnit*>(take(ctas * sizeof(fxr::attn8::CutUnit)));
        w.steps = reinterpret_cast<int32_t*>(take((size_t)(S * w.units) * sizeof(int32_t)));
        w.list = reinterpret_cast<uint16_t*>(take((size_t)(S * w.units) * (size_t)(w.n_pre + w.n_own) * sizeof(uint16_t)));
        w.groups = reinterpret_cast<uint32_t*>(take((size_t)(w.n_pre + S * w.n_own) * fxr::attn8::kBN * sizeof(uint32_t)));
        // room for it wherever a bound of w.rows takes it, so that the size is one of the bound alone
        auto many = [&](int32_t rows) {
            const int64_t units = (rows + fxr::attn8::kUnitRows - 1) / fxr::attn8::kUnitRows;
            return n_prefix == 0 && units >= kQ8WideUnits && S * units * d->n_heads * w.n_own >= (int64_t)kQ8WideSteps * sm_count();
        };
        w.wide = many(w.bounded ? w.rows : w.rows / 4);
        if (many(w.rows)) {
            const size_t end = off, bytes = (size_t)S * (size_t)d->n_tokens * (size_t)d->n_heads * (size_t)d->head_dim * 2;
            off = body;
            w.wide_rows = reinterpret_cast<int32_t*>(take(FXR_MAX_BATCH * sizeof(int32_t)));
            w.split = take(split_bytes(kSplitSlotsPerSm * sm_count()));
            w.wide_k = take(bytes);
            w.wide_v = take(bytes);
            off = std::max(off, end);
        }
    }
    w.total = off;
    return w;
}

// 2-D map over rows of 8-bit codes: boxes of `box_rows` rows x 128 bytes (a head), 128-byte swizzle.
int32_t make_code_tmap(CUtensorMap* map, const void* ptr, int64_t cols, int64_t rows, int64_t ld, uint32_t box_rows) {
    EncodeTiledFn fn = encode_fn();
    if (!fn) return fail(FXR_ERR_CUDA, "cuTensorMapEncodeTiled entry point unavailable");
    const cuuint64_t dims[2] = {(cuuint64_t)cols, (cuuint64_t)rows};
    const cuuint64_t strides[1] = {(cuuint64_t)ld};
    const cuuint32_t box[2] = {(cuuint32_t)fxr::attn8::kD, box_rows};
    const cuuint32_t estr[2] = {1, 1};
    const CUresult r = fn(map, CU_TENSOR_MAP_DATA_TYPE_UINT8, 2, const_cast<void*>(ptr), dims, strides, box, estr,
                          CU_TENSOR_MAP_INTERLEAVE_NONE, CU_TENSOR_MAP_SWIZZLE_128B, CU_TENSOR_MAP_L2_PROMOTION_L2_256B,
                          CU_TENSOR_MAP_FLOAT_OOB_FILL_NONE);
    if (r != CUDA_SUCCESS) return fail(FXR_ERR_INVALID, "cuTensorMapEncodeTiled failed (%d)", (int)r);
    return FXR_OK;
}

template <typename T, int F, int NQ>
int32_t launch_q8_rows(const fxr_frame_desc* d, const fxr::attn8::Params& p, cudaStream_t s) {
    static bool configured[kMaxDevices] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kMaxDevices) return fail(FXR_ERR_CUDA, "device %d", dev);
    if (!configured[dev]) {
        const cudaError_t e = cudaFuncSetAttribute(fxr::attn8::rows_kernel<T, F, NQ>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                                   (int)fxr::attn8::RowsShape<NQ>::smem);
        if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(rows_kernel)");
        configured[dev] = true;
    }
    const int64_t C = (int64_t)d->n_heads * d->head_dim;
    fxr::attn8::RowsMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    int32_t rc;
    for (int32_t b = 0; b < p.n_streams; ++b) {
        if ((rc = make_code_tmap(&maps.k[b], p.s[b].c.k, C, p.n_tokens, p.s[b].c.ld, fxr::attn8::kBlk)) != FXR_OK) return rc;
        if ((rc = make_code_tmap(&maps.v[b], p.s[b].c.v, C, p.n_tokens, p.s[b].c.ld, fxr::attn8::kBlk)) != FXR_OK) return rc;
    }
    if (p.n_prefix > 0) {
        if ((rc = make_code_tmap(&maps.pk, p.prefix.k, C, p.n_prefix, p.prefix.ld, fxr::attn8::kBlk)) != FXR_OK) return rc;
        if ((rc = make_code_tmap(&maps.pv, p.prefix.v, C, p.n_prefix, p.prefix.ld, fxr::attn8::kBlk)) != FXR_OK) return rc;
    }
    return cuda_status(launch_pdl(fxr::attn8::rows_kernel<T, F, NQ>, dim3(sm_count()), dim3(fxr::attn8::RowsShape<NQ>::threads),
                                  fxr::attn8::RowsShape<NQ>::smem, s, maps, p),
                       "rows_kernel launch");
}

template <typename T, int F>
int32_t launch_q8_tiles(const fxr_frame_desc* d, const fxr::attn8::Params& p, const Q8Work& w, cudaStream_t s) {
    static bool configured[kMaxDevices] = {false};
    int dev = 0;
    cudaGetDevice(&dev);
    if (dev < 0 || dev >= kMaxDevices) return fail(FXR_ERR_CUDA, "device %d", dev);
    if (!configured[dev]) {
        cudaError_t e = cudaFuncSetAttribute(fxr::attn8::tile_kernel<T, F>, cudaFuncAttributeMaxDynamicSharedMemorySize,
                                             (int)fxr::attn8::kTileSmem);
        cudaFuncAttributes fa{};
        if (e == cudaSuccess) e = cudaFuncGetAttributes(&fa, fxr::attn8::tile_kernel<T, F>);
        if (e != cudaSuccess) return cuda_status(e, "cudaFuncSetAttribute(tile_kernel)");
        // the warpgroups redistribute the launch's registers: it must have been compiled to hold them
        if ((uint32_t)fa.numRegs * fxr::attn8::kTileThreads < fxr::attn8::kTileRegPool)
            return fail(FXR_ERR_UNSUPPORTED, "tile_kernel compiled to %d registers", fa.numRegs);
        configured[dev] = true;
    }
    const int64_t C = (int64_t)d->n_heads * d->head_dim;
    fxr::attn8::TileMaps maps;
    std::memset(&maps, 0, sizeof(maps));
    int32_t rc;
    bool groups = p.pg != nullptr && p.n_prefix > 0;
    for (int32_t b = 0; b < p.n_streams; ++b) {
        if ((rc = make_tmap(&maps.q[b], p.s[b].qc, d->dtype, C, p.max_rows, p.s[b].ld_qc)) != FXR_OK) return rc;
        if ((rc = make_code_tmap(&maps.k[b], p.s[b].c.k, C, p.n_tokens, p.s[b].c.ld, fxr::attn8::kBN)) != FXR_OK) return rc;
        if ((rc = make_code_tmap(&maps.v[b], p.s[b].c.v, C, p.n_tokens, p.s[b].c.ld, fxr::attn8::kBN)) != FXR_OK) return rc;
        groups = groups || p.s[b].qg != nullptr || p.s[b].kg != nullptr;
    }
    if (p.n_prefix > 0) {
        if ((rc = make_code_tmap(&maps.pk, p.prefix.k, C, p.n_prefix, p.prefix.ld, fxr::attn8::kBN)) != FXR_OK) return rc;
        if ((rc = make_code_tmap(&maps.pv, p.prefix.v, C, p.n_prefix, p.prefix.ld, fxr::attn8::kBN)) != FXR_OK) return rc;
    }
    fxr::attn8::TileParams a{};
    a.p = p;
    a.n_pre = w.n_pre;
    a.n_own = w.n_own;
    a.units_cap = w.units;
    a.part = w.part;
    a.cuts = w.cuts;
    // a bound that the caller gave is taken to be tight: where its units would run whole, they do
    const int64_t units = (int64_t)w.units * d->n_heads * p.n_streams;
    const fxr::attn8::TileSchedule sc = fxr::attn8::tile_schedule((int32_t)(units * (w.n_pre + w.n_own)), (int32_t)units, sm_count());
    a.may_cut = groups || !w.bounded || sc.per > 0 || sc.parts > 0;
    if (groups) {
        const cudaError_t e = launch_pdl(fxr::attn8::visible_steps_kernel, dim3(w.units, p.n_streams), dim3(fxr::attn8::kVisThreads), 0,
                                         s, a, w.steps, w.list, w.groups);
        if (e != cudaSuccess) return cuda_status(e, "visible_steps_kernel launch");
        a.steps = w.steps;
        a.list = w.list;
        a.groups = w.groups;
    }
    cudaError_t e = launch_pdl(fxr::attn8::tile_kernel<T, F>, dim3(sm_count()), dim3(fxr::attn8::kTileThreads),
                               fxr::attn8::kTileSmem, s, maps, a);
    if (e != cudaSuccess) return cuda_status(e, "tile_kernel launch");
    if (!a.may_cut) return FXR_OK;
    e = launch_pdl(fxr::attn8::combine_kernel<T>, dim3(sm_count() * fxr::attn8::kCombineCtas), dim3(fxr::attn8::kCombineThreads), 0,
                   s, p, static_cast<const float*>(w.part), static_cast<const fxr::attn8::CutUnit*>(w.cuts));
    return cuda_status(e, "combine_kernel launch");
}

// Without groups and prefix: the caches in 16 bits, then the 16-bit attention.
template <typename T, int F>
int32_t launch_q8_wide(const fxr_frame_desc* d, const fxr::attn8::Params& p, const Q8Work& w, cudaStream_t s) {
    const int32_t slots = kSplitSlotsPerSm * sm_count();
    const SplitArea split = split_area(0, w.split, split_bytes(slots), d->n_heads);
    const int64_t C = (int64_t)d->n_heads * d->head_dim;
    fxr::q8::ExpandArgs a{};
    AttnStreamArgs st[FXR_MAX_BATCH];
    for (int32_t b = 0; b < p.n_streams; ++b) {
        const size_t first = (size_t)b * (size_t)d->n_tokens * (size_t)C * 2;
        a.src[b] = p.s[b].c;
        a.count[b] = p.s[b].count;
        st[b] = AttnStreamArgs{p.s[b].qc, p.s[b].ld_qc, w.wide_rows + b, w.wide_k + first, w.wide_v + first, p.s[b].idx, p.s[b].out,
                               nullptr, p.max_rows};
    }
    a.n_streams = p.n_streams;
    a.n_tokens = p.n_tokens;
    a.n_heads = p.n_heads;
    a.max_rows = p.max_rows;
    a.k = w.wide_k;
    a.v = w.wide_v;
    a.rows = w.wide_rows;
    a.zero = reinterpret_cast<uint4*>(split.cnt);
    a.n_zero = (int32_t)((size_t)split.slots * kSplitCntBytes / sizeof(uint4));
    const int64_t units = (int64_t)d->n_tokens * d->n_heads * (fxr::kHeadDim / 16);
    const int grid = (int)std::max<int64_t>(1, std::min<int64_t>((units + fxr::q8::kReadThreads - 1) / fxr::q8::kReadThreads,
                                                                (int64_t)sm_count() * 64));
    const int32_t rc = cuda_status(launch_pdl(fxr::q8::q8_expand_kernel<T, F>, dim3(grid, p.n_streams), dim3(fxr::q8::kReadThreads), 0, s, a),
                                   "q8_expand_kernel launch");
    if (rc != FXR_OK) return rc;
    fxr_frame_desc packed = *d;
    packed.ld_cache = C;
    // Units cut between CTAs read their keys out of step, which costs L2 hits: a step then takes 1.1 times
    // one of whole units and more (4224 rows over 16896 keys: 1000 us cut, 905 whole; 3300 rows 818, and 845;
    // 2304 rows over 4608 keys 142, and 158). The kernel would cut at equal steps; without a bound (the rows are not known here) it decides.
    const int64_t n = (int64_t)w.units * d->n_heads * p.n_streams, ctas = sm_count();
    const float whole = (float)((n + ctas - 1) / ctas) * ((float)w.n_own + fxr::attn2::kItemOverheadSteps);
    const float each = (float)(n * w.n_own) / (float)ctas;
    const float cut = each + fxr::attn2::kItemOverheadSteps * (each / (float)w.n_own + 1.f) + 2.f * fxr::attn2::kCutOverheadSteps;
    const bool may_cut = !w.bounded || whole > 1.1f * cut;
    return launch_attention_streams<T>(&packed, p.n_streams, st, may_cut ? split : SplitArea{}, s);
}

int32_t check_groups(const uint32_t* g, const char* what) {
    return (reinterpret_cast<uintptr_t>(g) & 3u) ? fail(FXR_ERR_INVALID, "%s must be 4-byte aligned", what) : FXR_OK;
}

int32_t check_q8_attention(const fxr_frame_desc* desc, int32_t n_streams, const fxr_q8_stream* streams, const fxr_q8_cache* prefix,
                           const uint32_t* prefix_groups) {
    int32_t st;
    if (prefix && (st = check_q8_cache(desc, prefix, 0, "prefix")) != FXR_OK) return st;
    if ((st = check_groups(prefix_groups, "prefix_groups")) != FXR_OK) return st;
    const int64_t C = (int64_t)desc->n_heads * desc->head_dim;
    for (int32_t b = 0; b < n_streams; ++b) {
        const fxr_q8_stream& s = streams[b];
        if ((st = check_q8_cache(desc, &s.cache, desc->n_tokens, "stream cache")) != FXR_OK) return st;
        if (s.cache.format != streams[0].cache.format || (prefix && s.cache.format != prefix->format))
            return fail(FXR_ERR_INVALID, "stream %d: the caches of a call share one format", b);
        if (!s.qc || !s.idx || !s.count || !s.out) return fail(FXR_ERR_INVALID, "stream %d: null pointer", b);
        if (!aligned16(s.qc) || !aligned16(s.out)) return fail(FXR_ERR_INVALID, "stream %d: qc/out must be 16-byte aligned", b);
        if (s.ld_qc < C || (s.ld_qc % 8)) return fail(FXR_ERR_INVALID, "stream %d: ld_qc must be a multiple of 8, >= n_heads*head_dim", b);
        if ((st = check_groups(s.q_groups, "q_groups")) != FXR_OK || (st = check_groups(s.k_groups, "k_groups")) != FXR_OK) return st;
    }
    return FXR_OK;
}

}  // namespace

extern "C" {

size_t fxr_q8_save_row_bytes(const fxr_frame_desc* desc) {
    if (!desc || desc->n_heads <= 0 || desc->head_dim <= 0) return 0;
    return (size_t)q8_save_bytes(desc);
}

int32_t fxr_gather_norm_rope_q8(const fxr_frame_desc* desc, const void* q, const void* k, const void* v,
                                const int32_t* mask, const int32_t* idx, const int32_t* count, const int32_t* pos,
                                const float* norm_q, const float* norm_k, void* qc, int64_t ld_qc,
                                const fxr_q8_cache* cache, void* save, void* stream) {
    int32_t st = check_desc(desc, false);
    if (st != FXR_OK) return st;
    if ((st = check_q8_cache(desc, cache, desc->n_tokens, "fxr_gather_norm_rope_q8")) != FXR_OK) return st;
    if (desc->n_tokens == 0) return FXR_OK;
    if (!q || !k || !v || !mask || !idx || !count || !norm_q || !norm_k || !qc || (desc->rope_n_axes > 0 && !pos))
        return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v) || !aligned16(qc) || (save && !aligned16(save)))
        return fail(FXR_ERR_INVALID, "Q/K/V/qc/save must be 16-byte aligned");
    if (ld_qc < (int64_t)desc->n_heads * desc->head_dim || (ld_qc % 8))
        return fail(FXR_ERR_INVALID, "ld_qc must be a multiple of 8, >= n_heads*head_dim");
    fxr::q8::WriteArgs a{};
    a.q = q;
    a.k = k;
    a.v = v;
    a.mask = mask;
    a.idx = idx;
    a.count = count;
    a.pos = pos;
    a.norm_q = norm_q;
    a.norm_k = norm_k;
    a.qc = qc;
    a.ld_qc = ld_qc;
    a.ld_qkv = desc->ld_qkv;
    a.save = static_cast<uint8_t*>(save);
    return launch_q8_write(desc, cache, a, false, desc->n_tokens, static_cast<cudaStream_t>(stream));
}

int32_t fxr_cache_write_q8(const fxr_frame_desc* desc, const void* cache_k, const void* cache_v, const int32_t* idx,
                           const int32_t* count, int32_t host_count, const fxr_q8_cache* cache, void* stream) {
    int32_t st = check_desc(desc, false);
    if (st != FXR_OK) return st;
    if ((st = check_q8_cache(desc, cache, desc->n_tokens, "fxr_cache_write_q8")) != FXR_OK) return st;
    if (!count && host_count < 0) return fail(FXR_ERR_INVALID, "neither count nor host_count");
    if (!count && host_count > desc->n_tokens) return fail(FXR_ERR_INVALID, "host_count %d > n_tokens", host_count);
    if (desc->n_tokens == 0 || (!count && host_count == 0)) return FXR_OK;
    if (!cache_k || !cache_v) return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!aligned16(cache_k) || !aligned16(cache_v)) return fail(FXR_ERR_INVALID, "cache_k/cache_v must be 16-byte aligned");
    fxr::q8::WriteArgs a{};
    a.k = cache_k;
    a.v = cache_v;
    a.idx = idx;
    a.count = count;
    a.host_count = host_count;
    a.ld_qkv = desc->ld_cache;
    return launch_q8_write(desc, cache, a, true, count ? desc->n_tokens : host_count, static_cast<cudaStream_t>(stream));
}

int32_t fxr_cache_read_q8(const fxr_frame_desc* desc, const fxr_q8_cache* cache, const int32_t* idx, const int32_t* count,
                          int32_t host_count, void* k, void* v, int64_t ld, void* stream) {
    NvtxRange nvtx_("fxr:q8_read");
    int32_t st = check_desc(desc, false);
    if (st != FXR_OK) return st;
    if ((st = check_q8_cache(desc, cache, 0, "fxr_cache_read_q8")) != FXR_OK) return st;
    if (!count && host_count < 0) return fail(FXR_ERR_INVALID, "neither count nor host_count");
    if (!count && host_count > cache->n_rows) return fail(FXR_ERR_INVALID, "host_count %d > %d cache rows", host_count, cache->n_rows);
    if (cache->n_rows == 0 || (!count && host_count == 0)) return FXR_OK;
    if (!k || !v) return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!aligned16(k) || !aligned16(v)) return fail(FXR_ERR_INVALID, "k/v must be 16-byte aligned");
    if (ld < (int64_t)desc->n_heads * desc->head_dim || (ld % 8))
        return fail(FXR_ERR_INVALID, "ld must be a multiple of 8, >= n_heads*head_dim");
    const int32_t bound = host_count > 0 ? std::min(host_count, cache->n_rows) : cache->n_rows;
    fxr::q8::ReadArgs a{q8_arg(cache), idx, count, host_count, k, v, ld, cache->n_rows, bound, desc->n_heads};
    const int64_t units = (int64_t)bound * desc->n_heads * (fxr::kHeadDim / 16);
    // CTAs per SM at most: short ones that the hardware balances for a whole cache (16896 rows in a graph:
    // 58 us against 67 us with 16), fewer where most may find nothing to do (1153 of 4608 rows: 6.3 against 6.8)
    const int64_t ctas = (units + fxr::q8::kReadThreads - 1) / fxr::q8::kReadThreads, sms = sm_count();
    const int grid = (int)std::max<int64_t>(1, std::min(ctas, sms * (ctas > sms * 32 ? 64 : 16)));
    return q8_dispatch(desc->dtype, cache->format, [&](auto t, auto f) -> int32_t {
        using T = decltype(t);
        constexpr int F = decltype(f)::value;
        return cuda_status(launch_pdl(fxr::q8::q8_read_kernel<T, F>, dim3(grid), dim3(fxr::q8::kReadThreads), 0,
                                      static_cast<cudaStream_t>(stream), a),
                           "q8_read_kernel launch");
    });
}

int32_t fxr_restore_rows_q8(const fxr_frame_desc* desc, const int32_t* mask, const int32_t* idx, const int32_t* count,
                            const void* save, const fxr_q8_cache* cache, void* stream) {
    NvtxRange nvtx_("fxr:q8_restore");
    int32_t st = check_desc(desc, false);
    if (st != FXR_OK) return st;
    if ((st = check_q8_cache(desc, cache, desc->n_tokens, "fxr_restore_rows_q8")) != FXR_OK) return st;
    if (desc->n_tokens == 0) return FXR_OK;
    if (!mask || !idx || !count || !save) return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!aligned16(save)) return fail(FXR_ERR_INVALID, "save must be 16-byte aligned");
    fxr::q8::RestoreArgs a{q8_arg(cache), mask, idx, count, static_cast<const uint8_t*>(save), q8_save_bytes(desc),
                           desc->n_tokens, desc->n_heads};
    return cuda_status(launch_pdl(fxr::q8::q8_restore_kernel, dim3(grid_rows(desc->n_tokens, 8)), dim3(256), 0,
                                  static_cast<cudaStream_t>(stream), a),
                       "q8_restore_kernel launch");
}

size_t fxr_attention_q8_workspace_size(const fxr_frame_desc* desc, int32_t n_streams, int32_t n_prefix, int32_t max_rows) {
    if (!desc || desc->n_heads <= 0 || desc->n_tokens < 0 || n_streams <= 0 || n_prefix < 0) return 0;
    return carve_q8(desc, n_streams, n_prefix, max_rows, nullptr).total;
}

int32_t fxr_attention_q8(const fxr_frame_desc* desc, int32_t n_streams, const fxr_q8_stream* streams,
                         const fxr_q8_cache* prefix, const uint32_t* prefix_groups, int32_t max_rows, void* workspace,
                         size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_("fxr:attention_q8");
    int32_t st = check_desc(desc, true);
    if (st != FXR_OK) return st;
    if (n_streams < 0) return fail(FXR_ERR_INVALID, "n_streams < 0");
    if (n_streams == 0 || desc->n_tokens == 0) return FXR_OK;
    if (!streams) return fail(FXR_ERR_INVALID, "null streams");
    if ((st = check_q8_attention(desc, n_streams, streams, prefix, prefix_groups)) != FXR_OK) return st;
    const int32_t n_prefix = prefix ? prefix->n_rows : 0;
    const Q8Work w = carve_q8(desc, n_streams, n_prefix, max_rows, workspace);
    if (!workspace) return fail(FXR_ERR_INVALID, "null workspace");
    if (!aligned16(workspace)) return fail(FXR_ERR_INVALID, "workspace must be 16-byte aligned");
    if (workspace_bytes < w.total) return fail(FXR_ERR_WORKSPACE, "workspace %zu < required %zu", workspace_bytes, w.total);
    if (w.few && w.line >= INT32_MAX) return fail(FXR_ERR_UNSUPPORTED, "too many keys x heads x row groups for one call (%lld)", (long long)w.line);
    if (!w.few && (int64_t)(w.n_pre + w.n_own) * w.units * desc->n_heads * std::min(n_streams, FXR_MAX_BATCH) >= INT32_MAX)
        return fail(FXR_ERR_UNSUPPORTED, "too many rows x keys x heads for one call");
    if (!w.few && w.n_pre + w.n_own > 0x7fff)
        return fail(FXR_ERR_UNSUPPORTED, "%d key rows: more than 32767 tiles of 128", n_prefix + desc->n_tokens);
    for (int32_t b0 = 0; b0 < n_streams; b0 += FXR_MAX_BATCH) {
        fxr::attn8::Params p{};
        p.n_streams = std::min(n_streams - b0, FXR_MAX_BATCH);
        for (int32_t b = 0; b < p.n_streams; ++b) {
            const fxr_q8_stream& s = streams[b0 + b];
            p.s[b] = fxr::attn8::Stream{s.qc, s.idx, s.count, s.out, s.q_groups, s.k_groups, s.ld_qc, q8_arg(&s.cache)};
        }
        bool groups = false;
        for (int32_t b = 0; b < p.n_streams; ++b) groups = groups || p.s[b].qg != nullptr || p.s[b].kg != nullptr;
        if (prefix) p.prefix = q8_arg(prefix);
        p.pg = prefix_groups;
        p.n_tokens = desc->n_tokens;
        p.n_prefix = n_prefix;
        p.n_heads = desc->n_heads;
        p.max_rows = w.rows;
        p.ld_out = desc->ld_out;
        p.scale_log2 = (desc->softmax_scale > 0.f ? desc->softmax_scale : 1.0f / std::sqrt((float)desc->head_dim)) * 1.4426950408889634f;
        p.part = w.part;
        p.cnt = w.cnt;
        st = q8_dispatch(desc->dtype, streams[0].cache.format, [&](auto t, auto f) -> int32_t {
            using T = decltype(t);
            constexpr int F = decltype(f)::value;
            const cudaStream_t cs = static_cast<cudaStream_t>(stream);
            if (!w.few) return w.wide && !groups ? launch_q8_wide<T, F>(desc, p, w, cs) : launch_q8_tiles<T, F>(desc, p, w, cs);
            return w.tiles == 1   ? launch_q8_rows<T, F, 1>(desc, p, cs)
                   : w.tiles == 2 ? launch_q8_rows<T, F, 2>(desc, p, cs)
                                  : launch_q8_rows<T, F, 4>(desc, p, cs);
        });
        if (st != FXR_OK) return st;
    }
    return FXR_OK;
}

}  // extern "C"

namespace {

struct Q8FrameViews {
    int32_t* count;
    int32_t* idx;
    void* qc;
    void* save;
    char* attn;
    size_t attn_bytes, total;
};

Q8FrameViews carve_q8_frame(const fxr_frame_desc* d, int32_t n_prefix, int32_t max_rows, void* ws) {
    Q8FrameViews v{};
    const size_t N = (size_t)(d->n_tokens > 0 ? d->n_tokens : 1), C = (size_t)d->n_heads * d->head_dim;
    size_t off = 0;
    char* b = static_cast<char*>(ws);
    auto take = [&](size_t bytes) {
        char* p = b ? b + off : nullptr;
        off = align_up(off + bytes, 256);
        return p;
    };
    v.count = reinterpret_cast<int32_t*>(take(sizeof(int32_t)));
    v.idx = reinterpret_cast<int32_t*>(take(N * sizeof(int32_t)));
    v.qc = take(N * C * dtype_bytes(d->dtype));
    v.save = take(N * (size_t)q8_save_bytes(d));
    v.attn_bytes = carve_q8(d, 1, n_prefix, max_rows, nullptr).total;
    v.attn = take(v.attn_bytes);
    v.total = off;
    return v;
}

}  // namespace

extern "C" {

size_t fxr_frame_q8_workspace_size(const fxr_frame_desc* desc, int32_t n_prefix, int32_t max_rows) {
    if (!desc || dtype_bytes(desc->dtype) == 0 || desc->n_heads <= 0 || desc->head_dim <= 0 || desc->n_tokens < 0 || n_prefix < 0)
        return 0;
    return carve_q8_frame(desc, n_prefix, max_rows, nullptr).total;
}

int32_t fxr_frame_forward_q8(const fxr_frame_desc* desc, const void* q, const void* k, const void* v, int32_t* mask,
                             const uint8_t* valid, const int32_t* pos, const float* norm_q, const float* norm_k,
                             const fxr_q8_cache* cache, const uint32_t* q_groups, const uint32_t* k_groups,
                             const fxr_q8_cache* prefix, const uint32_t* prefix_groups, int32_t max_rows, void* out,
                             void* workspace, size_t workspace_bytes, void* stream) {
    NvtxRange nvtx_("fxr:frame_q8");
    int32_t st = check_desc(desc, true);
    if (st != FXR_OK) return st;
    if (desc->n_tokens == 0) return FXR_OK;
    if (!cache || !mask || !out) return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!workspace) return fail(FXR_ERR_INVALID, "null workspace");
    if (!aligned16(workspace)) return fail(FXR_ERR_INVALID, "workspace must be 16-byte aligned");
    const int32_t n_prefix = prefix ? prefix->n_rows : 0;
    if (n_prefix < 0) return fail(FXR_ERR_INVALID, "prefix: n_rows < 0");
    const Q8FrameViews w = carve_q8_frame(desc, n_prefix, max_rows, workspace);
    if (workspace_bytes < w.total) return fail(FXR_ERR_WORKSPACE, "workspace %zu < required %zu", workspace_bytes, w.total);
    const int64_t C = (int64_t)desc->n_heads * desc->head_dim;
    // every argument is looked at before the first launch
    const fxr_q8_stream s{w.qc, C, w.idx, w.count, out, q_groups, k_groups, *cache};
    if ((st = check_q8_attention(desc, 1, &s, prefix, prefix_groups)) != FXR_OK) return st;
    if (!q || !k || !v || !norm_q || !norm_k || (desc->rope_n_axes > 0 && !pos)) return fail(FXR_ERR_INVALID, "null pointer argument");
    if (!aligned16(q) || !aligned16(k) || !aligned16(v)) return fail(FXR_ERR_INVALID, "Q/K/V must be 16-byte aligned");
    fxr::CompactArgs ca{};
    ca.s[0] = fxr::CompactStream{mask, valid, w.idx, w.count, fxr::RestoreList{}};
    // the compaction also zeroes the attention's arrivals
    st = launch_compact_streams(ca, 1, desc->n_tokens, SplitArea{}, stream, w.attn,
                                carve_q8(desc, 1, n_prefix, max_rows, nullptr).zero_bytes);
    if (st != FXR_OK) return st;
    if ((st = fxr_gather_norm_rope_q8(desc, q, k, v, mask, w.idx, w.count, pos, norm_q, norm_k, w.qc, C, cache, w.save, stream)) != FXR_OK)
        return st;
    if ((st = fxr_attention_q8(desc, 1, &s, prefix, prefix_groups, max_rows, w.attn, w.attn_bytes, stream)) != FXR_OK) return st;
    return fxr_restore_rows_q8(desc, mask, w.idx, w.count, w.save, cache, stream);
}

}  // extern "C"
