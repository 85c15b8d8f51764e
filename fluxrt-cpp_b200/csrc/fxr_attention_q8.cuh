// fxr_attention_q8.cuh — attention of executed rows over the 8-bit spatial cache (sm_100a).
//
//   out[idx[m]] = sum_j p_mj v_j / sum_j p_mj,   p_mj = allow(m, j) * exp(scale * q_m . k_j)
// over the rows of a prefix that every stream of the launch shares and then the stream's own rows;
// allow(m, j) = (q_groups[idx[m]] & k_groups[j]) != 0. A row that sees no key gives zeros.
//
// A key whose K or V scale is not finite (its 16-bit row held an infinity or NaN) makes the rows that
// see it NaN and no others: its score is set to NaN before the mask and its V codes count as zeros.
#pragma once

#include "fxr_attention2.cuh"
#include "fxr_q8.cuh"

namespace fxr {
namespace attn8 {

using q8::Cache;

struct Stream {
    const void* qc;
    const int32_t* idx;
    const int32_t* count;
    void* out;
    const uint32_t* qg;          // [n_tokens] or NULL
    const uint32_t* kg;          // [n_tokens] or NULL
    int64_t ld_qc;
    Cache c;
};

struct Params {
    Stream s[kMaxBatch];
    Cache prefix;
    const uint32_t* pg;          // [n_prefix] or NULL
    int32_t n_streams, n_tokens, n_prefix, n_heads;
    int32_t max_rows;            // compact rows of a stream beyond this one are not computed
    int64_t ld_out;
    float scale_log2;
    float* part;                 // partial results, kRowsSlotFloats each
    int32_t* cnt;                // [n_heads] arrivals, zero between launches
};

// ---------------------------------------------------------------------------------------------
// Few rows per stream: bound by reading the cache once. One CTA per SM takes items of (16 rows, head,
// key range); its 8 warps walk the range in blocks of 32 keys, each with its own running maximum,
// sum and O, so that no warp waits for another inside the loop. A warp streams its blocks through a
// ring of 3 in shared memory with 16-byte asynchronous copies (8 KB of codes per block: ~190 KB in
// flight per SM). The codes become 16-bit operands in registers, on their way from shared memory to
// mma.m16n8k16 (tcgen05 reads operands from memory and wants 128 rows; these calls have a few):
//   S = Q K^T: a lane's B operand of a 16-dim step is 4 codes of one key. The order of the 128 dims
//     inside a dot product is free, so the lane takes 16 consecutive bytes for four steps, and Q's
//     fragments are loaded in the same order.
//   O += P V: the operand pairs two keys of one dim: one byte permute takes both codes. A lane's 16
//     column tiles are 16 consecutive dims (dim = 16 * column + tile).
// K scales multiply the scores in 32 bits. A V scale is split into 2^e * f, f in [1, 2): f multiplies
// P before its one rounding to T, 2^e the codes, exactly (all of the scale on P would push it into
// f16's subnormals; all of it on V would cost a second rounding). bf16 P holds the whole product.
// Rows of several streams share an MMA tile against the prefix (its codes are read once for every 16
// of all streams' rows); own rows are per stream. The key range of an item is the shortest multiple
// of 128 that gives every item a CTA at once, or whole sources when there are more (row, head)
// groups than CTAs. Partial results (O, maximum, sum) meet in L2: the last item of a head to arrive
// combines that head's rows in key order, so the result does not depend on the order of arrival.
// ---------------------------------------------------------------------------------------------
constexpr int kRowsWarps = 8;
constexpr int kRowsThreads = 32 * kRowsWarps;
constexpr int kRowsTile = 16;
constexpr int kBlk = 32;                       // keys per block
constexpr int kDepth = 3;                      // ring
constexpr int kChunkUnit = 128;                // key ranges are multiples of this
constexpr uint32_t kBlkBytes = kBlk * 128;     // codes of one of K, V
constexpr uint32_t kOffScale = 2 * kBlkBytes;  // K scales, V scales (kBlk x 2 bytes each), groups
constexpr uint32_t kOffGroup = kOffScale + 2 * kBlk * 2;
constexpr uint32_t kRingSlot = kOffGroup + kBlk * 4;
constexpr uint32_t kRingWarp = kDepth * kRingSlot;
constexpr int kPadRow = 132;                   // floats per O row in the warps' exchange
constexpr uint32_t kRowsSmem = kRowsWarps * kRingWarp + 2 * kRowsWarps * kRowsTile * 4;
constexpr int kRowsSlotFloats = kRowsTile * kHeadDim + 2 * kRowsTile;
static_assert(kRowsWarps * kRowsTile * kPadRow * 4 <= kRowsWarps * kRingWarp, "exchange fits the ring");

__device__ __forceinline__ void cp_async16(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.cg.shared.global [%0], [%1], 16, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async4(uint32_t dst, const void* src, uint32_t bytes) {
    asm volatile("cp.async.ca.shared.global [%0], [%1], 4, %2;" ::"r"(dst), "l"(src), "r"(bytes) : "memory");
}
__device__ __forceinline__ void cp_async_commit() { asm volatile("cp.async.commit_group;" ::: "memory"); }
template <int N> __device__ __forceinline__ void cp_async_wait() {
    asm volatile("cp.async.wait_group %0;" ::"n"(N) : "memory");
}
__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}
__device__ __forceinline__ uint32_t lds32(uint32_t a) {
    uint32_t v;
    asm volatile("ld.shared.u32 %0, [%1];" : "=r"(v) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ uint2 lds64(uint32_t a) {
    uint2 v;
    asm volatile("ld.shared.v2.u32 {%0,%1}, [%2];" : "=r"(v.x), "=r"(v.y) : "r"(a) : "memory");
    return v;
}

template <typename T>
__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <>
__device__ __forceinline__ void mma16816<__nv_bfloat16>(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3,
                                                        uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
template <>
__device__ __forceinline__ void mma16816<__half>(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0,
                                                 uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}

__device__ __forceinline__ bool finite(float x) { return (__float_as_uint(x) & 0x7f800000u) != 0x7f800000u; }

// The launch's division into items, the same on every thread: a function of the counts.
struct RowsPlan {
    int32_t rows[kMaxBatch];     // of each stream
    int32_t total;               // of all streams
    int32_t gp;                  // 16-row groups of the packed rows (prefix items), 0 without a prefix
    int32_t go;                  // of the streams' own items, all streams
    int32_t len;                 // keys of an item
    int32_t np, no;              // items per group: prefix, own
    int32_t items;
};

__device__ __forceinline__ RowsPlan rows_plan(const Params& p) {
    RowsPlan r{};
#pragma unroll
    for (int b = 0; b < kMaxBatch; ++b) {
        r.rows[b] = 0;
        if (b < p.n_streams) {
            const int32_t c = *p.s[b].count;
            r.rows[b] = max(0, min(c, p.max_rows));
            if (c > p.max_rows && blockIdx.x == 0 && threadIdx.x == 0) atomicOr(&g_error_word, kErrBounds);
        }
        r.total += r.rows[b];
        r.go += (r.rows[b] + kRowsTile - 1) / kRowsTile;
    }
    if (r.total == 0) return r;
    r.gp = p.n_prefix > 0 ? (r.total + kRowsTile - 1) / kRowsTile : 0;
    const int32_t groups = p.n_heads * (r.gp + r.go), grid = (int32_t)gridDim.x;
    const int32_t target = (groups + grid - 1) / grid * grid;
    const int32_t longest = max(p.n_prefix, p.n_tokens);
    const int64_t keys = (int64_t)p.n_heads * ((int64_t)r.gp * p.n_prefix + (int64_t)r.go * p.n_tokens);
    r.len = max(1, (int32_t)(keys / ((int64_t)target * kChunkUnit))) * kChunkUnit;
    for (;;) {
        r.np = (p.n_prefix + r.len - 1) / r.len;
        r.no = (p.n_tokens + r.len - 1) / r.len;
        r.items = p.n_heads * (r.gp * r.np + r.go * r.no);
        if (r.items <= target || r.len >= longest) break;
        r.len += kChunkUnit;
    }
    return r;
}

// Packed row pr -> stream and compact row.
__device__ __forceinline__ void unpack_row(const Params& p, const RowsPlan& r, int32_t pr, int32_t& b, int32_t& m) {
    b = -1;
    m = pr;
#pragma unroll
    for (int k = 0; k < kMaxBatch; ++k) {
        if (b < 0 && k < p.n_streams) {
            if (m < r.rows[k]) b = k;
            else m -= r.rows[k];
        }
    }
}

// Rows of head h from the partial results of every item, a warp per row, 4 dims per lane.
template <typename T>
__device__ __noinline__ void rows_combine(const Params& p, const RowsPlan& r, int32_t h) {
    const int lane = threadIdx.x & 31;
    for (int32_t pr = threadIdx.x >> 5; pr < r.total; pr += kRowsWarps) {
        int32_t b, m;
        unpack_row(p, r, pr, b, m);
        int32_t base = p.n_heads * r.gp * r.np, groups = 0;
        const Stream* st = &p.s[0];
#pragma unroll
        for (int k = 0; k < kMaxBatch; ++k) {
            const int32_t g = (r.rows[k] + kRowsTile - 1) / kRowsTile;
            if (k < b) base += p.n_heads * g * r.no;
            if (k == b) {
                groups = g;
                st = &p.s[k];
            }
        }
        const int32_t n_pre = r.gp > 0 ? r.np : 0, n = n_pre + r.no;
        const int32_t pre0 = (h * r.gp + pr / kRowsTile) * r.np, own0 = base + (h * groups + m / kRowsTile) * r.no;
        auto slot = [&](int32_t c) { return p.part + (int64_t)(c < n_pre ? pre0 + c : own0 + c - n_pre) * kRowsSlotFloats; };
        auto row_of = [&](int32_t c) { return c < n_pre ? pr % kRowsTile : m % kRowsTile; };
        float top = -INFINITY;
        for (int32_t c = lane; c < n; c += 32) top = fmaxf(top, __ldcg(slot(c) + kRowsTile * kHeadDim + row_of(c)));
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, o));
        if (top == -INFINITY) top = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        float l = 0.f;
#pragma unroll 4
        for (int32_t c = 0; c < n; ++c) {
            const float* q = slot(c);
            const int32_t rr = row_of(c);
            const float w = ex2_approx(__ldcg(q + kRowsTile * kHeadDim + rr) - top);
            l += w * __ldcg(q + kRowsTile * kHeadDim + kRowsTile + rr);
            const float4 x = __ldcg(reinterpret_cast<const float4*>(q + rr * kHeadDim) + lane);
            acc.x += w * x.x;
            acc.y += w * x.y;
            acc.z += w * x.z;
            acc.w += w * x.w;
        }
        const int32_t i = st->idx[m];
        if (i < 0 || i >= p.n_tokens) {
            if (lane == 0) atomicOr(&g_error_word, kErrBounds);
            continue;
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        T* out = static_cast<T*>(st->out) + (int64_t)i * p.ld_out + (int64_t)h * kHeadDim;
        *reinterpret_cast<uint2*>(out + 4 * lane) =
            make_uint2(StoreT<T>::pack2(acc.x * inv, acc.y * inv), StoreT<T>::pack2(acc.z * inv, acc.w * inv));
    }
}

template <typename T, int F>
__global__ void __launch_bounds__(kRowsThreads, 1) rows_kernel(const __grid_constant__ Params p) {
    extern __shared__ __align__(128) uint8_t smem[];
    __shared__ int32_t last;
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t ring = smem_u32(smem) + warp * kRingWarp;
    float* xo = reinterpret_cast<float*>(smem);                                     // [warp][16][kPadRow]
    float* xm = reinterpret_cast<float*>(smem + kRowsWarps * kRingWarp);            // [warp][16] maxima, then sums
    pdl_launch_dependents();
    pdl_wait();
    const RowsPlan r = rows_plan(p);
    const int32_t pre_items = p.n_heads * r.gp * r.np;

    for (int32_t item = blockIdx.x; item < r.items; item += gridDim.x) {
        // ---- the item: 16 rows of head h against keys [k0, k0 + n) of one source
        const bool pre = item < pre_items;
        int32_t h, grp, chunk, b_own = 0, n_src;
        Cache c = p.prefix;
        const uint32_t* kg = p.pg;
        if (pre) {
            chunk = item % r.np;
            const int32_t e = item / r.np;
            h = e / r.gp;
            grp = e - h * r.gp;
            n_src = p.n_prefix;
        } else {
            int32_t e = item - pre_items, groups = 1;
            b_own = -1;
#pragma unroll
            for (int k = 0; k < kMaxBatch; ++k) {
                const int32_t gk = (r.rows[k] + kRowsTile - 1) / kRowsTile, n_k = p.n_heads * gk * r.no;
                if (b_own < 0 && k < p.n_streams) {
                    if (e < n_k) {
                        b_own = k;
                        groups = gk;
                        c = p.s[k].c;
                        kg = p.s[k].kg;
                    } else {
                        e -= n_k;
                    }
                }
            }
            chunk = e % r.no;
            e /= r.no;
            h = e / groups;
            grp = e - h * groups;
            n_src = p.n_tokens;
        }
        const int32_t k0 = chunk * r.len;
        const int32_t n_keys = min(r.len, n_src - k0), n_blk = (n_keys + kBlk - 1) / kBlk;

        const uint8_t* ck = c.k + (int64_t)h * kHeadDim;
        const uint8_t* cv = c.v + (int64_t)h * kHeadDim;
        const T* ks = static_cast<const T*>(c.ks) + (int64_t)h * c.ld_scale;
        const T* vs = static_cast<const T*>(c.vs) + (int64_t)h * c.ld_scale;
        // ---- asynchronous copies of block b of this warp's walk into ring slot `slot`. Keys past the
        // source are filled with zeros (scales in groups of 8, whose rows are padded to 8).
        auto fetch = [&](int32_t b, int slot) {
            const uint32_t dst = ring + slot * kRingSlot;
            const int32_t key0 = k0 + b * kBlk;
            const int32_t row = lane >> 3, ch = lane & 7;
#pragma unroll
            for (int i = 0; i < kBlk / 4; ++i) {
                const int32_t rr = i * 4 + row, key = key0 + rr;
                const bool in = key < n_src;
                const int64_t off = (int64_t)(in ? key : 0) * c.ld + ch * 16;
                cp_async16(dst + rr * 128 + ((ch ^ ((rr & 1) << 2)) << 4), ck + off, in ? 16u : 0u);
                cp_async16(dst + kBlkBytes + rr * 128 + ((ch ^ (rr & 7)) << 4), cv + off, in ? 16u : 0u);
            }
            if (lane < 8) {
                const int32_t key = key0 + (lane & 3) * 8;
                const bool in = key < n_src;
                cp_async16(dst + kOffScale + lane * 16, (lane < 4 ? ks : vs) + (in ? key : 0), in ? 16u : 0u);
            }
            if (kg != nullptr) {
                const bool in = key0 + lane < n_src;
                cp_async4(dst + kOffGroup + lane * 4, kg + (in ? key0 + lane : 0), in ? 4u : 0u);
            }
        };
#pragma unroll
        for (int d = 0; d < kDepth - 1; ++d) {
            const int32_t b = warp + d * kRowsWarps;
            if (b < n_blk) fetch(b, d);
            cp_async_commit();
        }

        // ---- the queries: rows g and g + 8 of the group, fragments in the order of the codes
        uint32_t qa[2][16];
        uint32_t qg[2];
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            int32_t b = b_own, m = grp * kRowsTile + g + 8 * e;
            bool live = true;
            if (pre) {
                const int32_t pr = m;
                live = pr < r.total;
                unpack_row(p, r, live ? pr : 0, b, m);
            }
            const Stream* st = &p.s[0];
#pragma unroll
            for (int k = 0; k < kMaxBatch; ++k)
                if (k == b) {
                    st = &p.s[k];
                    live = live && m < r.rows[k];
                }
            const T* q = static_cast<const T*>(st->qc) + (int64_t)m * st->ld_qc + (int64_t)h * kHeadDim + t * 16;
#pragma unroll
            for (int cc = 0; cc < 2; ++cc)
#pragma unroll
                for (int w = 0; w < 2; ++w) {
                    const uint4 x = live ? *reinterpret_cast<const uint4*>(q + cc * 64 + w * 8) : make_uint4(0, 0, 0, 0);
                    qa[e][cc * 8 + w * 4 + 0] = x.x;
                    qa[e][cc * 8 + w * 4 + 1] = x.y;
                    qa[e][cc * 8 + w * 4 + 2] = x.z;
                    qa[e][cc * 8 + w * 4 + 3] = x.w;
                }
            qg[e] = 0xffffffffu;
            if (live && st->qg != nullptr) {
                const int32_t i = st->idx[m];
                qg[e] = (i >= 0 && i < p.n_tokens) ? st->qg[i] : 0u;
            }
        }

        float o[16][4];
#pragma unroll
        for (int j = 0; j < 16; ++j)
#pragma unroll
            for (int e = 0; e < 4; ++e) o[j][e] = 0.f;
        float m_run[2] = {-INFINITY, -INFINITY}, l_run[2] = {0.f, 0.f};
        const float sc = p.scale_log2 * q8::code_scale<T, F>();

        int slot = 0;
        for (int32_t b = warp; b < n_blk; b += kRowsWarps) {
            {
                const int32_t nb = b + (kDepth - 1) * kRowsWarps;
                int ns = slot + kDepth - 1;
                if (ns >= kDepth) ns -= kDepth;
                if (nb < n_blk) fetch(nb, ns);
                cp_async_commit();
                cp_async_wait<kDepth - 1>();
                __syncwarp();
            }
            const uint32_t at = ring + slot * kRingSlot;
            // S = Q K^T, four tiles of 8 keys
            float s[4][4];
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                s[nt][0] = s[nt][1] = s[nt][2] = s[nt][3] = 0.f;
                const uint32_t row = at + (nt * 8 + g) * 128, x4 = (uint32_t)(g & 1) << 2;
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const uint4 k4 = lds128(row + (((uint32_t)(cc * 4 + t) ^ x4) << 4));
                    const uint32_t w[4] = {k4.x, k4.y, k4.z, k4.w};
#pragma unroll
                    for (int j = 0; j < 4; ++j)
                        mma16816<T>(s[nt], qa[0][cc * 8 + 2 * j], qa[1][cc * 8 + 2 * j], qa[0][cc * 8 + 2 * j + 1],
                                    qa[1][cc * 8 + 2 * j + 1], q8::decode2<T, F>(w[j], w[j], 0, 1),
                                    q8::decode2<T, F>(w[j], w[j], 2, 3));
                }
            }
            // scales, masks
            float v_sc[4][2];            // what P is multiplied with
            uint32_t v_pow[4];           // f16: the pairs' powers of two
            const int32_t left = n_keys - b * kBlk;
            float bm[2] = {-INFINITY, -INFINITY};
#pragma unroll
            for (int nt = 0; nt < 4; ++nt) {
                const float2 k2 = StoreT<T>::unpack2(lds32(at + kOffScale + (nt * 8 + 2 * t) * 2));
                const float2 v2 = StoreT<T>::unpack2(lds32(at + kOffScale + kBlk * 2 + (nt * 8 + 2 * t) * 2));
                const float kk[2] = {k2.x, k2.y};
                float vv[2] = {v2.x, v2.y};
                uint32_t seen[2] = {0xffffffffu, 0xffffffffu};
                if (kg != nullptr) {
                    const uint2 g2 = lds64(at + kOffGroup + (nt * 8 + 2 * t) * 4);
                    seen[0] = g2.x;
                    seen[1] = g2.y;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const bool v_ok = finite(vv[e]);
                    const float f = v_ok && finite(kk[e]) ? kk[e] * sc : __uint_as_float(0x7fc00000u);
                    v_sc[nt][e] = v_ok ? vv[e] : 0.f;
                    if constexpr (StoreT<T>::kUmmaFormat == 0) {
                        vv[e] = v_sc[nt][e];
                        v_sc[nt][e] = __uint_as_float((__float_as_uint(vv[e]) & 0x007fffffu) | 0x3f800000u);
                        vv[e] = __uint_as_float(__float_as_uint(vv[e]) & 0x7f800000u) * q8::code_scale<T, F>();
                    }
                    const bool in = nt * 8 + 2 * t + e < left;
                    s[nt][e] = in && (seen[e] & qg[0]) ? s[nt][e] * f : -INFINITY;
                    s[nt][2 + e] = in && (seen[e] & qg[1]) ? s[nt][2 + e] * f : -INFINITY;
                    bm[0] = fmaxf(bm[0], s[nt][e]);
                    bm[1] = fmaxf(bm[1], s[nt][2 + e]);
                }
                if constexpr (StoreT<T>::kUmmaFormat == 0) v_pow[nt] = StoreT<T>::pack2(vv[0], vv[1]);
            }
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                bm[e] = fmaxf(bm[e], __shfl_xor_sync(0xffffffffu, bm[e], 1));
                bm[e] = fmaxf(bm[e], __shfl_xor_sync(0xffffffffu, bm[e], 2));
            }
            // the running maxima move only where one grows by more than 2^8 (P stays below that)
            if (__any_sync(0xffffffffu, bm[0] > m_run[0] + 8.f || bm[1] > m_run[1] + 8.f)) {
                float al[2];
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const float mn = fmaxf(m_run[e], bm[e]);
                    al[e] = mn == m_run[e] ? 1.f : ex2_approx(m_run[e] - mn);
                    m_run[e] = mn;
                    l_run[e] *= al[e];
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    o[j][0] *= al[0];
                    o[j][1] *= al[0];
                    o[j][2] *= al[1];
                    o[j][3] *= al[1];
                }
            }
            uint32_t pa[4][2];
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                const float mu = m_run[e] == -INFINITY ? 0.f : m_run[e];
#pragma unroll
                for (int nt = 0; nt < 4; ++nt) {
                    const float p0 = ex2_approx(s[nt][2 * e] - mu), p1 = ex2_approx(s[nt][2 * e + 1] - mu);
                    l_run[e] += p0 + p1;
                    pa[nt][e] = StoreT<T>::pack2(p0 * v_sc[nt][0], p1 * v_sc[nt][1]);
                }
            }
            // O += P V, two steps of 16 keys
#pragma unroll
            for (int kt = 0; kt < 2; ++kt) {
                uint32_t w[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t row = kt * 16 + 2 * t + (e & 1) + (e >> 1) * 8;
                    const uint4 v4 = lds128(at + kBlkBytes + row * 128 + (((uint32_t)g ^ (row & 7)) << 4));
                    w[e][0] = v4.x;
                    w[e][1] = v4.y;
                    w[e][2] = v4.z;
                    w[e][3] = v4.w;
                }
#pragma unroll
                for (int j = 0; j < 16; ++j) {
                    uint32_t b0 = q8::decode2<T, F>(w[0][j >> 2], w[1][j >> 2], j & 3, j & 3);
                    uint32_t b1 = q8::decode2<T, F>(w[2][j >> 2], w[3][j >> 2], j & 3, j & 3);
                    if constexpr (StoreT<T>::kUmmaFormat == 0) {
                        b0 = q8::mul2<T>(b0, v_pow[2 * kt]);
                        b1 = q8::mul2<T>(b1, v_pow[2 * kt + 1]);
                    }
                    mma16816<T>(o[j], pa[2 * kt][0], pa[2 * kt][1], pa[2 * kt + 1][0], pa[2 * kt + 1][1], b0, b1);
                }
            }
            __syncwarp();
            if (++slot == kDepth) slot = 0;
        }
        cp_async_wait<0>();
        __syncthreads();
        // ---- the warps' results meet: O[row][8 * tile + column], then each thread 8 dims of one row
#pragma unroll
        for (int e = 0; e < 2; ++e) {
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 1);
            l_run[e] += __shfl_xor_sync(0xffffffffu, l_run[e], 2);
            float* dst = xo + (warp * kRowsTile + g + 8 * e) * kPadRow + 2 * t;
#pragma unroll
            for (int j = 0; j < 16; ++j) *reinterpret_cast<float2*>(dst + 8 * j) = make_float2(o[j][2 * e], o[j][2 * e + 1]);
            if (t == 0) {
                xm[warp * kRowsTile + g + 8 * e] = m_run[e];
                xm[(kRowsWarps + warp) * kRowsTile + g + 8 * e] = l_run[e];
            }
        }
        __syncthreads();
        {
            const int row = threadIdx.x >> 4, cc = threadIdx.x & 15;
            float top = -INFINITY;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) top = fmaxf(top, xm[w * kRowsTile + row]);
            const float mu = top == -INFINITY ? 0.f : top;
            float acc[8], l = 0.f;
#pragma unroll
            for (int e = 0; e < 8; ++e) acc[e] = 0.f;
#pragma unroll
            for (int w = 0; w < kRowsWarps; ++w) {
                const float f = ex2_approx(xm[w * kRowsTile + row] - mu);
                l += f * xm[(kRowsWarps + w) * kRowsTile + row];
                const float* src = xo + (w * kRowsTile + row) * kPadRow + (cc >> 1) + (cc & 1) * 64;
#pragma unroll
                for (int e = 0; e < 8; ++e) acc[e] += f * src[8 * e];   // dim 16 * (cc / 2) + 8 * (cc % 2) + e
            }
            float* dst = p.part + (int64_t)item * kRowsSlotFloats;
            float4* d4 = reinterpret_cast<float4*>(dst + row * kHeadDim + cc * 8);
            d4[0] = make_float4(acc[0], acc[1], acc[2], acc[3]);
            d4[1] = make_float4(acc[4], acc[5], acc[6], acc[7]);
            if (cc == 0) {
                dst[kRowsTile * kHeadDim + row] = top;
                dst[kRowsTile * kHeadDim + kRowsTile + row] = l;
            }
        }
        __threadfence();
        __syncthreads();
        if (threadIdx.x == 0) {
            const int32_t all = r.gp * r.np + r.go * r.no;
            const int32_t before = atom_add_acq_rel_gpu(p.cnt + h, 1);
            last = before == all - 1;
            if (last) p.cnt[h] = 0;      // for the next launch
        }
        __syncthreads();
        if (last) rows_combine<T>(p, r, h);
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows per stream: bound by the tensor core. The two-tile schedule of the 16-bit attention
// (fxr_attention2.cuh: 256 compact query rows of one head per unit, 128 keys per step, S and O in
// tensor memory, P written over S, lazy rescaling, units cut between CTAs when whole ones would leave
// SMs idle) with K and V tiles that arrive as codes: a fourth warpgroup turns each 128 x 128 tile of
// codes in shared memory into the 16-bit tile that tcgen05.mma reads, T(code * scale), one row per
// thread, in the 128-byte swizzle on both sides (every access of 8 lanes covers all banks). TMA moves
// codes only: half the bytes of the 16-bit cache.
// Warps (512 threads): 0-7 softmax of tile 0 / 1, 8 TMA producer, 9 tensor memory and the MMA-issuing
// thread, 10 scheduler (writes the CTA's items into a 2-slot ring in shared memory, so that no other
// role carries the bookkeeping), 11 idle, 12-15 converters.
// Prefix rows come first, then the stream's own; a source's last tile is filled with zeros and its
// scores masked. With visibility groups, visible_steps_kernel lists for every 256-row unit the tiles
// that some row of it sees, and which of them all its rows see whole; the others are masked score by
// score. Rows that see nothing end with a maximum of -inf and store zeros.
// ---------------------------------------------------------------------------------------------
constexpr int kBM = 128, kUnitRows = 2 * kBM, kBN = 128, kD = kHeadDim;
constexpr int kTileThreads = 512;
constexpr int kProducerWarp = 8, kMmaWarp = 9, kSchedWarp = 10, kConvWarp = 12;
constexpr uint32_t kSpan = 128 * 128;            // bytes of 128 rows x one 128-byte swizzle span
constexpr uint32_t kTile = 2 * kSpan;            // a 128 x 128 16-bit tile
constexpr int kTiles = 4, kRaws = 2;             // rings: converted tiles, code tiles
constexpr uint32_t kTmemColumns = 512, kColS = 0, kColO = 256;
constexpr uint32_t kRegsSoftmax = 176, kRegsOther = 80;
constexpr uint32_t kTileRegPool = 256 * kRegsSoftmax + 256 * kRegsOther;
static_assert(kTileRegPool == kTileThreads * 128, "the warpgroups' shares are the launch's registers");
constexpr int kPolyPeriod = 4;
constexpr float kItemSteps = 2.0f, kCutSteps = 4.5f;   // as the 16-bit kernel's schedule, in steps
constexpr int kPartSlots = 4;                    // partial tiles a CTA may write
constexpr int kPartFloats = kBM * kD + 2 * kBM;
constexpr int kPartWarps = 8;                    // arrival counters per cut unit
constexpr uint32_t kMixed = 1u << 24;            // step information: tile | left << 16 | kMixed

struct TileMaps {
    CUtensorMap q[kMaxBatch], k[kMaxBatch], v[kMaxBatch], pk, pv;
};

// One item: a unit's steps [s0, s0 + n) of its list. n = 0 ends the walk.
struct Item {
    const CUtensorMap* tq;
    const CUtensorMap* tk;
    const CUtensorMap* tv;
    const void* ks;              // own scales of the head
    const void* vs;
    const int32_t* idx;
    const uint32_t* qg;
    void* out;
    const uint16_t* list;        // visible steps of the unit, NULL: all
    int32_t n, s0, head, row0, rows;
    int32_t cut;                 // part of a unit
    int32_t c_first, c_last;     // CTAs that hold the unit's parts
    int32_t i0;                  // its first iteration in the launch
    int32_t stream;
};

enum Bar : uint32_t {
    kQFull = 0, kQEmpty,
    kRawFull, kRawEmpty = kRawFull + kRaws,
    kFull = kRawEmpty + kRaws, kEmpty = kFull + kTiles,
    kSFull = kEmpty + kTiles, kPHalf0 = kSFull + 2, kPHalf1 = kPHalf0 + 2, kPVDone = kPHalf1 + 2, kOFree = kPVDone + 2,
    kItemFull = kOFree + 2, kItemEmpty = kItemFull + 2,
    kDrain = kItemEmpty + 2,
    kNumBars
};
constexpr uint32_t kItemReaders = 1 + 1 + 4 + 8;  // producer, MMA, converter warps, softmax warps
constexpr uint32_t kSmQ = 0, kSmTiles = 2 * kTile, kSmRaw = kSmTiles + kTiles * kTile;
constexpr uint32_t kSmGroup = kSmRaw + kRaws * kSpan;      // [softmax thread] the row's groups
constexpr uint32_t kSmItem = kSmGroup + 256 * 4;
constexpr uint32_t kSmInfo = kSmItem + 2 * 160;            // [4] step information
constexpr uint32_t kSmBar = kSmInfo + 16;
constexpr uint32_t kSmTmem = kSmBar + kNumBars * 8, kSmAbort = kSmTmem + 4;
constexpr uint32_t kTileSmem = kSmBar + 256 + 1024;
static_assert(sizeof(Item) <= 160 && kNumBars * 8 + 8 <= 256 && kSmBar % 8 == 0 && kSmItem % 16 == 0, "shared memory layout");
static_assert(kTileSmem <= 232448, "shared memory budget");

struct TileParams {
    Params p;
    int32_t n_pre, n_own;        // key tiles of the prefix and of a stream's own rows
    int32_t units_cap;           // units of a stream at most (rows of steps / list)
    const int32_t* steps;        // [stream][units_cap] listed steps, NULL: every unit runs all tiles
    const uint16_t* list;        // [stream][units_cap][n_pre + n_own] tile | 0x8000 where it needs the masks
    const uint32_t* groups;      // [n_pre + n_streams * n_own][128] key groups, zeros past a source's end
    float* part;                 // [grid][kPartSlots][kPartFloats]
    int32_t* cnt;                // [grid][kPartWarps], zero between launches
};

// ---- visible steps --------------------------------------------------------------------------------
// CTA (unit, stream): the sets of its 256 rows against every key tile's union and intersection. The
// CTAs of unit 0 also copy the key groups into tiles padded with zeros. A few microseconds for any
// frame: each CTA reads the 4-byte sets of all keys once.
constexpr int kVisThreads = 256;

__global__ void __launch_bounds__(kVisThreads) visible_steps_kernel(const __grid_constant__ TileParams a, int32_t* steps,
                                                                    uint16_t* list, uint32_t* groups) {
    __shared__ uint32_t any_row;
    __shared__ uint32_t all_of[kVisThreads], any_of[kVisThreads];
    __shared__ uint32_t row_word[kUnitRows];      // the rows' distinct sets (distinct within a warp)
    __shared__ int32_t n_words;
    pdl_launch_dependents();
    pdl_wait();
    const int b = blockIdx.y, unit = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const Params& p = a.p;
    const uint32_t *qg = nullptr, *kg = nullptr;
    const int32_t *idx = nullptr, *count = nullptr;
#pragma unroll
    for (int k = 0; k < kMaxBatch; ++k)
        if (k == b) {
            qg = p.s[k].qg;
            kg = p.s[k].kg;
            idx = p.s[k].idx;
            count = p.s[k].count;
        }
    const int32_t rows = max(0, min(*count, p.max_rows)), row = unit * kUnitRows + (int32_t)threadIdx.x;
    if (unit * kUnitRows >= rows && unit > 0) return;
    if (threadIdx.x == 0) {
        any_row = 0;
        n_words = 0;
    }
    __syncthreads();
    uint32_t mine = 0xffffffffu;
    const bool live = row < rows;
    if (live && qg != nullptr) {
        const int32_t i = idx[row];
        mine = i >= 0 && i < p.n_tokens ? qg[i] : 0u;
    }
    const uint32_t w_any = __reduce_or_sync(0xffffffffu, live ? mine : 0u);
    if (lane == 0) atomicOr(&any_row, w_any);
    const uint32_t same = __match_any_sync(0xffffffffu, mine) & __ballot_sync(0xffffffffu, live);
    if (live && lane == __ffs(same) - 1) row_word[atomicAdd(&n_words, 1)] = mine;
    __syncthreads();
    const uint32_t seen_by = any_row;
    const int32_t tiles = a.n_pre + a.n_own;
    uint16_t* out = list + ((int64_t)b * a.units_cap + unit) * tiles;
    int32_t n = 0;
    for (int32_t t0 = 0; t0 < tiles; t0 += kVisThreads) {
        const int32_t n_t = min(kVisThreads, tiles - t0);
        // union and intersection of each tile's key sets (warp per tile, 4 keys per lane)
        for (int32_t e = warp; e < n_t; e += kVisThreads / 32) {
            const int32_t t = t0 + e;
            const bool pre = t < a.n_pre;
            const uint32_t* src = pre ? p.pg : kg;
            const int32_t key0 = (pre ? t : t - a.n_pre) * kBN + 4 * lane, n_src = pre ? p.n_prefix : p.n_tokens;
            uint32_t w[4], un = 0, in = 0xffffffffu;
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                w[k] = key0 + k < n_src ? (src != nullptr ? src[key0 + k] : 0xffffffffu) : 0u;
                un |= w[k];
                in &= w[k];
            }
            if (unit == 0 && (!pre || b == 0))
                *reinterpret_cast<uint4*>(groups + ((int64_t)(pre ? t : t + b * a.n_own) * kBN + 4 * lane)) =
                    make_uint4(w[0], w[1], w[2], w[3]);
            un = __reduce_or_sync(0xffffffffu, un);
            in = __reduce_and_sync(0xffffffffu, in);
            if (lane == 0) {
                any_of[e] = un;
                all_of[e] = in;
            }
        }
        __syncthreads();
        // thread e: is tile t0 + e seen, and whole by every row?
        const int32_t e = threadIdx.x;
        const bool seen = e < n_t && (any_of[e] & seen_by) != 0;
        bool whole = seen;
        if (seen) {
            const uint32_t in = all_of[e];
            for (int32_t r = 0; r < n_words && whole; ++r) whole = (row_word[r] & in) != 0;
        }
        __syncthreads();
        // compact the seen tiles in order (any_of is free now: the warps' counts)
        const uint32_t vote = __ballot_sync(0xffffffffu, seen);
        if (lane == 0) any_of[warp] = __popc(vote);
        __syncthreads();
        int32_t at = n, all = 0;
        for (int w = 0; w < kVisThreads / 32; ++w) {
            at += w < warp ? (int32_t)any_of[w] : 0;
            all += (int32_t)any_of[w];
        }
        if (seen) out[at + __popc(vote & ((1u << lane) - 1u))] = (uint16_t)((t0 + e) | (whole ? 0 : 0x8000));
        n += all;
        __syncthreads();
    }
    if (threadIdx.x == 0) {
        if (n == 0) out[0] = 0x8000;             // a unit that sees nothing runs one masked tile: zeros
        steps[b * a.units_cap + unit] = max(n, 1);
    }
}

// 128 consecutive columns as four loads and one wait in one statement: a thread of a 512-thread CTA is
// compiled for 128 registers outside the softmax branch, less than a single 128-column load needs.
#define FXR_TMEM_LD4X32(taddr, r)                                                                                     \
    asm volatile(                                                                                                     \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"                                                                    \
        "%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,"                                                      \
        "%16,%17,%18,%19,%20,%21,%22,%23,%24,%25,%26,%27,%28,%29,%30,%31}, [%128];\n\t"                               \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"                                                                    \
        "%32,%33,%34,%35,%36,%37,%38,%39,%40,%41,%42,%43,%44,%45,%46,%47,"                                            \
        "%48,%49,%50,%51,%52,%53,%54,%55,%56,%57,%58,%59,%60,%61,%62,%63}, [%129];\n\t"                               \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"                                                                    \
        "%64,%65,%66,%67,%68,%69,%70,%71,%72,%73,%74,%75,%76,%77,%78,%79,"                                            \
        "%80,%81,%82,%83,%84,%85,%86,%87,%88,%89,%90,%91,%92,%93,%94,%95}, [%130];\n\t"                               \
        "tcgen05.ld.sync.aligned.32x32b.x32.b32 {"                                                                    \
        "%96,%97,%98,%99,%100,%101,%102,%103,%104,%105,%106,%107,%108,%109,%110,%111,"                                \
        "%112,%113,%114,%115,%116,%117,%118,%119,%120,%121,%122,%123,%124,%125,%126,%127}, [%131];\n\t"               \
        "tcgen05.wait::ld.sync.aligned;"                                                                              \
        : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]), "=r"(r[4]), "=r"(r[5]), "=r"(r[6]), "=r"(r[7]),             \
          "=r"(r[8]), "=r"(r[9]), "=r"(r[10]), "=r"(r[11]), "=r"(r[12]), "=r"(r[13]), "=r"(r[14]), "=r"(r[15]),       \
          "=r"(r[16]), "=r"(r[17]), "=r"(r[18]), "=r"(r[19]), "=r"(r[20]), "=r"(r[21]), "=r"(r[22]), "=r"(r[23]),     \
          "=r"(r[24]), "=r"(r[25]), "=r"(r[26]), "=r"(r[27]), "=r"(r[28]), "=r"(r[29]), "=r"(r[30]), "=r"(r[31]),     \
          "=r"(r[32]), "=r"(r[33]), "=r"(r[34]), "=r"(r[35]), "=r"(r[36]), "=r"(r[37]), "=r"(r[38]), "=r"(r[39]),     \
          "=r"(r[40]), "=r"(r[41]), "=r"(r[42]), "=r"(r[43]), "=r"(r[44]), "=r"(r[45]), "=r"(r[46]), "=r"(r[47]),     \
          "=r"(r[48]), "=r"(r[49]), "=r"(r[50]), "=r"(r[51]), "=r"(r[52]), "=r"(r[53]), "=r"(r[54]), "=r"(r[55]),     \
          "=r"(r[56]), "=r"(r[57]), "=r"(r[58]), "=r"(r[59]), "=r"(r[60]), "=r"(r[61]), "=r"(r[62]), "=r"(r[63]),     \
          "=r"(r[64]), "=r"(r[65]), "=r"(r[66]), "=r"(r[67]), "=r"(r[68]), "=r"(r[69]), "=r"(r[70]), "=r"(r[71]),     \
          "=r"(r[72]), "=r"(r[73]), "=r"(r[74]), "=r"(r[75]), "=r"(r[76]), "=r"(r[77]), "=r"(r[78]), "=r"(r[79]),     \
          "=r"(r[80]), "=r"(r[81]), "=r"(r[82]), "=r"(r[83]), "=r"(r[84]), "=r"(r[85]), "=r"(r[86]), "=r"(r[87]),     \
          "=r"(r[88]), "=r"(r[89]), "=r"(r[90]), "=r"(r[91]), "=r"(r[92]), "=r"(r[93]), "=r"(r[94]), "=r"(r[95]),     \
          "=r"(r[96]), "=r"(r[97]), "=r"(r[98]), "=r"(r[99]), "=r"(r[100]), "=r"(r[101]), "=r"(r[102]), "=r"(r[103]), \
          "=r"(r[104]), "=r"(r[105]), "=r"(r[106]), "=r"(r[107]), "=r"(r[108]), "=r"(r[109]), "=r"(r[110]), "=r"(r[111]),\
          "=r"(r[112]), "=r"(r[113]), "=r"(r[114]), "=r"(r[115]), "=r"(r[116]), "=r"(r[117]), "=r"(r[118]), "=r"(r[119]),\
          "=r"(r[120]), "=r"(r[121]), "=r"(r[122]), "=r"(r[123]), "=r"(r[124]), "=r"(r[125]), "=r"(r[126]), "=r"(r[127])\
        : "r"(taddr), "r"((taddr) + 32u), "r"((taddr) + 64u), "r"((taddr) + 96u)                                      \
        : "memory")

// Orders this thread's shared-memory writes before the asynchronous proxy's reads of them.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

// ---- pieces of the tile kernel --------------------------------------------------------------------
// Maximum that is NaN where an operand is (a NaN score must reach its row).
__device__ __forceinline__ float max3n(float a, float b, float c) {
    float d;
    asm("max.NaN.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}
__device__ __forceinline__ float max2n(float a, float b) {
    float d;
    asm("max.NaN.f32 %0, %1, %2;" : "=f"(d) : "f"(a), "f"(b));
    return d;
}

// Scratch slot of the part that CTA c holds of a unit whose iterations start at i0: its first item
// unless the unit starts inside c's range behind others.
__device__ __forceinline__ int64_t part_at(int32_t i0, int32_t per, int32_t c, int t) {
    const int k = i0 > c * per ? 1 : 0;
    return (((int64_t)c * 2 + k) * 2 + t) * kPartFloats;
}

// The last part of a unit to arrive combines row r of tile t over all parts, in key order.
template <typename T>
__device__ __forceinline__ void combine_parts(const float* part, int32_t i0, int32_t per, int32_t c0, int32_t c1, int t, int r,
                                              T* out_row) {
    float top = -INFINITY;
    for (int32_t c = c0; c <= c1; ++c) top = fmaxf(top, __ldcg(part + part_at(i0, per, c, t) + kBM * kD + r));
    if (top == -INFINITY) top = 0.f;
    float l = 0.f;
    for (int32_t c = c0; c <= c1; ++c) {
        const float* q = part + part_at(i0, per, c, t) + kBM * kD + r;
        l += ex2_approx(__ldcg(q) - top) * __ldcg(q + kBM);
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
#pragma unroll 1
    for (int h = 0; h < 4; ++h) {
        float acc[32];
#pragma unroll
        for (int k = 0; k < 32; ++k) acc[k] = 0.f;
        for (int32_t c = c0; c <= c1; ++c) {
            const float* q = part + part_at(i0, per, c, t);
            const float w = ex2_approx(__ldcg(q + kBM * kD + r) - top);
#pragma unroll
            for (int k = 0; k < 8; ++k) {
                const float4 x = __ldcg(reinterpret_cast<const float4*>(q) + (h * 8 + k) * kBM + r);
                acc[4 * k] += w * x.x;
                acc[4 * k + 1] += w * x.y;
                acc[4 * k + 2] += w * x.z;
                acc[4 * k + 3] += w * x.w;
            }
        }
        if (out_row != nullptr) {
            uint4* dst = reinterpret_cast<uint4*>(out_row + 32 * h);
#pragma unroll
            for (int k = 0; k < 4; ++k)
                dst[k] = make_uint4(StoreT<T>::pack2(acc[8 * k] * inv, acc[8 * k + 1] * inv),
                                    StoreT<T>::pack2(acc[8 * k + 2] * inv, acc[8 * k + 3] * inv),
                                    StoreT<T>::pack2(acc[8 * k + 4] * inv, acc[8 * k + 5] * inv),
                                    StoreT<T>::pack2(acc[8 * k + 6] * inv, acc[8 * k + 7] * inv));
        }
    }
}

// End of an item that is part of a unit: its O rows, maxima and sums go to scratch, O is released,
// and the warp whose arrival completes the unit combines its 32 rows. Out of line, as in the 16-bit
// kernel, so that the step loop around it keeps its code.
template <typename T>
__device__ __noinline__ void cut_epilogue(float* part, int32_t* counters, int32_t per, const Item* it, int t, int r, int warp,
                                          uint32_t tO, float m_run, float l_run, uint32_t ofree, T* out_row) {
    const int32_t c = (int32_t)blockIdx.x, i0 = it->i0, c_first = it->c_first, c_last = it->c_last;
    float* slot = part + part_at(i0, per, c, t);
#pragma unroll 1
    for (int h = 0; h < 4; ++h) {
        uint32_t o[32];
        FXR_TMEM_LD32(tO + h * 32u, o);
#pragma unroll
        for (int k = 0; k < 8; ++k)
            reinterpret_cast<float4*>(slot)[(h * 8 + k) * kBM + r] =
                make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                            __uint_as_float(o[4 * k + 3]));
    }
    slot[kBM * kD + r] = m_run;
    slot[kBM * kD + kBM + r] = l_run;
    tc_fence_before();
    mbar_arrive(ofree);
    __threadfence();
    __syncwarp();
    int32_t before = 0;
    if (lane_id() == 0) before = atom_add_acq_rel_gpu(counters + c_last * kPartWarps + warp, 1);
    before = __shfl_sync(0xffffffffu, before, 0);
    if (before != c_last - c_first) return;
    if (lane_id() == 0) counters[c_last * kPartWarps + warp] = 0;   // for the next launch
    __threadfence();
    combine_parts<T>(part, i0, per, c_first, c_last, t, r, out_row);
}

template <typename T, int F>
__global__ void __launch_bounds__(kTileThreads, 1) tile_kernel(const __grid_constant__ TileMaps maps,
                                                               const __grid_constant__ TileParams a) {
    extern __shared__ uint8_t smem_raw[];
    const uint32_t raw = smem_u32(smem_raw);
    const uint32_t base = (raw + 1023u) & ~1023u;
    uint8_t* gbase = smem_raw + (base - raw);
    auto bar = [&](uint32_t i) { return base + kSmBar + 8u * i; };
    volatile uint32_t* tmem_slot = reinterpret_cast<volatile uint32_t*>(gbase + kSmTmem);
    volatile int* abort = reinterpret_cast<volatile int*>(gbase + kSmAbort);
    auto item_at = [&](uint32_t k) { return reinterpret_cast<Item*>(gbase + kSmItem + (k & 1) * 160); };
    volatile uint32_t* info = reinterpret_cast<volatile uint32_t*>(gbase + kSmInfo);
    const int warp = threadIdx.x >> 5;
    const uint32_t lane = lane_id();
    const Params& p = a.p;

    if (threadIdx.x == 0) {
        mbar_init(bar(kQFull), 1);
        mbar_init(bar(kQEmpty), 1);
        for (int s = 0; s < kRaws; ++s) {
            mbar_init(bar(kRawFull + s), 1);
            mbar_init(bar(kRawEmpty + s), 4);
        }
        for (int s = 0; s < kTiles; ++s) {
            mbar_init(bar(kFull + s), 4);
            mbar_init(bar(kEmpty + s), 1);
        }
        for (int t = 0; t < 2; ++t) {
            mbar_init(bar(kSFull + t), 1);
            mbar_init(bar(kPHalf0 + t), kBM);
            mbar_init(bar(kPHalf1 + t), kBM);
            mbar_init(bar(kPVDone + t), 1);
            mbar_init(bar(kOFree + t), kBM);
            mbar_init(bar(kItemFull + t), 1);
            mbar_init(bar(kItemEmpty + t), kItemReaders);
        }
        mbar_init(bar(kDrain), 1);
        *abort = 0;
        fence_mbar_init();
    }
    if (warp == kMmaWarp) {
        tmem_alloc(smem_u32((const void*)tmem_slot), kTmemColumns);
        tmem_relinquish();
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    // iterations per CTA when units are cut, 0 for whole units; the same on every thread
    const int32_t n_steps = a.n_pre + a.n_own;
    int32_t per = 0;
    int64_t total = 0;
    int32_t n_units = 0;
    {
#pragma unroll
        for (int b = 0; b < kMaxBatch; ++b)
            if (b < p.n_streams) {
                const int32_t units = (max(0, min(*p.s[b].count, p.max_rows)) + kUnitRows - 1) / kUnitRows;
                n_units += units * p.n_heads;
                if (a.steps == nullptr) {
                    total += (int64_t)units * p.n_heads * n_steps;
                } else {
                    int32_t sum = 0;
                    for (int32_t u = (int32_t)lane; u < units; u += 32) sum += a.steps[b * a.units_cap + u];
                    total += (int64_t)__reduce_add_sync(0xffffffffu, sum) * p.n_heads;
                }
            }
        const int32_t grid = (int32_t)gridDim.x;
        const int64_t each = (total + grid - 1) / grid;
        const float avg = n_units > 0 ? (float)total / (float)n_units : 0.f;
        const float whole = (float)((n_units + grid - 1) / grid) * (avg + kItemSteps);
        const float cut = (float)each + kItemSteps * ((float)each / fmaxf(avg, 1.f) + 1.f) + 2.f * kCutSteps;
        if (cut < whole && each < (1 << 28) && total < (1ll << 31)) per = (int32_t)each;
    }

    if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        // ---------------- converters: one row of the tile per thread ----------------
        auto wwait = [&](uint32_t b_, uint32_t par_) -> bool { return __all_sync(0xffffffffu, mbar_wait(b_, par_, abort)); };
        const uint32_t r = (uint32_t)(warp - kConvWarp) * 32 + lane, x = r & 7;
        constexpr uint32_t fmt16 = StoreT<T>::kUmmaFormat;
        uint32_t in = 0, step = 0;     // tiles converted, steps
        bool ok = true;
        for (uint32_t k = 0; ok; ++k) {
            if (!wwait(bar(kItemFull + (k & 1)), (k >> 1) & 1)) break;
            const Item* it = item_at(k);
            const int32_t n = it->n, s0 = it->s0;
            if (n == 0) break;
            const uint16_t* list = it->list;
            const T* own_k = static_cast<const T*>(it->ks);
            const T* own_v = static_cast<const T*>(it->vs);
            const T* pre_k = static_cast<const T*>(p.prefix.ks) + (int64_t)it->head * p.prefix.ld_scale;
            const T* pre_v = static_cast<const T*>(p.prefix.vs) + (int64_t)it->head * p.prefix.ld_scale;
            uint32_t word, next_word = list ? list[s0] : (uint32_t)s0;
            // the next step's scales are on their way, as bits, while this step is converted
            uint16_t next_k, next_v;
            auto scales = [&](uint32_t w, uint16_t& k_, uint16_t& v_) {
                const int32_t tile = (int32_t)(list ? w & 0x7fffu : w);
                const bool pre = tile < a.n_pre;
                const int32_t key = (pre ? tile : tile - a.n_pre) * kBN + (int32_t)r;
                const bool in_src = key < (pre ? p.n_prefix : p.n_tokens);
                k_ = v_ = 0;
                if (in_src) {
                    k_ = __ldg(reinterpret_cast<const uint16_t*>(pre ? pre_k : own_k) + key);
                    v_ = __ldg(reinterpret_cast<const uint16_t*>(pre ? pre_v : own_v) + key);
                }
            };
            scales(next_word, next_k, next_v);
            for (int32_t j = 0; ok && j < n; ++j, ++step) {
                word = next_word;
                float sk = StoreT<T>::unpack2(next_k).x, sv = StoreT<T>::unpack2(next_v).x;
                if (j + 1 < n) {
                    next_word = list ? list[s0 + j + 1] : (uint32_t)(s0 + j + 1);
                    scales(next_word, next_k, next_v);
                }
                // a row that is not finite: its scores are NaN, its V counts as zeros
                if (!finite(sv) || !finite(sk)) sk = __uint_as_float(0x7fc00000u);
                if (!finite(sv)) sv = 0.f;
#pragma unroll 1
                for (int kv = 0; kv < 2; ++kv, ++in) {
                    const uint32_t rs = in % kRaws, ts = in % kTiles;
                    if (!wwait(bar(kRawFull + rs), (in / kRaws) & 1)) { ok = false; break; }
                    const uint32_t src = base + kSmRaw + rs * kSpan + r * 128;
                    const uint32_t dst = base + kSmTiles + ts * kTile + r * 128;
                    const float f = kv == 0 ? sk : sv;
                    if (kv == 0 && r == 0) {
                        const int32_t tile = (int32_t)(list ? word & 0x7fffu : word);
                        const bool pre = tile < a.n_pre;
                        const int32_t left = pre ? p.n_prefix - tile * kBN : p.n_tokens - (tile - a.n_pre) * kBN;
                        info[step & 3] = (uint32_t)tile | ((uint32_t)min(left, kBN) << 16) | (list && (word & 0x8000u) ? kMixed : 0u);
                    }
                    uint4 q[8];
#pragma unroll
                    for (uint32_t c = 0; c < 8; ++c) q[c] = lds128(src + ((c ^ x) << 4));
                    if (in >= kTiles && !wwait(bar(kEmpty + ts), (in / kTiles - 1) & 1)) { ok = false; break; }
                    auto convert = [&](auto dec) {
                        dec.scale(StoreT<T>::pack2(f, f));
#pragma unroll
                        for (uint32_t c = 0; c < 8; ++c) {
                            uint4 lo, hi;
                            q8::decode16(q[c], dec, lo, hi);
                            if (c == 7) {        // the codes are in registers: their buffer is free
                                __syncwarp();
                                if (lane == 0) mbar_arrive(bar(kRawEmpty + rs));
                            }
                            const uint32_t d = dst + (c >> 2) * kSpan;
                            sts128(d + (((2 * (c & 3)) ^ x) << 4), lo);
                            sts128(d + (((2 * (c & 3) + 1) ^ x) << 4), hi);
                        }
                    };
                    if constexpr (F == q8::kE4m3 && fmt16 == 1) {
                        if (__all_sync(0xffffffffu, !(f >= q8::kSmallScale))) convert(q8::SmallScaleDecoder{});
                        else convert(q8::Decoder<T, F>{});
                    } else {
                        convert(q8::Decoder<T, F>{});
                    }
                    fence_async_smem();      // the tensor core reads the tile through the async proxy
                    __syncwarp();
                    if (lane == 0) mbar_arrive(bar(kFull + ts));
                }
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kItemEmpty + (k & 1)));
        }
    } else if (warp >= kProducerWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        if (warp == kProducerWarp) {
            if (lane == 0) {
                // ---------------- TMA producer ----------------
                uint32_t out = 0, q_it = 0;
                bool ok = true;
                auto load = [&](const CUtensorMap* tm, int32_t head, int32_t key0) -> bool {
                    const uint32_t rs = out % kRaws;
                    if (out >= kRaws && !mbar_wait(bar(kRawEmpty + rs), (out / kRaws - 1) & 1, abort)) return false;
                    mbar_arrive_expect_tx(bar(kRawFull + rs), kSpan);
                    tma_load_2d(base + kSmRaw + rs * kSpan, tm, bar(kRawFull + rs), head * kD, key0);
                    ++out;
                    return true;
                };
                for (uint32_t k = 0; ok; ++k) {
                    if (!mbar_wait(bar(kItemFull + (k & 1)), (k >> 1) & 1, abort)) break;
                    const Item* it = item_at(k);
                    const int32_t n = it->n, s0 = it->s0, head = it->head;
                    if (n == 0) break;
                    if (q_it > 0 && !mbar_wait(bar(kQEmpty), (q_it - 1) & 1, abort)) break;
                    mbar_arrive_expect_tx(bar(kQFull), 2 * kTile);
                    for (int t = 0; t < 2; ++t) {
                        const uint32_t dq = base + kSmQ + t * kTile;
                        tma_load_2d(dq, it->tq, bar(kQFull), head * kD, it->row0 + t * kBM);
                        tma_load_2d(dq + kSpan, it->tq, bar(kQFull), head * kD + 64, it->row0 + t * kBM);
                    }
                    ++q_it;
                    for (int32_t j = 0; ok && j < n; ++j) {
                        const int32_t tile = it->list ? it->list[s0 + j] & 0x7fff : s0 + j;
                        const bool pre = tile < a.n_pre;
                        const int32_t key0 = (pre ? tile : tile - a.n_pre) * kBN;
                        ok = load(pre ? &maps.pk : it->tk, head, key0) && load(pre ? &maps.pv : it->tv, head, key0);
                    }
                    if (ok) mbar_arrive(bar(kItemEmpty + (k & 1)));
                }
                if (*abort) {
                    if (q_it > 0) attn::mbar_wait_drain(bar(kQFull), (q_it - 1) & 1);
                    for (uint32_t e = out > kRaws ? out - kRaws : 0; e < out; ++e)
                        attn::mbar_wait_drain(bar(kRawFull + e % kRaws), (e / kRaws) & 1);
                }
            }
        } else if (warp == kMmaWarp) {
            if (lane == 0) {
                // ---------------- MMA issuer (order and waits of the 16-bit kernel) ----------------
                constexpr uint32_t fmt = StoreT<T>::kUmmaFormat;
                constexpr uint32_t idesc_qk = make_idesc_f16(fmt, 0, kBM, kBN);
                constexpr uint32_t idesc_pv = make_idesc_f16(fmt, 1, kBM, kD);
                uint32_t acq = 0, rel = 0, q_it = 0, g = 0, done = 0;
                bool ok = true, issued = false;
                auto wait = [&](uint32_t b_, uint32_t par_) { return mbar_wait_spin(b_, par_, abort); };
                auto acquire = [&]() -> uint32_t {
                    const uint32_t st = acq % kTiles;
                    if (!wait(bar(kFull + st), (acq / kTiles) & 1)) return 0;
                    ++acq;
                    return base + kSmTiles + st * kTile;
                };
                auto release = [&]() {
                    umma_commit(bar(kEmpty + rel % kTiles));
                    ++rel;
                };
                auto qk = [&](int t, uint32_t sK) {
                    const uint64_t dq = smem_desc_sw128(base + kSmQ + t * kTile, 16, 1024);
                    const uint64_t dk = smem_desc_sw128(sK, 16, 1024);
#pragma unroll
                    for (int k = 0; k < kD / 16; ++k) {
                        const uint64_t off = ((k >> 2) * kSpan + (k & 3) * 32u) >> 4;
                        umma_ss(tmem + kColS + t * 128u, dq + off, dk + off, idesc_qk, k > 0 ? 1u : 0u);
                    }
                    umma_commit(bar(kSFull + t));
                };
                auto pv = [&](int t, uint32_t sV, int h, bool acc) {
                    const uint64_t dv = smem_desc_sw128(sV, kSpan, 1024);
#pragma unroll
                    for (int k = 4 * h; k < 4 * h + 4; ++k)
                        umma_ts(tmem + kColO + t * 128u, tmem + kColS + t * 128u + k * 8u, dv + (uint64_t)((k * 2048u) >> 4),
                                idesc_pv, (acc || k > 0) ? 1u : 0u);
                };
                for (uint32_t it_no = 0; ok; ++it_no) {
                    if (!wait(bar(kItemFull + (it_no & 1)), (it_no >> 1) & 1)) break;
                    const int32_t n = item_at(it_no)->n;
                    mbar_arrive(bar(kItemEmpty + (it_no & 1)));
                    if (n == 0) break;
                    if (!wait(bar(kQFull), q_it & 1)) break;
                    ++q_it;
                    if (g > 0 && (!wait(bar(kPVDone + 0), (g - 1) & 1) || !wait(bar(kPVDone + 1), (g - 1) & 1))) break;
                    uint32_t sK = acquire();
                    if (!sK) break;
                    tc_fence_after();
                    issued = true;
                    qk(0, sK);
                    qk(1, sK);
                    release();
                    if (n == 1) umma_commit(bar(kQEmpty));
                    for (int32_t j = 0; j < n; ++j, ++g) {
                        const uint32_t sV = acquire();
                        if (!sV) { ok = false; break; }
                        const bool more = j + 1 < n;
#pragma unroll 1
                        for (int t = 0; t < 2; ++t) {
                            if (!wait(bar(kPHalf0 + t), g & 1)) { ok = false; break; }
                            if (j == 0 && done > 0 && !wait(bar(kOFree + t), (done - 1) & 1)) { ok = false; break; }
                            tc_fence_after();
                            pv(t, sV, 0, j > 0);
                            if (!wait(bar(kPHalf1 + t), g & 1)) { ok = false; break; }
                            tc_fence_after();
                            pv(t, sV, 1, true);
                            umma_commit(bar(kPVDone + t));
                            if (t == 1) release();
                            if (more) {
                                if (t == 0) {
                                    sK = acquire();
                                    if (!sK) { ok = false; break; }
                                }
                                // S_t(j+1) overwrites P_t(j): O_t += P_t(j) V_j has to be complete
                                if (!wait(bar(kPVDone + t), g & 1)) { ok = false; break; }
                                tc_fence_after();
                                qk(t, sK);
                                if (t == 1) {
                                    release();
                                    if (j + 2 == n) umma_commit(bar(kQEmpty));
                                }
                            }
                        }
                        if (!ok) break;
                    }
                    ++done;
                }
                if (*abort && issued) {
                    umma_commit(bar(kDrain));
                    attn::mbar_wait_drain(bar(kDrain), 0);
                }
            }
        } else if (warp == kSchedWarp) {
            // ---------------- scheduler ----------------
            const int32_t grid = (int32_t)gridDim.x, c = (int32_t)blockIdx.x;
            int64_t cur = per > 0 ? (int64_t)c * per : c;
            const int64_t end = per > 0 ? min(total, cur + per) : n_units;
            for (uint32_t k = 0;; ++k) {
                const bool more = cur < end;
                // the unit: stream, head, first row, steps, first iteration
                int32_t b = -1, rows = 0, head = 0, unit = 0, cnt = n_steps;
                int64_t rest = cur, i0 = cur;
                if (more) {
                    int32_t units = 1;
#pragma unroll
                    for (int s = 0; s < kMaxBatch; ++s)
                        if (b < 0 && s < p.n_streams) {
                            const int32_t m = max(0, min(*p.s[s].count, p.max_rows));
                            const int32_t u = (m + kUnitRows - 1) / kUnitRows;
                            int64_t span = u;             // per head, in units or iterations
                            if (per > 0) {
                                if (a.steps == nullptr) {
                                    span = (int64_t)u * n_steps;
                                } else {
                                    int32_t sum = 0;
                                    for (int32_t e = (int32_t)lane; e < u; e += 32) sum += a.steps[s * a.units_cap + e];
                                    span = __reduce_add_sync(0xffffffffu, sum);
                                }
                            }
                            if (rest < span * p.n_heads) {
                                b = s;
                                rows = m;
                                units = u;
                                head = (int32_t)(rest / span);
                                rest -= head * span;
                            } else {
                                rest -= span * p.n_heads;
                            }
                        }
                    if (per == 0) {
                        unit = (int32_t)rest;
                        if (a.steps) cnt = a.steps[b * a.units_cap + unit];
                    } else if (a.steps == nullptr) {
                        unit = (int32_t)(rest / n_steps);
                        i0 = cur - (rest - (int64_t)unit * n_steps);
                    } else {
                        int32_t left = (int32_t)rest;     // iterations into the head's units
                        bool found = false;
                        for (int32_t e0 = 0; e0 < units && !found; e0 += 32) {
                            const int32_t mine = e0 + (int32_t)lane < units ? a.steps[b * a.units_cap + e0 + lane] : 0;
                            int32_t upto = mine;
#pragma unroll
                            for (int o = 1; o < 32; o <<= 1) {
                                const int32_t x = __shfl_up_sync(0xffffffffu, upto, o);
                                if ((int)lane >= o) upto += x;
                            }
                            const uint32_t hit = __ballot_sync(0xffffffffu, left < upto);
                            if (hit) {
                                const int f = __ffs(hit) - 1;
                                unit = e0 + f;
                                cnt = __shfl_sync(0xffffffffu, mine, f);
                                i0 = cur - (left - (__shfl_sync(0xffffffffu, upto, f) - cnt));
                                found = true;
                            } else {
                                left -= __shfl_sync(0xffffffffu, upto, 31);
                            }
                        }
                    }
                }
                if (k >= 2 && !__all_sync(0xffffffffu, mbar_wait(bar(kItemEmpty + (k & 1)), ((k >> 1) - 1) & 1, abort))) break;
                Item* it = item_at(k);
                const int32_t s0 = per > 0 ? (int32_t)(cur - i0) : 0;
                const int32_t n = !more ? 0 : per > 0 ? min(cnt - s0, (int32_t)(end - cur)) : cnt;
                if (lane == 0) {
                    it->n = n;
                    if (n > 0) {
#pragma unroll
                        for (int s = 0; s < kMaxBatch; ++s)
                            if (s == b) {
                                it->tq = &maps.q[s];
                                it->tk = &maps.k[s];
                                it->tv = &maps.v[s];
                                it->ks = static_cast<const T*>(p.s[s].c.ks) + (int64_t)head * p.s[s].c.ld_scale;
                                it->vs = static_cast<const T*>(p.s[s].c.vs) + (int64_t)head * p.s[s].c.ld_scale;
                                it->idx = p.s[s].idx;
                                it->qg = p.s[s].qg;
                                it->out = p.s[s].out;
                                if (*p.s[s].count > p.max_rows && unit == 0 && head == 0) atomicOr(&g_error_word, kErrBounds);
                            }
                        it->s0 = s0;
                        it->head = head;
                        it->row0 = unit * kUnitRows;
                        it->rows = rows;
                        it->list = a.steps ? a.list + ((int64_t)b * a.units_cap + unit) * n_steps : nullptr;
                        it->cut = n < cnt;
                        it->i0 = (int32_t)i0;
                        it->c_first = per > 0 ? (int32_t)(i0 / per) : 0;
                        it->c_last = per > 0 ? (int32_t)((i0 + cnt - 1) / per) : 0;
                        it->stream = b;
                    }
                    mbar_arrive(bar(kItemFull + (k & 1)));
                }
                __syncwarp();
                if (n == 0) break;
                cur += per > 0 ? n : grid;
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 %0;" ::"n"(kRegsSoftmax));
        // ---------------- softmax / epilogue: one thread per query row ----------------
        auto wwait = [&](uint32_t b_, uint32_t par_) -> bool { return __all_sync(0xffffffffu, mbar_wait(b_, par_, abort)); };
        const int t = warp >> 2;
        const int r = ((warp & 3) << 5) | (int)lane;
        const uint32_t lane_off = (uint32_t)((warp & 3) * 32) << 16;
        const uint32_t tS = tmem + lane_off + kColS + t * 128u, tO = tmem + lane_off + kColO + t * 128u;
        const float c = p.scale_log2;
        const float2 c2 = make_float2(c, c);
        volatile uint32_t* my_groups = reinterpret_cast<volatile uint32_t*>(gbase + kSmGroup) + threadIdx.x;
        uint32_t s_it = 0;
        bool ok = true;
        for (uint32_t k = 0; ok; ++k) {
            if (!wwait(bar(kItemFull + (k & 1)), (k >> 1) & 1)) break;
            const Item* it = item_at(k);
            const int32_t n = it->n;
            if (n == 0) break;
            const bool live = it->row0 + t * kBM + r < it->rows;
            if (it->list != nullptr) {
                uint32_t w = 0;
                if (live) {
                    w = 0xffffffffu;
                    if (it->qg != nullptr) {
                        const int32_t i = it->idx[it->row0 + t * kBM + r];
                        w = i >= 0 && i < p.n_tokens ? it->qg[i] : 0u;
                    }
                }
                *my_groups = w;
            }
            float m_run = -INFINITY, l_run = 0.f;
            for (int32_t j = 0; j < n; ++j, ++s_it) {
                if (!wwait(bar(kSFull + t), s_it & 1)) { ok = false; break; }
                tc_fence_after();
                uint32_t s[128];
                FXR_TMEM_LD4X32(tS, s);
                const uint32_t what = info[s_it & 3];
                const bool mixed = (what & kMixed) != 0;
                if (mixed) {
                    const int32_t tile = (int32_t)(what & 0xffffu);
                    const uint4* kg = reinterpret_cast<const uint4*>(a.groups) +
                                      (int64_t)(tile < a.n_pre ? tile : tile + it->stream * a.n_own) * (kBN / 4);
                    const uint32_t qg = *my_groups;
#pragma unroll
                    for (int q = 0; q < 32; ++q) {
                        const uint4 w = __ldg(kg + q);
                        s[4 * q] = (w.x & qg) ? s[4 * q] : 0xff800000u;
                        s[4 * q + 1] = (w.y & qg) ? s[4 * q + 1] : 0xff800000u;
                        s[4 * q + 2] = (w.z & qg) ? s[4 * q + 2] : 0xff800000u;
                        s[4 * q + 3] = (w.w & qg) ? s[4 * q + 3] : 0xff800000u;
                    }
                } else {
                    const int32_t left = (int32_t)((what >> 16) & 0xffu);
                    if (left < kBN) {
#pragma unroll
                        for (int cc = 0; cc < 128; ++cc)
                            if (cc >= left) s[cc] = 0xff800000u;
                    }
                }
                float mp[8];
#pragma unroll
                for (int q = 0; q < 8; ++q) mp[q] = max2n(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1]));
#pragma unroll
                for (int i = 1; i < 8; ++i)
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        mp[q] = max3n(mp[q], __uint_as_float(s[16 * i + 2 * q]), __uint_as_float(s[16 * i + 2 * q + 1]));
                const float mx = max3n(max3n(mp[0], mp[1], mp[2]), max3n(mp[3], mp[4], mp[5]), max2n(mp[6], mp[7])) * c;
                if (mx != mx) l_run = mx;        // a NaN score: the row is NaN
                if (j == 0) {
                    m_run = mx;
                } else if (__any_sync(0xffffffffu, live && mx > m_run + attn2::kRescaleThreshold)) {
                    // O_t has no product in flight: S_t(j) was issued after O_t += P_t(j-1) V completed
                    const float m_new = fmaxf(m_run, mx);
                    const float alpha = m_new == m_run ? 1.f : ex2_approx(m_run - m_new);
                    l_run *= alpha;
                    m_run = m_new;
#pragma unroll 1
                    for (int h = 0; h < 4; ++h) {
                        uint32_t o[32];
                        FXR_TMEM_LD32(tO + h * 32u, o);
#pragma unroll
                        for (int q = 0; q < 32; ++q) o[q] = __float_as_uint(__uint_as_float(o[q]) * alpha);
                        FXR_TMEM_ST32(tO + h * 32u, o);
                    }
                }
                const float nm = m_run == -INFINITY ? 0.f : -m_run;
                const float2 nm2 = make_float2(nm, nm);
                float2 acc[4] = {make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f), make_float2(0.f, 0.f)};
                uint32_t* pk = s;
#pragma unroll
                for (int hh = 0; hh < 2; ++hh) {
                    if (mixed) {
                        // masked scores have to vanish exactly (the polynomial ends at 2^-125)
#pragma unroll
                        for (int q = 32 * hh; q < 32 * hh + 32; ++q) {
                            const float2 x = attn::ffma2(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), c2, nm2);
                            const float2 e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                            acc[q & 3] = attn::fadd2(acc[q & 3], e);
                            pk[q] = StoreT<T>::pack2(e.x, e.y);
                        }
                    } else {
#pragma unroll
                        for (int q = 32 * hh; q < 32 * hh + 32; ++q) {
                            const float2 x = attn::ffma2(make_float2(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1])), c2, nm2);
                            float2 e;
                            if ((q % kPolyPeriod) == kPolyPeriod - 1) e = attn::ex2_poly2(x);
                            else e = make_float2(ex2_approx(x.x), ex2_approx(x.y));
                            acc[q & 3] = attn::fadd2(acc[q & 3], e);
                            pk[q] = StoreT<T>::pack2(e.x, e.y);
                        }
                    }
                    FXR_TMEM_ST32(tS + 32u * hh, (pk + 32 * hh));
                    tc_fence_before();
                    mbar_arrive(bar((hh == 0 ? kPHalf0 : kPHalf1) + t));
                }
                const float2 a01 = attn::fadd2(attn::fadd2(acc[0], acc[1]), attn::fadd2(acc[2], acc[3]));
                l_run += a01.x + a01.y;
            }
            if (!ok) break;
            if (!wwait(bar(kPVDone + t), (s_it - 1) & 1)) break;
            tc_fence_after();
            T* out_row = nullptr;
            if (live) {
                const int32_t i = it->idx[it->row0 + t * kBM + r];
                if (i >= 0 && i < p.n_tokens)
                    out_row = static_cast<T*>(it->out) + (int64_t)i * p.ld_out + (int64_t)it->head * kD;
                else
                    atomicOr(&g_error_word, kErrBounds);
            }
            if (m_run == -INFINITY) l_run = 0.f;      // the row saw nothing
            if (it->cut) {
                cut_epilogue<T>(a.part, a.cnt, per, it, t, r, warp, tO, m_run, l_run, bar(kOFree + t), out_row);
            } else {
                const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t o[32];
                    FXR_TMEM_LD32(tO + h * 32u, o);
                    if (out_row != nullptr) {
                        uint4* dst = reinterpret_cast<uint4*>(out_row + 32 * h);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            dst[q] = make_uint4(
                                StoreT<T>::pack2(__uint_as_float(o[8 * q]) * inv, __uint_as_float(o[8 * q + 1]) * inv),
                                StoreT<T>::pack2(__uint_as_float(o[8 * q + 2]) * inv, __uint_as_float(o[8 * q + 3]) * inv),
                                StoreT<T>::pack2(__uint_as_float(o[8 * q + 4]) * inv, __uint_as_float(o[8 * q + 5]) * inv),
                                StoreT<T>::pack2(__uint_as_float(o[8 * q + 6]) * inv, __uint_as_float(o[8 * q + 7]) * inv));
                    }
                }
                tc_fence_before();
                mbar_arrive(bar(kOFree + t));
            }
            __syncwarp();
            if (lane == 0) mbar_arrive(bar(kItemEmpty + (k & 1)));
        }
    }

    __syncwarp();
    tc_fence_before();
    __syncthreads();
    if (warp == kMmaWarp) {
        tc_fence_after();
        tmem_dealloc(tmem, kTmemColumns);
    }
}

}  // namespace attn8
}  // namespace fxr
