// fxr_attention_q8.cuh — attention of executed rows over the 8-bit spatial cache (sm_100a).
//
//   out[idx[m]] = sum_j p_mj v_j / sum_j p_mj,   p_mj = allow(m, j) * exp(scale * q_m . k_j)
// over the rows of a prefix that every stream of the launch shares and then the stream's own rows;
// allow(m, j) = (q_groups[idx[m]] & k_groups[j]) != 0. A row that sees no key gives zeros.
//
// A key whose K or V scale is not finite (its 16-bit row held an infinity or NaN) makes the rows that
// see it NaN and no others: its score is set to NaN before the mask and its V codes count as zeros.
#pragma once

#include "fxr_attention.cuh"
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
    int32_t slots;
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

}  // namespace attn8
}  // namespace fxr
