// fxr_attention_q8.cuh — attention of executed rows over the 8-bit spatial cache (sm_100a).
//
//   out[idx[m]] = sum_j p_mj v_j / sum_j p_mj,   p_mj = allow(m, j) * exp(scale * q_m . k_j)
// over the rows of a prefix that every stream of the launch shares and then the stream's own rows;
// allow(m, j) = (q_groups[idx[m]] & k_groups[j]) != 0. A row that sees no key gives zeros.
//
// A key whose K or V scale is not valid (its 16-bit row held an infinity or NaN) makes the rows that
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
    int32_t* cnt;                // [own group][n_heads] arrivals, zero between launches
};

// ---------------------------------------------------------------------------------------------
// Few rows per stream: bound by reading the cache once. Work is laid on a line of columns, each the
// keys of one source for one head and one group of 8, 16 or 32 rows: first (head, group of the packed
// rows of all streams) against the prefix, so that the prefix is read once for every group of packed rows
// (16, or 32 where a stream may have more than 16), then (stream, head, group) against the stream's own
// rows. Where there are at least as many
// CTAs as columns, every column is cut into parts of one length, the shortest (in units of 64 keys)
// that gives every part a CTA of its own. Otherwise the line is cut into one range per CTA, and a range
// covers a few items (parts of columns). An item costs its CTA about 6 us besides its keys (queries,
// first copies, exchange, arrival: as long as 700 keys), so ranges that straddle columns are avoided
// where they can be.
// A CTA's 8 or 16 warps walk an item in blocks of 16 keys, each warp with its own running maximum, sum and
// O, so that none waits for another. A warp streams its blocks through a ring in shared memory by
// TMA (4 KB of codes per block: ~130 KB in flight per SM; one lane issues a block's copies, where
// 16-byte asynchronous copies cost every lane eight addresses). The codes
// become 16-bit operands in registers, between shared memory and mma.m16n8k16 with keys, then dims,
// as its 16 rows and queries as its 8 columns (tcgen05 reads its operands from memory and wants 128
// rows; these calls have a few):
//   S^T = K Q^T: a lane holds codes of keys g and g + 8. The order of the 128 dims inside a dot
//     product is free, so it takes 16 consecutive bytes for four steps of 16 dims, and reads Q's
//     fragments in the same order.
//   O^T += V^T P^T: an operand pairs two keys of one dim; one byte permute takes both codes. A lane's
//     rows in the 8 row tiles are 16 consecutive dims. P^T changes from the accumulators' to the
//     operand's layout by an 8 x 8 transpose (movmatrix).
// All operands are f16, whatever the frame's type: it holds the codes exactly, and the codes reach it in
// fewer instructions than bf16. bf16 queries are brought to f16 by a power of two per row (exactly, but
// for elements below 2^-24 of the row's largest). K scales multiply the scores in 32 bits. V scales
// multiply P before its one rounding; the running maximum is that of score + log2(V scale), the weight of
// a key's codes, so that P stays in f16's range whatever the scales are, and a large V that a row hardly
// sees, or not at all, costs the others no precision. (A weight below 2^-14 of the largest is a subnormal of
// f16, off by up to 2^-25 of the largest.) Error against 64 bits: 0.0017 of the outputs' root mean square in
// bf16 and 0.00024 in f16, nearly all of it the rounding of the output.
// Partial results (O, maximum, sum) meet in L2: the last of a row group's parts to arrive combines
// them in key order, so the result does not depend on the order of arrival.
// ---------------------------------------------------------------------------------------------
constexpr int kRowsMax = 32;                   // rows of a group, at most
constexpr int kBlk = 16;                       // keys per block
constexpr int kUnitKeys = 64;                  // columns are cut at multiples of this
constexpr int kMaxRowsPerStream = 32;          // what the launch accepts
constexpr int kGroupsPerStream = kMaxRowsPerStream / 8;
constexpr uint32_t kBlkBytes = kBlk * 128;     // codes of one of K, V (128-byte swizzle)
constexpr uint32_t kRingSlot = 2 * kBlkBytes;
constexpr int kPadRow = 132;                   // floats per O row in the warps' exchange
constexpr uint32_t kQPad = 272;                // bytes per query row
constexpr int kRowsSlotFloats = kRowsMax * kHeadDim + 2 * kRowsMax;
// Shape of the kernel for groups of 8 * NQ rows: up to 16 rows 16 warps with 128 registers and a ring of
// 3 blocks each; 32 rows, whose O alone is 128 registers, 8 warps and rings of 5.
template <int NQ> struct RowsShape {
    static constexpr int rows = 8 * NQ, warps = NQ > 2 ? 8 : 16, threads = 32 * warps, depth = NQ > 2 ? 5 : 3;
    static constexpr uint32_t ring_warp = depth * kRingSlot;
    static constexpr uint32_t at_q = warps * ring_warp;
    static constexpr uint32_t at_m = at_q + rows * kQPad;               // maxima, sums: [rows][warps]; queries' factors
    static constexpr uint32_t at_bar = at_m + (2 * warps + 1) * rows * 4;
    static constexpr uint32_t smem = at_bar + warps * depth * 8 + 1024; // + alignment slack
    static_assert(warps * rows * kPadRow * 4 <= warps * ring_warp, "the exchange fits the ring");
    static_assert(smem <= 230000 && at_bar % 8 == 0, "shared memory budget");
};

// Orders this thread's shared-memory accesses before later ones of the asynchronous proxy.
__device__ __forceinline__ void fence_async_smem() { asm volatile("fence.proxy.async.shared::cta;" ::: "memory"); }

__device__ __forceinline__ uint4 lds128(uint32_t a) {
    uint4 v;
    asm volatile("ld.shared.v4.u32 {%0,%1,%2,%3}, [%4];" : "=r"(v.x), "=r"(v.y), "=r"(v.z), "=r"(v.w) : "r"(a) : "memory");
    return v;
}
__device__ __forceinline__ void sts128(uint32_t a, const uint4& v) {
    asm volatile("st.shared.v4.u32 [%0], {%1,%2,%3,%4};" ::"r"(a), "r"(v.x), "r"(v.y), "r"(v.z), "r"(v.w) : "memory");
}

__device__ __forceinline__ void mma16816(float* d, uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm("mma.sync.aligned.m16n8k16.row.col.f32.f16.f16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
        : "+f"(d[0]), "+f"(d[1]), "+f"(d[2]), "+f"(d[3])
        : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
// 8 x 8 matrix of 16-bit values over a warp, transposed.
__device__ __forceinline__ uint32_t transpose8(uint32_t x) {
    uint32_t y;
    asm("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(y) : "r"(x));
    return y;
}

__device__ __forceinline__ float lg2_approx(float x) {
    float y;
    asm("lg2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}

// Row g of an MMA's 8-row half holds key key_of(g) of the block, and a lane's 16 dims of V are chunk
// key_of(g): in the 128-byte swizzle, neighbouring rows of the fragments then touch different banks.
__device__ __forceinline__ int key_of(int g) { return ((g & 1) << 2) | (g >> 1); }

struct RowsMaps {
    CUtensorMap k[kMaxBatch], v[kMaxBatch], pk, pv;
};

// The launch's division, a function of the counts; each CTA computes it into shared memory.
struct RowsPlan {
    int32_t rows[kMaxBatch];     // of each stream
    int32_t first[kMaxBatch];    // its first packed row
    int32_t group0[kMaxBatch];   // its first own group
    int32_t total;               // rows of all streams
    int32_t gp, go;              // groups: packed rows (0 without a prefix), own
    int32_t up, uo;              // units of a prefix column, of an own column
    int32_t len;                 // units of a part, 0: the line is cut into ranges
    int32_t np, no;              // parts of a prefix column, of an own column
    int32_t per;                 // units of a CTA's range
    int32_t line;                // units in all (the host refuses calls of 2^31 or more)
};

// A column of the line, prefix columns first: its head, group and units.
struct Column {
    int32_t head, group, stream, units, start;
};

template <int R>
__device__ __forceinline__ Column column(const RowsPlan& r, int32_t n_heads, int32_t index) {
    Column c;
    const int32_t pre = n_heads * r.gp;
    if (index < pre) {
        c.head = index / r.gp;
        c.group = index - c.head * r.gp;
        c.stream = -1;
        c.units = r.up;
        c.start = index * r.up;
        return c;
    }
    int32_t e = index - pre;
    c.start = pre * r.up + e * r.uo;
    c.units = r.uo;
    c.stream = 0;
#pragma unroll
    for (int b = 0; b < kMaxBatch - 1; ++b) {
        const int32_t n = n_heads * ((r.rows[b] + R - 1) / R);
        if (c.stream == b && e >= n) {
            e -= n;
            c.stream = b + 1;
        }
    }
    const int32_t groups = (r.rows[c.stream] + R - 1) / R;
    c.head = e / groups;
    c.group = e - c.head * groups;
    return c;
}

// One item: keys [k0, k0 + n_keys) of a column. Kept in shared memory: across the step loop the warps
// have no registers to spare.
struct RowsItem {
    int32_t head, group, stream, live;
    int32_t k0, n_keys, slot;
    int32_t at;                  // ranges: the next unit of the line
};

// The parts of column `index` are `n` consecutive scratch slots from `slot`. (Ranges: part c of column x,
// the one that CTA c holds, is slot x + c, which grows along the line with every cut.)
__device__ __forceinline__ void parts_of(const RowsPlan& r, int32_t n_heads, int32_t index, int32_t& slot, int32_t& n) {
    const int32_t pre = n_heads * r.gp;
    const bool is_pre = index < pre;
    if (r.len > 0) {
        slot = is_pre ? index * r.np : pre * r.np + (index - pre) * r.no;
        n = is_pre ? r.np : r.no;
    } else {
        const int32_t start = is_pre ? index * r.up : pre * r.up + (index - pre) * r.uo;
        const int32_t first = start / r.per;
        slot = index + first;
        n = (start + (is_pre ? r.up : r.uo) - 1) / r.per - first + 1;
    }
}

// Own group (stream b, group g) of head h: every part of its rows, in key order, a warp per row.
template <typename T, int R>
__device__ __noinline__ void rows_combine(const Params& p, const RowsPlan& r, int32_t h, int32_t b, int32_t g) {
    const int lane = threadIdx.x & 31, warps = blockDim.x >> 5;
    for (int32_t m = g * R + (threadIdx.x >> 5); m < min((g + 1) * R, r.rows[b]); m += warps) {
        const int32_t* idx = nullptr;
        void* out_base = nullptr;
#pragma unroll
        for (int k = 0; k < kMaxBatch; ++k)
            if (k == b) {
                idx = p.s[k].idx;
                out_base = p.s[k].out;
            }
        const int32_t i = idx[m];
        // parts: the packed row's prefix column's, then the own column's
        int32_t n_pre = 0, pre_slot = 0, own_slot, n;
        const int32_t pr = r.first[b] + m;
        if (r.gp > 0) parts_of(r, p.n_heads, h * r.gp + pr / R, pre_slot, n_pre);
        const int32_t groups = (r.rows[b] + R - 1) / R;
        parts_of(r, p.n_heads, p.n_heads * (r.gp + r.group0[b]) + h * groups + g, own_slot, n);
        n += n_pre;
        auto slot = [&](int32_t c) {
            return p.part + (int64_t)(c < n_pre ? pre_slot + c : own_slot + c - n_pre) * kRowsSlotFloats;
        };
        auto row_of = [&](int32_t c) { return c < n_pre ? pr % R : m % R; };
        // 32 parts at a time: lane c holds part c's maximum and sum, all lanes 8 parts' positions, every load
        // of a round in flight together (one round trip to L2 for up to 8 parts)
        float top = -INFINITY, l = 0.f;
        float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
        for (int32_t c0 = 0; c0 < n; c0 += 32) {
            float m_c = -INFINITY, l_c = 0.f;
            if (c0 + lane < n) {
                const float* q = slot(c0 + lane) + kRowsMax * kHeadDim + row_of(c0 + lane);
                m_c = __ldcg(q);
                l_c = __ldcg(q + kRowsMax);
            }
            float w = 0.f;
            for (int32_t c1 = c0; c1 < min(n, c0 + 32); c1 += 8) {
                float4 x[8];
#pragma unroll
                for (int k = 0; k < 8; ++k)
                    x[k] = c1 + k < n ? __ldcg(reinterpret_cast<const float4*>(slot(c1 + k) + row_of(c1 + k) * kHeadDim) + lane)
                                      : make_float4(0.f, 0.f, 0.f, 0.f);
                if (c1 == c0) {
                    float t = m_c;
#pragma unroll
                    for (int o = 16; o > 0; o >>= 1) t = fmaxf(t, __shfl_xor_sync(0xffffffffu, t, o));
                    t = fmaxf(t, top);
                    const float base = t == -INFINITY ? 0.f : t, al = ex2_approx(top - base);
                    l *= al;
                    acc = make_float4(acc.x * al, acc.y * al, acc.z * al, acc.w * al);
                    top = t;
                    w = ex2_approx(m_c - base);
                    l += w * l_c;
                }
#pragma unroll
                for (int k = 0; k < 8; ++k) {
                    const float wc = __shfl_sync(0xffffffffu, w, c1 + k - c0);
                    acc.x += wc * x[k].x;
                    acc.y += wc * x[k].y;
                    acc.z += wc * x[k].z;
                    acc.w += wc * x[k].w;
                }
            }
        }
#pragma unroll
        for (int o = 16; o > 0; o >>= 1) l += __shfl_xor_sync(0xffffffffu, l, o);
        if (i < 0 || i >= p.n_tokens) {
            if (lane == 0) atomicOr(&g_error_word, kErrBounds);
            continue;
        }
        const float inv = l == 0.f ? 0.f : 1.0f / l;
        // position 8 d + e of a stored row is dim 16 key_of(e) + d: this lane's e = 4 (lane & 1) + 0..3
        uint16_t* out = reinterpret_cast<uint16_t*>(static_cast<T*>(out_base) + (int64_t)i * p.ld_out + (int64_t)h * kHeadDim) +
                        (lane >> 1);
        const uint32_t lo = StoreT<T>::pack2(acc.x * inv, acc.y * inv), hi = StoreT<T>::pack2(acc.z * inv, acc.w * inv);
        const int e = 4 * (lane & 1);
        out[16 * key_of(e)] = (uint16_t)lo;
        out[16 * key_of(e + 1)] = (uint16_t)(lo >> 16);
        out[16 * key_of(e + 2)] = (uint16_t)hi;
        out[16 * key_of(e + 3)] = (uint16_t)(hi >> 16);
    }
}

// NQ: 8-row tiles of a group.
template <typename T, int F, int NQ>
__global__ void __launch_bounds__(RowsShape<NQ>::threads, 1) rows_kernel(const __grid_constant__ RowsMaps maps, const __grid_constant__ Params p) {
    using Sh = RowsShape<NQ>;
    constexpr int R = Sh::rows, kRowsWarps = Sh::warps, kDepth = Sh::depth;
    extern __shared__ uint8_t smem_raw[];
    uint8_t* smem = smem_raw + ((1024u - (smem_u32(smem_raw) & 1023u)) & 1023u);
    __shared__ RowsPlan r;
    __shared__ RowsItem item;
    __shared__ int abort;
    __shared__ uint32_t ready;                 // own groups whose last part this CTA delivered
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
    const int g = lane >> 2, t = lane & 3;
    const uint32_t base = smem_u32(smem), ring = base + warp * Sh::ring_warp, q_at = base + Sh::at_q;
    const uint32_t bars = base + Sh::at_bar + warp * kDepth * 8;
    uint32_t it = 0;                           // blocks of this warp so far
    if (threadIdx.x == 0) abort = 0;
    if (lane == 0) {
        for (int d = 0; d < kDepth; ++d) mbar_init(bars + 8 * d, 1);
        fence_mbar_init();
    }
    float* xo = reinterpret_cast<float*>(smem);                                     // [warp][R][kPadRow]
    float* xm = reinterpret_cast<float*>(smem + Sh::at_m);                        // [R][warp] maxima, then sums
    pdl_launch_dependents();
    pdl_wait();
    if (warp == 0) {
        int32_t m = 0, c = 0;
#pragma unroll
        for (int b = 0; b < kMaxBatch; ++b)
            if (b == lane && b < p.n_streams) c = *p.s[b].count;
        m = max(0, min(c, p.max_rows));
        if (c > p.max_rows && blockIdx.x == 0) atomicOr(&g_error_word, kErrBounds);
        const int32_t groups = (m + R - 1) / R;
        int32_t rows_to = m, groups_to = groups;      // inclusive sums over the streams
#pragma unroll
        for (int o = 1; o < kMaxBatch; o <<= 1) {
            const int32_t x = __shfl_up_sync(0xffffffffu, rows_to, o), y = __shfl_up_sync(0xffffffffu, groups_to, o);
            if (lane >= o) {
                rows_to += x;
                groups_to += y;
            }
        }
        if (lane < kMaxBatch) {
            r.rows[lane] = m;
            r.first[lane] = rows_to - m;
            r.group0[lane] = groups_to - groups;
        }
        if (lane == kMaxBatch - 1) {
            r.total = rows_to;
            r.go = groups_to;
            r.gp = p.n_prefix > 0 ? (rows_to + R - 1) / R : 0;
            r.up = (p.n_prefix + kUnitKeys - 1) / kUnitKeys;
            r.uo = (p.n_tokens + kUnitKeys - 1) / kUnitKeys;
            r.line = p.n_heads * (r.gp * r.up + r.go * r.uo);
            const int32_t grid = (int32_t)gridDim.x;
            r.per = (r.line + grid - 1) / grid;
            r.len = r.np = r.no = 0;
            if (rows_to > 0 && p.n_heads * (r.gp + r.go) <= grid) {
                r.len = r.per;       // from the length that would do without remainders
                for (;; ++r.len) {
                    r.np = (r.up + r.len - 1) / r.len;
                    r.no = (r.uo + r.len - 1) / r.len;
                    if (p.n_heads * (r.gp * r.np + r.go * r.no) <= grid) break;
                }
            }
        }
    }
    __syncthreads();

    for (bool first = true;; first = false) {
        if (threadIdx.x == 0) {
            // ---- the item: units [u0, u0 + n) of a column
            int32_t col = -1, u0 = 0, n = 0;
            if (r.len > 0) {
                const int32_t pre_items = p.n_heads * r.gp * r.np, e = (int32_t)blockIdx.x;
                if (first && e < pre_items + p.n_heads * r.go * r.no) {
                    col = e < pre_items ? e / r.np : p.n_heads * r.gp + (e - pre_items) / r.no;
                    u0 = (e < pre_items ? e % r.np : (e - pre_items) % r.no) * r.len;
                    n = r.len;
                    item.slot = e;
                }
            } else {
                const int32_t pre_units = p.n_heads * r.gp * r.up;
                const int32_t begin = (int32_t)min((int64_t)r.line, (int64_t)blockIdx.x * r.per);
                const int32_t end = (int32_t)min((int64_t)r.line, (int64_t)begin + r.per), at = first ? begin : item.at;
                if (at < end) {
                    col = at < pre_units ? at / r.up : p.n_heads * r.gp + (at - pre_units) / r.uo;
                    u0 = at - (at < pre_units ? col * r.up : pre_units + (col - p.n_heads * r.gp) * r.uo);
                    n = end - at;
                    item.slot = col + (int32_t)blockIdx.x;
                }
                item.at = at;
            }
            item.n_keys = 0;
            if (col >= 0) {
                const Column cl = column<R>(r, p.n_heads, col);
                n = min(n, cl.units - u0);
                item.at += n;
                item.head = cl.head;
                item.group = cl.group;
                item.stream = cl.stream;
                item.live = min(R, (cl.stream < 0 ? r.total : r.rows[cl.stream]) - cl.group * R);
                item.k0 = u0 * kUnitKeys;
                item.n_keys = min(n * kUnitKeys, (cl.stream < 0 ? p.n_prefix : p.n_tokens) - item.k0);
            }
        }
        __syncthreads();
        const int32_t n_keys = item.n_keys, n_blk = (n_keys + kBlk - 1) / kBlk;
        if (n_keys == 0) break;
        const int32_t h = item.head, k0 = item.k0, stream = item.stream;
        const bool pre = stream < 0;
        const void *ks0 = p.prefix.ks, *vs0 = p.prefix.vs;
        int64_t ld_scale = p.prefix.ld_scale;
        const uint32_t* kg = p.pg;
        const CUtensorMap *tk = &maps.pk, *tv = &maps.pv;
#pragma unroll
        for (int k = 0; k < kMaxBatch; ++k)
            if (k == stream) {
                ks0 = p.s[k].c.ks;
                vs0 = p.s[k].c.vs;
                ld_scale = p.s[k].c.ld_scale;
                kg = p.s[k].kg;
                tk = &maps.k[k];
                tv = &maps.v[k];
            }
        const uint16_t* ks = static_cast<const uint16_t*>(ks0) + (int64_t)h * ld_scale + k0;
        const uint16_t* vs = static_cast<const uint16_t*>(vs0) + (int64_t)h * ld_scale + k0;
        if (kg != nullptr) kg += k0;
        // ---- copies of block b of this warp's walk, the `nth` that it takes. Codes past the source are zeros.
        auto fetch = [&](int32_t b, uint32_t nth) {
            if (lane == 0) {
                const uint32_t slot = nth % kDepth, bar = bars + 8 * slot, dst = ring + slot * kRingSlot;
                mbar_arrive_expect_tx(bar, kRingSlot);
                tma_load_2d(dst, tk, bar, h * kHeadDim, k0 + b * kBlk);
                tma_load_2d(dst + kBlkBytes, tv, bar, h * kHeadDim, k0 + b * kBlk);
            }
        };
        // a block's 16 K and 16 V scales, one per lane, a block ahead (two copies fewer per block than by TMA: 12
        // rows over 16896 keys 32.2 us, and 32.6)
        uint32_t sc_next = 0;
        auto scales_of = [&](int32_t b) {
            const int32_t key = b * kBlk + (int32_t)(lane & 15);
            sc_next = key < n_keys ? __ldg((lane < 16 ? ks : vs) + key) : 0u;
        };
        uint32_t g_next[2] = {0xffffffffu, 0xffffffffu};     // groups of this lane's keys, a block ahead
        auto groups_of = [&](int32_t b) {
            if (kg != nullptr) {
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int32_t key = b * kBlk + key_of(g) + 8 * e;
                    g_next[e] = key < n_keys ? __ldg(kg + key) : 0u;
                }
            }
        };
        auto begin_walk = [&]() {
#pragma unroll
            for (int d = 0; d < kDepth - 1; ++d) {
                const int32_t b = warp + d * kRowsWarps;
                if (b < n_blk) fetch(b, it + d);
            }
            scales_of(warp);
            groups_of(warp);
        };
        begin_walk();

        // ---- queries into shared memory (a 16-byte piece per thread), this lane's rows' groups
        auto row_at = [&](int32_t e, int32_t& b, int32_t& m) -> bool {      // row e of the group
            m = item.group * R + e;
            b = stream;
            if (!pre) return m < r.rows[b];
            if (m >= r.total) return false;
            b = 0;
#pragma unroll
            for (int k = 1; k < kMaxBatch; ++k)
                if (k < p.n_streams && m >= r.first[k]) b = k;
            m -= r.first[b];
            return true;
        };
        auto stream_of = [&](int32_t b) {
            const Stream* st = &p.s[0];
#pragma unroll
            for (int k = 1; k < kMaxBatch; ++k)
                if (k == b) st = &p.s[k];
            return st;
        };
        float* q_factor = xm + 2 * kRowsWarps * R;      // what a row's queries were divided by
        for (int e0 = threadIdx.x; e0 < R * 16; e0 += Sh::threads) {      // whole warps: a row per half-warp
            int32_t b, m;
            uint4 x = make_uint4(0, 0, 0, 0);
            if (row_at(e0 >> 4, b, m)) {
                const Stream* st = stream_of(b);
                x = *reinterpret_cast<const uint4*>(static_cast<const T*>(st->qc) + (int64_t)m * st->ld_qc + (int64_t)h * kHeadDim +
                                                    (e0 & 15) * 8);
            }
            float factor = 1.f;
            if constexpr (StoreT<T>::kUmmaFormat == 1) {
                // the largest magnitude's exponent: bf16 bits, doubled to drop the sign
                uint32_t top = 0;
                uint32_t* w = &x.x;
#pragma unroll
                for (int e = 0; e < 4; ++e) top = max(top, max(w[e] & 0x7fffu, (w[e] >> 16) & 0x7fffu));
#pragma unroll
                for (int e = 8; e > 0; e >>= 1) top = max(top, __shfl_xor_sync(0xffffffffu, top, e));
                // to [2^10, 2^11); the exponent is kept where both the factor and its inverse are normal
                const int e = min(max((int)(top >> 7), 20), 254) - 137;
                factor = __int_as_float((127 + e) << 23);
                const float inv = __int_as_float((127 - e) << 23);
#pragma unroll
                for (int k = 0; k < 4; ++k) {
                    const float2 v = StoreT<T>::unpack2(w[k]);
                    w[k] = StoreT<__half>::pack2(v.x * inv, v.y * inv);
                }
            }
            if ((e0 & 15) == 0) q_factor[e0 >> 4] = factor;
            sts128(q_at + (e0 >> 4) * kQPad + (e0 & 15) * 16, x);
        }
        uint32_t qg[NQ][2];
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int e = 0; e < 2; ++e) {
                int32_t b, m;
                qg[q][e] = 0xffffffffu;
                if (row_at(8 * q + 2 * t + e, b, m)) {
                    const Stream* st = stream_of(b);
                    if (st->qg != nullptr) {
                        const int32_t i = st->idx[m];
                        qg[q][e] = (i >= 0 && i < p.n_tokens) ? st->qg[i] : 0u;
                    }
                }
            }
        bool any_empty = false;      // a row that sees nothing needs its mask where the keys have none
#pragma unroll
        for (int q = 0; q < NQ; ++q) any_empty = any_empty || qg[q][0] == 0 || qg[q][1] == 0;
        any_empty = __any_sync(0xffffffffu, any_empty);
        if (threadIdx.x == 0) ready = 0;
        __syncthreads();

        float o[NQ][8][4], m_run[NQ][2], l_run[NQ][2];
        float qs[NQ][2];                     // score factors of this lane's queries
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int d = 0; d < 2; ++d) qs[q][d] = p.scale_log2 * q_factor[8 * q + 2 * t + d];
        auto walk = [&](auto any_code) {
            constexpr bool kAnyCode = decltype(any_code)::value;
#pragma unroll
            for (int q = 0; q < NQ; ++q) {
#pragma unroll
                for (int j = 0; j < 8; ++j)
#pragma unroll
                    for (int e = 0; e < 4; ++e) o[q][j][e] = 0.f;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    m_run[q][e] = -INFINITY;
                    l_run[q][e] = 0.f;
                }
            }
            uint32_t issued = it + min(kDepth - 1, (n_blk - warp + kRowsWarps - 1) / kRowsWarps);
            for (int32_t b = warp; b < n_blk; b += kRowsWarps, ++it) {
                if (b + (kDepth - 1) * kRowsWarps < n_blk) {
                    fetch(b + (kDepth - 1) * kRowsWarps, it + kDepth - 1);
                    ++issued;
                }
                const uint32_t seen[2] = {g_next[0], g_next[1]};
                const uint32_t sc = sc_next;
                scales_of(b + kRowsWarps);
                groups_of(b + kRowsWarps);
                const uint32_t slot = it % kDepth;
                if (!__all_sync(0xffffffffu, mbar_wait(bars + 8 * slot, (it / kDepth) & 1, &abort))) break;
                const uint8_t* blk_p = smem + warp * Sh::ring_warp + slot * kRingSlot;
                // S^T = K Q^T
                float s[NQ][4];
#pragma unroll
                for (int q = 0; q < NQ; ++q) s[q][0] = s[q][1] = s[q][2] = s[q][3] = 0.f;
#pragma unroll
                for (int cc = 0; cc < 2; ++cc) {
                    const uint32_t off = key_of(g) * 128 + ((uint32_t)((cc * 4 + t) ^ key_of(g)) << 4);
                    const uint4 ka = *reinterpret_cast<const uint4*>(blk_p + off), kb = *reinterpret_cast<const uint4*>(blk_p + off + 8 * 128);
                    const uint32_t wa[4] = {q8::code_word<F>(ka.x), q8::code_word<F>(ka.y), q8::code_word<F>(ka.z), q8::code_word<F>(ka.w)};
                    const uint32_t wb[4] = {q8::code_word<F>(kb.x), q8::code_word<F>(kb.y), q8::code_word<F>(kb.z), q8::code_word<F>(kb.w)};
#pragma unroll
                    for (int jp = 0; jp < 2; ++jp) {
                        uint4 q4[NQ];
#pragma unroll
                        for (int q = 0; q < NQ; ++q)
                            q4[q] = *reinterpret_cast<const uint4*>(smem + Sh::at_q + (g + 8 * q) * kQPad + (cc * 64 + t * 16 + jp * 8) * 2);
#pragma unroll
                        for (int jj = 0; jj < 2; ++jj) {
                            const int j = 2 * jp + jj;
                            const uint32_t a0 = q8::code_pair<F, kAnyCode>(wa[j], false), a1 = q8::code_pair<F, kAnyCode>(wb[j], false);
                            const uint32_t a2 = q8::code_pair<F, kAnyCode>(wa[j], true), a3 = q8::code_pair<F, kAnyCode>(wb[j], true);
#pragma unroll
                            for (int q = 0; q < NQ; ++q)
                                mma16816(s[q], a0, a1, a2, a3, jj ? q4[q].z : q4[q].x, jj ? q4[q].w : q4[q].y);
                        }
                    }
                }
                // scales and masks: this lane's keys, key_of(g) and 8 behind it
                float v_sc[2], v_log[2];     // what P is multiplied with, its logarithm
                const int32_t left = n_keys - b * kBlk;
                bool grow = false;
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int key = key_of(g) + 8 * e;
                    const float kk = StoreT<T>::unpack2(__shfl_sync(0xffffffffu, sc, key)).x;
                    const float vv = StoreT<T>::unpack2(__shfl_sync(0xffffffffu, sc, kBlk + key)).x;
                    const bool v_ok = q8::valid_scale<T, F>(vv);
                    const float f = v_ok && q8::valid_scale<T, F>(kk) ? kk : __uint_as_float(0x7fc00000u);
                    v_sc[e] = v_ok ? vv : 0.f;
                    // (bounded below, so that exp2(score - maximum) stays finite: V scales under 2^-100 lose bits)
                    v_log[e] = fmaxf(lg2_approx(v_sc[e]), -100.f);
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int d = 0; d < 2; ++d) s[q][2 * e + d] *= f * qs[q][d];
                }
                if (kg != nullptr || left < kBlk) {
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const bool in = key_of(g) + 8 * e < left;
#pragma unroll
                        for (int q = 0; q < NQ; ++q)
#pragma unroll
                            for (int d = 0; d < 2; ++d)
                                if (!in || (seen[e] & qg[q][d]) == 0) s[q][2 * e + d] = -INFINITY;
                    }
                } else if (any_empty) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int d = 0; d < 2; ++d)
                            if (qg[q][d] == 0) s[q][d] = s[q][2 + d] = -INFINITY;
                }
#pragma unroll
                for (int q = 0; q < NQ; ++q)
#pragma unroll
                    for (int d = 0; d < 2; ++d)
                        grow = grow || fmaxf(s[q][d] + v_log[0], s[q][2 + d] + v_log[1]) > m_run[q][d] + 8.f;
                // the running maxima move only where a weight passes one by more than 2^8 (P stays below that)
                if (__any_sync(0xffffffffu, grow)) {
#pragma unroll
                    for (int q = 0; q < NQ; ++q)
#pragma unroll
                        for (int d = 0; d < 2; ++d) {
                            float x = fmaxf(s[q][d] + v_log[0], s[q][2 + d] + v_log[1]);
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 4));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 8));
                            x = fmaxf(x, __shfl_xor_sync(0xffffffffu, x, 16));
                            const float mn = fmaxf(m_run[q][d], x);
                            const float al = mn == m_run[q][d] ? 1.f : ex2_approx(m_run[q][d] - mn);
                            m_run[q][d] = mn;
                            l_run[q][d] *= al;
#pragma unroll
                            for (int j = 0; j < 8; ++j) {
                                o[q][j][d] *= al;
                                o[q][j][2 + d] *= al;
                            }
                        }
                }
                uint32_t pb[NQ][2];
#pragma unroll
                for (int q = 0; q < NQ; ++q) {
                    float e_[4];
#pragma unroll
                    for (int d = 0; d < 2; ++d) {
                        const float mu = m_run[q][d] == -INFINITY ? 0.f : m_run[q][d];
                        e_[d] = ex2_approx(s[q][d] - mu);
                        e_[2 + d] = ex2_approx(s[q][2 + d] - mu);
                        l_run[q][d] += e_[d] + e_[2 + d];
                    }
                    pb[q][0] = transpose8(StoreT<__half>::pack2(e_[0] * v_sc[0], e_[1] * v_sc[0]));
                    pb[q][1] = transpose8(StoreT<__half>::pack2(e_[2] * v_sc[1], e_[3] * v_sc[1]));
                }
                // O^T += V^T P^T
                // (operand row index 2 t + x of a half is key key_of(2 t + x) = t + 4 x)
                uint32_t w[4][4];
#pragma unroll
                for (int e = 0; e < 4; ++e) {
                    const uint32_t row = t + 4 * (e & 1) + 8 * (e >> 1);
                    const uint4 v4 = *reinterpret_cast<const uint4*>(blk_p + kBlkBytes + row * 128 + (((uint32_t)key_of(g) ^ (row & 7)) << 4));
                    w[e][0] = q8::code_word<F>(v4.x);
                    w[e][1] = q8::code_word<F>(v4.y);
                    w[e][2] = q8::code_word<F>(v4.z);
                    w[e][3] = q8::code_word<F>(v4.w);
                }
#pragma unroll
                for (int j = 0; j < 8; ++j) {
                    // dims 2 j and 2 j + 1 of the lane's 16: the two keys' bytes side by side
                    const uint32_t lo = __byte_perm(w[0][j >> 1], w[1][j >> 1], (j & 1) ? 0x7362 : 0x5140);
                    const uint32_t hi = __byte_perm(w[2][j >> 1], w[3][j >> 1], (j & 1) ? 0x7362 : 0x5140);
                    const uint32_t a0 = q8::code_pair<F, kAnyCode>(lo, false), a1 = q8::code_pair<F, kAnyCode>(lo, true);
                    const uint32_t a2 = q8::code_pair<F, kAnyCode>(hi, false), a3 = q8::code_pair<F, kAnyCode>(hi, true);
#pragma unroll
                    for (int q = 0; q < NQ; ++q) mma16816(o[q][j], a0, a1, a2, a3, pb[q][0], pb[q][1]);
                }
                __syncwarp();
            }
            // after a timeout only: nothing may land in shared memory any more
            for (; it < issued; ++it) mbar_wait_drain_bounded(bars + 8 * (it % kDepth), (it / kDepth) & 1);
        };
        walk(std::false_type{});
        if constexpr (F == q8::kE4m3) {
            // The codes 0x7f and 0xff come out of the conversion as NaN, and 0 * NaN also reaches rows that do not
            // see them: where any row of the item is NaN, it runs again with the conversion that takes every code
            // for a number. (That conversion for all items: 12 rows over 16896 keys 35.6 us, and 31.4; 8 streams
            // of 48 rows together, 4608 shared + 2304 own keys, 84.6 and 75.4.)
            float sum = 0.f;
#pragma unroll
            for (int q = 0; q < NQ; ++q)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    sum = fmaf(l_run[q][e], 0.f, sum);
#pragma unroll
                    for (int j = 0; j < 8; ++j) sum = fmaf(o[q][j][e], 0.f, fmaf(o[q][j][2 + e], 0.f, sum));
                }
            if (__syncthreads_or(sum != sum) && !abort) {
                begin_walk();
                walk(std::true_type{});
            }
        }
        __syncthreads();
        if (abort) return;
        // ---- the warps' results meet: position 8 d + g of a row is d of lane g's 16 dims (tile j holds
        // d = 2 j and 2 j + 1), then a row per warp, four positions per lane
        const int live = item.live;
#pragma unroll
        for (int q = 0; q < NQ; ++q)
#pragma unroll
            for (int d = 0; d < 2; ++d) {
                const int row = 8 * q + 2 * t + d;
                float* dst = xo + (warp * R + row) * kPadRow + g;
                if (row < live) {
#pragma unroll
                    for (int j = 0; j < 8; ++j) {
                        dst[16 * j] = o[q][j][d];
                        dst[16 * j + 8] = o[q][j][2 + d];
                    }
                }
                float l = l_run[q][d];
                l += __shfl_xor_sync(0xffffffffu, l, 4);
                l += __shfl_xor_sync(0xffffffffu, l, 8);
                l += __shfl_xor_sync(0xffffffffu, l, 16);
                if (g == 0) {
                    xm[row * kRowsWarps + warp] = m_run[q][d];
                    xm[(R + row) * kRowsWarps + warp] = l;
                }
            }
        __syncthreads();
        for (int row = warp; row < live; row += kRowsWarps) {
            const float m_w = lane < kRowsWarps ? xm[row * kRowsWarps + lane] : -INFINITY;
            float top = m_w;
#pragma unroll
            for (int e = kRowsWarps / 2; e > 0; e >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, e));
            top = __shfl_sync(0xffffffffu, top, 0);
            const float f = ex2_approx(m_w - (top == -INFINITY ? 0.f : top));
            float l = lane < kRowsWarps ? f * xm[(R + row) * kRowsWarps + lane] : 0.f;
#pragma unroll
            for (int e = kRowsWarps / 2; e > 0; e >>= 1) l += __shfl_xor_sync(0xffffffffu, l, e);
            float4 acc = make_float4(0.f, 0.f, 0.f, 0.f);
#pragma unroll
            for (int k = 0; k < kRowsWarps; ++k) {
                const float fk = __shfl_sync(0xffffffffu, f, k);
                const float4 x = *reinterpret_cast<const float4*>(xo + (k * R + row) * kPadRow + 4 * lane);
                acc.x += fk * x.x;
                acc.y += fk * x.y;
                acc.z += fk * x.z;
                acc.w += fk * x.w;
            }
            float* dst = p.part + (int64_t)item.slot * kRowsSlotFloats;
            *reinterpret_cast<float4*>(dst + row * kHeadDim + 4 * lane) = acc;
            if (lane == 0) {
                dst[kRowsMax * kHeadDim + row] = top;
                dst[kRowsMax * kHeadDim + kRowsMax + row] = l;
            }
        }
        __syncthreads();     // the arrivals below release what every thread stored
        // ---- arrivals: thread e for the e-th own group that the item's rows belong to
        if (threadIdx.x < 32) {
            int32_t b = -1, grp = 0, found = 0;
            if (item.stream >= 0) {
                if (lane == 0) {
                    b = item.stream;
                    grp = item.group;
                }
            } else {
                const int32_t r0 = item.group * R, r1 = min(r0 + R, r.total);     // packed rows
#pragma unroll
                for (int k = 0; k < kMaxBatch; ++k)
                    if (k < p.n_streams && r.rows[k] > 0) {
                        const int32_t a0 = max(r0, r.first[k]) - r.first[k], a1 = min(r1, r.first[k] + r.rows[k]) - r.first[k];
                        if (a1 > a0) {
                            const int32_t g0 = a0 / R, g1 = (a1 - 1) / R;
                            if (lane >= found && lane <= found + g1 - g0) {
                                b = k;
                                grp = g0 + lane - found;
                            }
                            found += g1 - g0 + 1;
                        }
                    }
            }
            bool done = false;
            if (b >= 0) {
                const int32_t groups = (r.rows[b] + R - 1) / R;
                int32_t unused, all;
                parts_of(r, p.n_heads, p.n_heads * (r.gp + r.group0[b]) + item.head * groups + grp, unused, all);
                if (r.gp > 0) {
                    const int32_t x0 = r.first[b] + grp * R, x1 = min(x0 + R, r.first[b] + r.rows[b]);
                    for (int32_t x = x0 / R; x <= (x1 - 1) / R; ++x) {
                        int32_t more;
                        parts_of(r, p.n_heads, item.head * r.gp + x, unused, more);
                        all += more;
                    }
                }
                int32_t* cnt = p.cnt + (r.group0[b] + grp) * p.n_heads + item.head;
                done = atom_add_acq_rel_gpu(cnt, 1) == all - 1;
                if (done) *cnt = 0;      // for the next launch
            }
            const uint32_t vote = __ballot_sync(0xffffffffu, done);
            if (lane == 0) ready = vote;
        }
        __syncthreads();
        for (uint32_t left = ready; left != 0; left &= left - 1) {
            const int e = __ffs(left) - 1;
            int32_t b = item.stream, grp = item.group;
            if (b < 0) {                 // the e-th own group again
                const int32_t r0 = item.group * R, r1 = min(r0 + R, r.total);
                int32_t found = 0;
#pragma unroll
                for (int k = 0; k < kMaxBatch; ++k)
                    if (k < p.n_streams && r.rows[k] > 0) {
                        const int32_t a0 = max(r0, r.first[k]) - r.first[k], a1 = min(r1, r.first[k] + r.rows[k]) - r.first[k];
                        if (a1 > a0) {
                            const int32_t g0 = a0 / R, g1 = (a1 - 1) / R;
                            if (e >= found && e <= found + g1 - g0) {
                                b = k;
                                grp = g0 + e - found;
                            }
                            found += g1 - g0 + 1;
                        }
                    }
            }
            rows_combine<T, R>(p, r, item.head, b, grp);
        }
        fence_async_smem();          // the next item's copies overwrite the exchange
        __syncthreads();
    }
}

// ---------------------------------------------------------------------------------------------
// Many rows per stream (but those that q8_expand_kernel and the 16-bit kernel serve): bound by the tensor core. The two-tile schedule of the 16-bit attention
// (fxr_attention2.cuh: 256 compact query rows of one head per unit, 128 keys per step, S and O in
// tensor memory, P written over S, lazy rescaling, units cut between CTAs when whole ones would leave
// SMs idle) with K and V tiles that arrive as codes: a fourth warpgroup turns each 128 x 128 tile of
// codes in shared memory into the 16-bit tile that tcgen05.mma reads, T(code * scale), one row per
// thread, in the 128-byte swizzle on both sides (every access of 8 lanes covers all banks). TMA moves
// codes only: half the bytes of the 16-bit cache.
// Warps (512 threads): 0-7 softmax of tile 0 / 1, 8 TMA producer, 9 tensor memory and the MMA
// issuer, 10 scheduler (writes the CTA's items into a 2-slot ring in shared memory, so that no other
// role carries the bookkeeping), 11 idle, 12-15 converters.
// Prefix rows come first, then the stream's own; a source's last tile is filled with zeros and its
// scores masked. With visibility groups, visible_steps_kernel lists for every 256-row unit the tiles
// that some row of it sees, and which of them all its rows see whole; the others are masked score by
// score. Rows that see nothing end with a maximum of -inf and store zeros.
// Rounded to T: K and V, as the read-back does, and P, since the products take 16-bit operands (half a step each;
// P in f16 below 2^-14: 2^-25); scores, maxima, sums and O are held in 32 bits. Error against 64 bits: 0.0034 of
// the outputs' root mean square in bf16 and 0.00042 in f16, twice that of the output's own rounding. Codes held
// exactly, as for few rows, would take two multiplications (K and V scale) for every score in the softmax
// warps, where the converters now take one for every element of a tile.
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
// Costs in steps (2.6 us each): an item's start and end; a cut (partial results, the combine's launch);
// a part in the combine of its unit.
constexpr float kItemSteps = 2.0f, kCutSteps = 2.5f, kPartSteps = 0.25f;
constexpr int kPartSlots = 4;                    // partial tiles a CTA may write
constexpr int kPartFloats = kBM * kD + 2 * kBM;
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
    float* part;                 // where the item's partial result goes, NULL: it is a whole unit
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

// How n_units units of `total` steps together run on `grid` CTAs: whole, round-robin (per = parts = 0);
// each unit in `parts` equal parts with a CTA each; or the launch's steps, unit after unit, in ranges of
// `per` per CTA. The cheapest by the costs above.
struct TileSchedule {
    int32_t per, parts;
};
__host__ __device__ inline TileSchedule tile_schedule(int32_t total, int32_t n_units, int32_t grid) {
    TileSchedule s{0, 0};
    if (n_units == 0) return s;
    const int32_t each = (total + grid - 1) / grid, most = grid / n_units;
    const float avg = (float)total / (float)n_units;
    float best = (float)((n_units + grid - 1) / grid) * (avg + kItemSteps);
    const float cut = (float)each + kItemSteps * ((float)each / avg + 1.f) + kCutSteps + kPartSteps * (avg / (float)each + 1.f);
    if (cut < best) {
        best = cut;
        s.per = each;
    }
    for (int32_t n = 2; n <= most && (float)n <= avg + 1.f; ++n) {
        const float even = ceilf(avg / (float)n) + kItemSteps + kCutSteps + kPartSteps * (float)n;
        if (even <= best) {
            best = even;
            s = TileSchedule{0, n};
        }
    }
    return s;
}

// A unit that was cut, in the entry of the CTA that holds its first part (which ends that CTA's range, so
// that there is one at most).
struct CutUnit {
    int32_t parts;               // 0: none
    int32_t stream, head, row0, rows;
    int32_t c_first, i0, per;
};

struct TileParams {
    Params p;
    int32_t n_pre, n_own;        // key tiles of the prefix and of a stream's own rows
    int32_t units_cap;           // units of a stream at most (rows of steps / list)
    const int32_t* steps;        // [stream][units_cap] listed steps, NULL: every unit runs all tiles
    const uint16_t* list;        // [stream][units_cap][n_pre + n_own] tile | 0x8000 where it needs the masks
    const uint32_t* groups;      // [n_pre + n_streams * n_own][128] key groups, zeros past a source's end
    int32_t may_cut;             // 0: whole units only (no combine follows)
    float* part;                 // [grid][kPartSlots][kPartFloats]
    CutUnit* cuts;               // [grid]
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
    // (rows whose set is empty are left out: their result is zeros whatever their scores)
    const uint32_t same = __match_any_sync(0xffffffffu, mine) & __ballot_sync(0xffffffffu, live && mine != 0);
    if (live && mine != 0 && lane == __ffs(same) - 1) row_word[atomicAdd(&n_words, 1)] = mine;
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

// ---- pieces of the tile kernel --------------------------------------------------------------------
// Scratch slot of the part that CTA c holds of a unit whose iterations start at i0: its first item
// unless the unit starts inside c's range behind others.
__device__ __forceinline__ int64_t part_at(int32_t i0, int32_t per, int32_t c, int t) {
    const int k = i0 > c * per ? 1 : 0;
    return (((int64_t)c * 2 + k) * 2 + t) * kPartFloats;
}

// End of an item that is part of a unit: its O rows, maxima and sums go to scratch and O is released.
// Out of line, as in the 16-bit kernel, so that the step loop around it keeps its code.
__device__ __noinline__ void cut_epilogue(float* slot, int r, uint32_t tO, float m_run, float l_run, bool blind, bool live,
                                          uint32_t ofree) {
    if (__any_sync(0xffffffffu, live)) {
#pragma unroll 1
        for (int h = 0; h < 4; ++h) {
            uint32_t o[32];
            FXR_TMEM_LD32(tO + h * 32u, o);
#pragma unroll
            for (int k = 0; k < 8; ++k)
                reinterpret_cast<float4*>(slot)[(h * 8 + k) * kBM + r] =
                    blind ? make_float4(0.f, 0.f, 0.f, 0.f)
                          : make_float4(__uint_as_float(o[4 * k]), __uint_as_float(o[4 * k + 1]), __uint_as_float(o[4 * k + 2]),
                                        __uint_as_float(o[4 * k + 3]));
        }
        slot[kBM * kD + r] = m_run;
        slot[kBM * kD + kBM + r] = l_run;
    }
    tc_fence_before();
    mbar_arrive(ofree);
}

// Cut units' parts into their rows, in key order: a warp takes 32 rows by 16 columns of a unit (a row per
// lane; partial O is stored column chunk by column chunk, so that its loads are whole lines), 16 CTAs
// a unit. A launch of its own, chained to the tile kernel's end: its warps spread over all SMs, where a
// combine by the last part to arrive read all of a unit's parts through one SM, 2.5 us per part (601 rows
// of two streams, documents: 50 us with that, 38.5 with this). It costs a call about 5 us, so calls whose
// units the host knows to stay whole go without.
constexpr int kCombineThreads = 128, kCombineCtas = 16;   // threads of a CTA, CTAs of a unit

template <typename T>
__global__ void __launch_bounds__(kCombineThreads) combine_kernel(const __grid_constant__ Params p, const float* part,
                                                                  const CutUnit* cuts) {
    pdl_launch_dependents();
    pdl_wait();
    const CutUnit u = cuts[blockIdx.x / kCombineCtas];
    if (u.parts == 0) return;
    const int lane = threadIdx.x & 31, w = (int)(blockIdx.x % kCombineCtas) * (kCombineThreads / 32) + (threadIdx.x >> 5);
    const int t = w >> 5, r = ((w >> 3) & 3) * 32 + lane, h = w & 7;     // tile, row, 16 columns
    const int32_t row = u.row0 + t * kBM + r;
    const bool live = row < u.rows;
    if (!__any_sync(0xffffffffu, live)) return;
    const int32_t* idx = nullptr;
    void* out = nullptr;
#pragma unroll
    for (int b = 0; b < kMaxBatch; ++b)
        if (b == u.stream) {
            idx = p.s[b].idx;
            out = p.s[b].out;
        }
    const int32_t i = live ? idx[row] : -1;
    constexpr int kAhead = 4;                            // parts whose loads are in flight together
    float top = -INFINITY, l = 0.f, acc[16];
#pragma unroll
    for (int k = 0; k < 16; ++k) acc[k] = 0.f;
    for (int32_t c = 0; c < u.parts; c += kAhead) {
        float4 x[kAhead][4];
        float m[kAhead], ls[kAhead], next = top;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const bool in = c + e < u.parts;
            const float* q = part + part_at(u.i0, u.per, u.c_first + (in ? c + e : c), t);
            m[e] = in ? __ldcg(q + kBM * kD + r) : -INFINITY;
            ls[e] = in ? __ldcg(q + kBM * kD + kBM + r) : 0.f;
#pragma unroll
            for (int k = 0; k < 4; ++k) x[e][k] = __ldcg(reinterpret_cast<const float4*>(q) + (h * 4 + k) * kBM + r);
        }
#pragma unroll
        for (int e = 0; e < kAhead; ++e) next = fmaxf(next, m[e]);
        const float base = next == -INFINITY ? 0.f : next, al = ex2_approx(top - base);
        top = next;
        l *= al;
#pragma unroll
        for (int k = 0; k < 16; ++k) acc[k] *= al;
#pragma unroll
        for (int e = 0; e < kAhead; ++e) {
            const float f = ex2_approx(m[e] - base);
            l += f * ls[e];
#pragma unroll
            for (int k = 0; k < 4; ++k) {
                acc[4 * k] += f * x[e][k].x;
                acc[4 * k + 1] += f * x[e][k].y;
                acc[4 * k + 2] += f * x[e][k].z;
                acc[4 * k + 3] += f * x[e][k].w;
            }
        }
    }
    if (!live) return;
    if (i < 0 || i >= p.n_tokens) {
        if (h == 0) atomicOr(&g_error_word, kErrBounds);
        return;
    }
    const float inv = l == 0.f ? 0.f : 1.0f / l;
    uint4* dst = reinterpret_cast<uint4*>(static_cast<T*>(out) + (int64_t)i * p.ld_out + (int64_t)u.head * kD + 16 * h);
#pragma unroll
    for (int k = 0; k < 2; ++k)
        dst[k] = make_uint4(StoreT<T>::pack2(acc[8 * k] * inv, acc[8 * k + 1] * inv),
                            StoreT<T>::pack2(acc[8 * k + 2] * inv, acc[8 * k + 3] * inv),
                            StoreT<T>::pack2(acc[8 * k + 4] * inv, acc[8 * k + 5] * inv),
                            StoreT<T>::pack2(acc[8 * k + 6] * inv, acc[8 * k + 7] * inv));
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
    __shared__ int32_t stream_rows[kMaxBatch];
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
    if (warp == kProducerWarp && (int32_t)lane < p.n_streams) {
        prefetch_tmap(&maps.q[lane]);
        prefetch_tmap(&maps.k[lane]);
        prefetch_tmap(&maps.v[lane]);
        if (lane == 0 && p.n_prefix > 0) {
            prefetch_tmap(&maps.pk);
            prefetch_tmap(&maps.pv);
        }
    }
    __syncwarp();
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = *tmem_slot;
    pdl_launch_dependents();
    pdl_wait();

    if (threadIdx.x < kMaxBatch) {
        int32_t c = 0;
#pragma unroll
        for (int b = 0; b < kMaxBatch; ++b)
            if (b == (int)threadIdx.x && b < p.n_streams) c = *p.s[b].count;
        if (c > p.max_rows && blockIdx.x == 0) atomicOr(&g_error_word, kErrBounds);
        stream_rows[threadIdx.x] = max(0, min(c, p.max_rows));
    }
    __syncthreads();
    if (warp >= kConvWarp) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 %0;" ::"n"(kRegsOther));
        // ---------------- converters: one row of the tile per thread ----------------
        auto wwait = [&](uint32_t b_, uint32_t par_) -> bool { return __all_sync(0xffffffffu, mbar_wait(b_, par_, abort)); };
        const uint32_t r = (uint32_t)(warp - kConvWarp) * 32 + lane, x = r & 7;
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
                // a row without a valid scale: its scores are NaN, its V counts as zeros
                const bool v_ok = q8::valid_scale<T, F>(sv);
                if (!v_ok || !q8::valid_scale<T, F>(sk)) sk = __uint_as_float(0x7fc00000u);
                if (!v_ok) sv = 0.f;
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
                    const uint32_t f2 = StoreT<T>::pack2(f, f);
                    auto store = [&](uint32_t c, const uint4& lo, const uint4& hi) {
                        const uint32_t d = dst + (c >> 2) * kSpan;
                        sts128(d + (((2 * (c & 3)) ^ x) << 4), lo);
                        sts128(d + (((2 * (c & 3) + 1) ^ x) << 4), hi);
                    };
                    auto tile_free = [&]() { return in < kTiles || wwait(bar(kEmpty + ts), (in / kTiles - 1) & 1); };
                    auto raw_done = [&]() {
                        __syncwarp();
                        if (lane == 0) mbar_arrive(bar(kRawEmpty + rs));
                    };
                    if (!tile_free()) { ok = false; break; }
                    // a loop of 4 chunks, not all 8 unrolled: the roles' code is longer than the instruction
                    // caches hold (a quarter of a 2048 px frame: 1070 us, unrolled 1195)
                    auto convert = [&](auto dec) {
                        dec.scale(f2);
                        uint4 next = lds128(src + (x << 4));
#pragma unroll 4
                        for (uint32_t c = 0; c < 8; ++c) {
                            const uint4 q = next;
                            if (c < 7) next = lds128(src + (((c + 1) ^ x) << 4));
                            uint4 lo, hi;
                            q8::decode16(q, dec, lo, hi);
                            store(c, lo, hi);
                        }
                    };
                    using Dec = q8::TileDecoder<T, F>;
                    if constexpr (Dec::has_limit) {
                        if (!__any_sync(0xffffffffu, fabsf(f) >= Dec::limit)) convert(typename Dec::small{});
                        else convert(typename Dec::any{});
                    } else {
                        convert(typename Dec::any{});
                    }
                    raw_done();
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
            // ---------------- MMA issuer (order and waits of the 16-bit kernel) ----------------
            // The whole warp walks, and its waits end alike on every lane, so that counters and
            // descriptors are uniform; one elected lane issues (1536 rows over 4608 keys: 93 us,
            // and 100 with a single lane that walks and issues).
            constexpr uint32_t fmt = StoreT<T>::kUmmaFormat;
            constexpr uint32_t idesc_qk = make_idesc_f16(fmt, 0, kBM, kBN);
            constexpr uint32_t idesc_pv = make_idesc_f16(fmt, 1, kBM, kD);
            uint32_t acq = 0, rel = 0, q_it = 0, g = 0, done = 0;
            bool ok = true, issued = false;
            auto wait = [&](uint32_t b_, uint32_t par_) -> bool { return __all_sync(0xffffffffu, mbar_wait_spin(b_, par_, abort)); };
            auto acquire = [&]() -> uint32_t {
                const uint32_t st = acq % kTiles;
                if (!wait(bar(kFull + st), (acq / kTiles) & 1)) return 0;
                ++acq;
                return base + kSmTiles + st * kTile;
            };
            auto release = [&]() {
                if (elect_one()) umma_commit(bar(kEmpty + rel % kTiles));
                ++rel;
            };
            auto qk = [&](int t, uint32_t sK) {
                const uint64_t dq = smem_desc_sw128(base + kSmQ + t * kTile, 16, 1024);
                const uint64_t dk = smem_desc_sw128(sK, 16, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 0; k < kD / 16; ++k) {
                        const uint64_t off = ((k >> 2) * kSpan + (k & 3) * 32u) >> 4;
                        umma_ss(tmem + kColS + t * 128u, dq + off, dk + off, idesc_qk, k > 0 ? 1u : 0u);
                    }
                    umma_commit(bar(kSFull + t));
                }
                __syncwarp();
            };
            auto pv = [&](int t, uint32_t sV, int h, bool acc) {
                const uint64_t dv = smem_desc_sw128(sV, kSpan, 1024);
                if (elect_one()) {
#pragma unroll
                    for (int k = 4 * h; k < 4 * h + 4; ++k)
                        umma_ts(tmem + kColO + t * 128u, tmem + kColS + t * 128u + k * 8u, dv + (uint64_t)((k * 2048u) >> 4),
                                idesc_pv, (acc || k > 0) ? 1u : 0u);
                    if (h == 1) umma_commit(bar(kPVDone + t));
                }
                __syncwarp();
            };
            for (uint32_t it_no = 0; ok; ++it_no) {
                if (!wait(bar(kItemFull + (it_no & 1)), (it_no >> 1) & 1)) break;
                const int32_t n = __shfl_sync(0xffffffffu, item_at(it_no)->n, 0);
                if (elect_one()) mbar_arrive(bar(kItemEmpty + (it_no & 1)));
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
                if (n == 1 && elect_one()) umma_commit(bar(kQEmpty));
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
                                if (j + 2 == n && elect_one()) umma_commit(bar(kQEmpty));
                            }
                        }
                    }
                    if (!ok) break;
                }
                ++done;
            }
            if (__any_sync(0xffffffffu, *abort != 0) && issued && elect_one()) {
                umma_commit(bar(kDrain));
                attn::mbar_wait_drain(bar(kDrain), 0);
            }
        } else if (warp == kSchedWarp) {
            // ---------------- scheduler: the CTA's items, by a schedule that every CTA computes alike ----------
            const int32_t n_steps = a.n_pre + a.n_own;
            int32_t per = 0, parts = 0, total = 0, n_units = 0;
#pragma unroll 1
            for (int b = 0; b < p.n_streams; ++b) {
                    const int32_t units = (stream_rows[b] + kUnitRows - 1) / kUnitRows;
                    n_units += units * p.n_heads;
                    if (a.steps == nullptr) {
                        total += units * p.n_heads * n_steps;
                    } else {
                        int32_t sum = 0;
                        for (int32_t u = (int32_t)lane; u < units; u += 32) sum += a.steps[b * a.units_cap + u];
                        total += __reduce_add_sync(0xffffffffu, sum) * p.n_heads;
                    }
                }
            if (a.may_cut) {
                const TileSchedule sc = tile_schedule(total, n_units, (int32_t)gridDim.x);
                per = sc.per;
                parts = sc.parts;
            }
            const int32_t grid = (int32_t)gridDim.x, c = (int32_t)blockIdx.x;
            int32_t cur = per > 0 ? (int32_t)min((int64_t)total, (int64_t)c * per) : parts > 0 ? c / parts : c;
            const int32_t end = per > 0 ? (int32_t)min((int64_t)total, (int64_t)cur + per) : n_units;
            bool cut_made = false;                        // (of lane 0)
            for (uint32_t k = 0;; ++k) {
                bool more = cur < end;
                // the unit: stream, head, first row, steps, first iteration
                int32_t b = -1, rows = 0, head = 0, unit = 0, cnt = n_steps, rest = cur, i0 = cur;
                if (more) {
                    int32_t units = 1;
#pragma unroll 1
                    for (int s = 0; b < 0 && s < p.n_streams; ++s) {
                            const int32_t m = stream_rows[s];
                            const int32_t u = (m + kUnitRows - 1) / kUnitRows;
                            int32_t span = u;             // per head, in units or iterations
                            if (per > 0) {
                                if (a.steps == nullptr) {
                                    span = u * n_steps;
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
                                head = rest / span;
                                rest -= head * span;
                            } else {
                                rest -= span * p.n_heads;
                            }
                        }
                    if (per == 0) {
                        unit = rest;
                        if (a.steps) cnt = a.steps[b * a.units_cap + unit];
                    } else if (a.steps == nullptr) {
                        unit = rest / n_steps;
                        i0 = cur - (rest - unit * n_steps);
                    } else {
                        int32_t left = rest;              // iterations into the head's units
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
                // the item's steps
                int32_t s0 = 0, n = cnt, of = 1;
                if (per > 0) {
                    s0 = cur - i0;
                    n = min(cnt - s0, end - cur);
                    of = (i0 + cnt - 1) / per - i0 / per + 1;
                } else if (parts > 0) {
                    const int32_t e = c - cur * parts;
                    of = min(parts, cnt);
                    more = more && e < of;
                    s0 = cnt * e / of;
                    n = cnt * (e + 1) / of - s0;
                    i0 = 0;                               // the part is the CTA's first item
                }
                if (!more) n = 0;
                if (lane == 0 && n > 0 && n < cnt && s0 == 0) {
                    a.cuts[c] = CutUnit{of, b, head, unit * kUnitRows, rows, c, i0, per};
                    cut_made = true;
                }
                if (k >= 2 && !__all_sync(0xffffffffu, mbar_wait(bar(kItemEmpty + (k & 1)), ((k >> 1) - 1) & 1, abort))) break;
                Item* it = item_at(k);
                if (lane == 0) {
                    it->n = n;
                    if (n > 0) {
                        const Stream& st = a.p.s[b];
                        it->tq = &maps.q[b];
                        it->tk = &maps.k[b];
                        it->tv = &maps.v[b];
                        it->ks = static_cast<const T*>(st.c.ks) + (int64_t)head * st.c.ld_scale;
                        it->vs = static_cast<const T*>(st.c.vs) + (int64_t)head * st.c.ld_scale;
                        it->idx = st.idx;
                        it->qg = st.qg;
                        it->out = st.out;
                        it->s0 = s0;
                        it->head = head;
                        it->row0 = unit * kUnitRows;
                        it->rows = rows;
                        it->list = a.steps ? a.list + ((int64_t)b * a.units_cap + unit) * n_steps : nullptr;
                        it->part = n < cnt ? a.part + part_at(i0, per, c, 0) : nullptr;
                        it->stream = b;
                    }
                    mbar_arrive(bar(kItemFull + (k & 1)));
                }
                __syncwarp();
                if (n == 0) break;
                cur = per > 0 ? cur + n : parts > 0 ? end : cur + grid;
            }
            if (a.may_cut && lane == 0 && !cut_made) a.cuts[c].parts = 0;
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
                for (int q = 0; q < 8; ++q) mp[q] = q8::max2n(__uint_as_float(s[2 * q]), __uint_as_float(s[2 * q + 1]));
#pragma unroll
                for (int i = 1; i < 8; ++i)
#pragma unroll
                    for (int q = 0; q < 8; ++q)
                        mp[q] = q8::max3n(mp[q], __uint_as_float(s[16 * i + 2 * q]), __uint_as_float(s[16 * i + 2 * q + 1]));
                const float mx = q8::max3n(q8::max3n(mp[0], mp[1], mp[2]), q8::max3n(mp[3], mp[4], mp[5]), q8::max2n(mp[6], mp[7])) * c;
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
            const bool blind = it->list != nullptr && *my_groups == 0;   // the row's set is empty
            if (blind) {
                m_run = -INFINITY;
                l_run = 0.f;
            } else if (m_run == -INFINITY && l_run == l_run) {
                l_run = 0.f;                          // the row saw nothing (a NaN stays the mark of a row that saw one)
            }
            if (it->part != nullptr) {
                cut_epilogue(it->part + t * kPartFloats, r, tO, m_run, l_run, blind, live, bar(kOFree + t));
            } else {
                T* out_row = nullptr;
                if (live) {
                    const int32_t i = it->idx[it->row0 + t * kBM + r];
                    if (i >= 0 && i < p.n_tokens)
                        out_row = static_cast<T*>(it->out) + (int64_t)i * p.ld_out + (int64_t)it->head * kD;
                    else
                        atomicOr(&g_error_word, kErrBounds);
                }
                const float inv = l_run == 0.f ? 0.f : 1.0f / l_run;
#pragma unroll 1
                for (int h = 0; h < 4; ++h) {
                    uint32_t o[32];
                    FXR_TMEM_LD32(tO + h * 32u, o);
                    if (out_row != nullptr) {
                        uint4* dst = reinterpret_cast<uint4*>(out_row + 32 * h);
#pragma unroll
                        for (int q = 0; q < 4; ++q)
                            dst[q] = blind ? make_uint4(0, 0, 0, 0) : make_uint4(
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
