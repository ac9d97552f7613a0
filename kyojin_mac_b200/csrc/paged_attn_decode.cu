// Attention over a paged cache for few rows a request and head (single tokens: G rows of one token), bound by reading K and V once from HBM.
//
// Two CTAs an SM, each four consumer warps and a producer warp that keeps a ring of 64-key stages full with tiled copies (one per page piece for K and V; a key is 256
// bytes, the pieces lie anywhere). A consumer warp owns 16 keys of every stage and everything about them, so the loop has no barrier among warps: with
// mma.m16n8k16 it forms S^T = K Q^T (keys on the M side: 8 rows fill the N side, no padding up to G = 8), keeps its own reference maximum and sum per row, turns the
// weights around in registers (movmatrix) and accumulates O^T = V^T P^T. tcgen05 would compute 128 rows for 8; here the tensor work is a sixth of the time the bytes take.
// The reference maximum of a row moves only when a score passes it by 2^8 (bf16: 2^15; a warp vote), so the usual stage needs no shuffle and no rescaling.
// Measured, 64 / 8 heads of 128: 64 sequences of 1000 to 16000 tokens 329 us = 6.7 TB/s, one of 778 tokens 9.8 us (both launches); counters: DRAM 1.01 x the necessary bytes,
// issue slots 17 %. Requests of up to 16 rows come here, since their loop needs no more than the bytes' time; with 32 rows (four tokens of 8 heads, 8000 cached) the prefill
// kernel takes 368 us for 64 requests, where the bytes take 320, and this one would read the keys again for every 16 rows.
// Places that no row sees may hold anything: their weights are selected, not multiplied, to 0, and their values are cleared in the V fragments.
#include <algorithm>

#include "paged_attn.cuh"

namespace kyb {

constexpr int DC_TILE = 64, DC_WARPS = 4, DC_THREADS = 32 * (DC_WARPS + 1);

template <typename T> __device__ __forceinline__ void mma_16816(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1);
template <> __device__ __forceinline__ void mma_16816<__half>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) { mma16816(c, a0, a1, a2, a3, b0, b1); }
template <> __device__ __forceinline__ void mma_16816<__nv_bfloat16>(float (&c)[4], uint32_t a0, uint32_t a1, uint32_t a2, uint32_t a3, uint32_t b0, uint32_t b1) {
    asm volatile("mma.sync.aligned.m16n8k16.row.col.f32.bf16.bf16.f32 {%0,%1,%2,%3}, {%4,%5,%6,%7}, {%8,%9}, {%0,%1,%2,%3};"
                 : "+f"(c[0]), "+f"(c[1]), "+f"(c[2]), "+f"(c[3])
                 : "r"(a0), "r"(a1), "r"(a2), "r"(a3), "r"(b0), "r"(b1));
}
__device__ __forceinline__ void ldsm4(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ void ldsm4_t(uint32_t (&r)[4], uint32_t a) {
    asm volatile("ldmatrix.sync.aligned.m8n8.x4.trans.shared.b16 {%0,%1,%2,%3}, [%4];" : "=r"(r[0]), "=r"(r[1]), "=r"(r[2]), "=r"(r[3]) : "r"(a) : "memory");
}
__device__ __forceinline__ uint32_t turn8x8(uint32_t v) {
    uint32_t d;
    asm volatile("movmatrix.sync.aligned.m8n8.trans.b16 %0, %1;" : "=r"(d) : "r"(v));
    return d;
}
__device__ __forceinline__ void consumer_barrier() { asm volatile("bar.sync 1, 128;" ::: "memory"); }

template <int D, int NT>
struct DecodeShape {
    static constexpr int ROWS = 8 * NT, STAGE = DC_TILE * D * 4, STAGES = D == 128 ? 3 : 6;      // a stage: K and V of 64 keys
    static constexpr int OFF_O = STAGES * STAGE, O_LD = D + 4, OFF_ML = OFF_O + ROWS * O_LD * 4, OFF_BAR = OFF_ML + (2 * DC_WARPS + 2) * ROWS * 4, SMEM = OFF_BAR + 16 * STAGES + 64;
    static constexpr size_t PART = (size_t)ROWS * (D + 2);                                       // floats of a part
};

using DecodeRuns = Runs<1, 0>;
__device__ __forceinline__ int request_units(const AttnParams& p, int r, int block) {
    int base;
    const int tokens = request_rows(p, r, base), kv = request_keys(p, r), nb = row_blocks(p, tokens, block);
    int n = 0;
    for (int b = 0; b < nb; ++b) n += DecodeRuns::units(key_span(p, tokens, kv, block, b, DC_TILE));
    return n * p.hkv;
}

// First item and length of this CTA's run: every thread of the block takes part; the result is in *out (shared).
__device__ __forceinline__ void find_run(const AttnParams& p, int block, Cursor* out, int* sums, unsigned long long* rows, int threads) {
    const int tid = threadIdx.x, lane = tid & 31, warp = tid >> 5, warps = threads / 32;
    unsigned mine = 0, seen = 0;
    bool falls = false;
    for (int r = tid; r < p.batch; r += threads) {
        int base;
        seen += (unsigned)request_rows(p, r, base), falls |= offsets_fall(p, r);
        if (seen > (unsigned)p.tokens) {                                    // (the sum over a request's blocks is a loop: it ends here where offsets fall)
            falls = true;
            break;
        }
        mine += (unsigned)request_units(p, r, block);
    }
    const int first = (int)mine;                                            // (this thread's only request when there are no more of them than threads)
    mine = __reduce_add_sync(0xffffffffu, mine);
    if (lane == 0) sums[warp] = (int)mine;
    if (tid == 0) out->left = 0;
    if (__syncthreads_or(falls) && !rows_hold(p, rows)) return;
    int total = 0;
    for (int w = 0; w < warps; ++w) total += sums[w];
    const int ctas = min((int)gridDim.x, total), c = blockIdx.x;
    const int u0 = c < ctas ? run_border(total, ctas, c) : 0, u1 = c < ctas ? run_border(total, ctas, c + 1) : 0;
    __syncthreads();
    int before = 0;
    for (int r0 = 0; r0 < p.batch && u1 > u0 && before <= u0; r0 += threads) {
        const int r = r0 + tid;
        const int n = r < p.batch ? (p.batch <= threads ? first : request_units(p, r, block)) : 0;
        int end = n;
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const int x = __shfl_up_sync(0xffffffffu, end, d);
            if (lane >= d) end += x;
        }
        if (lane == 31) sums[warp] = end;
        __syncthreads();
        int all = before;
        for (int w = 0; w < warps; ++w) {
            if (w < warp) end += sums[w];
            all += sums[w];
        }
        end += before;
        if (u0 >= end - n && u0 < end) {
            Cursor k;
            int at = u0 - (end - n);
            k.r = r, k.rb = 0, k.left = u1 - u0;
            k.load(p, block, DC_TILE);
            while (at >= DecodeRuns::units(k.s) * p.hkv) at -= DecodeRuns::units(k.s) * p.hkv, ++k.rb, k.s = key_span(p, k.tokens, k.kv, block, k.rb, DC_TILE);
            k.h = at / DecodeRuns::units(k.s);
            k.at = DecodeRuns::enter(k.s, at - k.h * DecodeRuns::units(k.s), k.left);
            if (k.at == k.s.n) k.next(p, block, DC_TILE);
            *out = k;
        }
        before = all;
        __syncthreads();
    }
    __syncthreads();
}

template <typename T, int D, int NT>
__global__ void __launch_bounds__(DC_THREADS, 2) paged_attn_decode_kernel(const __grid_constant__ CUtensorMap map_k, const __grid_constant__ CUtensorMap map_v, const AttnParams p) {
    using S = DecodeShape<D, NT>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    __shared__ Cursor start;
    __shared__ int sums[DC_WARPS + 1];
    __shared__ unsigned long long rows;
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u;
    uint8_t* const smem_g = smem_raw + (smem0 - smem_u32(smem_raw));
    const uint32_t full0 = smem0 + S::OFF_BAR, empty0 = full0 + 8 * S::STAGES;
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::STAGES; ++s) mbar_init_a(full0 + 8 * s, 1), mbar_init_a(empty0 + 8 * s, DC_WARPS);
        mbar_fence_init();
        prefetch_tmap(&map_k);
        prefetch_tmap(&map_v);
    }
    pdl_wait();                                                              // what is above runs while the kernel before drains
    find_run(p, S::ROWS, &start, sums, &rows, DC_THREADS);
    Cursor c = start;
    pdl_launch_dependents();
    const int page = 1 << p.page_log2, piece = min(page, DC_TILE), piece_log2 = min(p.page_log2, 6), pieces = DC_TILE >> piece_log2;
    bool failed = false;

    if (warp == DC_WARPS) {
        // ---- producer: lane i looks up the page of the item's piece `base + i`; K and V of a piece are issued by two lanes
        int s = 0, issued = 0;
        uint32_t parity = 1;                                                // a fresh barrier passes a wait on the previous phase
        for (int run; (run = c.run<DecodeRuns>()) > 0;) {
            int base = -64, ids = 0;
            for (int i = c.at; i < c.at + run && !failed; ++i) {
                if ((i - base) * pieces >= 32 || base < 0) {                // the next 32 pieces' pages at once
                    base = i;
                    const int x = lane >> (6 - piece_log2), t = i + x, key = t < c.s.n ? c.s.tile(t) * DC_TILE + ((lane & (pieces - 1)) << piece_log2) : p.cap;
                    // a piece that no row sees is read as if it lay behind the cache: zeros
                    const bool seen = key < c.s.end && (key + piece > c.s.lo || key < p.sinks);
                    ids = seen ? p.table[c.r * p.ld_table + (key >> p.page_log2)] : p.pages;
                    if ((unsigned)ids >= (unsigned)p.pages) ids = p.pages;
                }
                if (!wait_warp(empty0 + 8 * s, parity)) {
                    failed = true;
                    break;
                }
                const uint32_t stage = smem0 + s * S::STAGE, bar = full0 + 8 * s;
                if (lane == 0) mbar_expect_tx_a(bar, S::STAGE);
                __syncwarp();
                const int j = lane >> 1, id = __shfl_sync(0xffffffffu, ids, (i - base) * pieces + (j & (pieces - 1)));
                if (j < pieces) {
                    const int y = (c.s.tile(i) * DC_TILE + (j << piece_log2)) & (page - 1);
                    tma_load_5d(stage + (lane & 1) * (S::STAGE / 2) + j * (piece * D * 2), (lane & 1) ? &map_v : &map_k, 0, y, 0, c.h, id, bar);
                }
                ++issued;
                if (++s == S::STAGES) s = 0, parity ^= 1u;
            }
            if (failed) break;
            c.advance<DecodeRuns>(p, S::ROWS, DC_TILE, run);
        }
        if (failed)                                                         // copies in flight end before the block does
            for (int k = 0; k < min(issued, S::STAGES); ++k) {
                const int at = issued - 1 - k;
                mbar_wait_fast(full0 + 8 * (at % S::STAGES), (uint32_t)(at / S::STAGES) & 1u);
            }
    } else {
        // ---- consumers
        const int g = lane >> 2, t = lane & 3;
        float* const so = reinterpret_cast<float*>(smem_g + S::OFF_O);       // [row][D + 4]
        float* const sm = reinterpret_cast<float*>(smem_g + S::OFF_ML);      // [warp][row] maxima, then [warp][row] sums, then [row] maximum and sum of the item
        float* const sl = sm + DC_WARPS * S::ROWS;
        float* const sml = sl + DC_WARPS * S::ROWS;
        // ldmatrix source of this lane: its row of the warp's 16 keys, 16-byte chunk (column, swizzled) added per step
        const int k_row = lane & 15, v_row = ((lane >> 4) << 3) + (lane & 7), key_w = warp * 16;
        const uint32_t row_off = (uint32_t)((key_w >> piece_log2) * (piece * D * 2)), in_piece = (uint32_t)(key_w & (piece - 1));
        const uint32_t k_off = row_off + (in_piece + k_row) * 128u, v_off = (uint32_t)(S::STAGE / 2) + row_off + (in_piece + v_row) * 128u;
        const uint32_t half_step = (uint32_t)piece * 128u;
        int s = 0;
        uint32_t parity = 0;
        int4 begun = make_int4(0, 0, 0, 0);
        int flags = 0;
        for (int run; (run = c.run<DecodeRuns>()) > 0;) {
            const int from = c.at;
            uint32_t qf[NT][D / 16][2];
            int pos[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                const int row = c.s.row0 + 8 * n + g, tok = row / p.group;
                const bool on = 8 * n + g < c.s.rows;
                const T* q = reinterpret_cast<const T*>(p.q) + (int64_t)(c.row_base + (on ? tok : 0)) * p.q_t + (int64_t)(c.h * p.group + (on ? row - tok * p.group : 0)) * p.q_h;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    qf[n][k][0] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t) : 0u;
                    qf[n][k][1] = on ? *reinterpret_cast<const uint32_t*>(q + 16 * k + 2 * t + 8) : 0u;
                }
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int rr = 8 * n + 2 * t + e;
                    pos[n][e] = rr < c.s.rows ? c.kv - c.tokens + (c.s.row0 + rr) / p.group : -1;
                }
            }
            float o[D / 16][NT][4], m[NT][2], l[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n) {
                m[n][0] = m[n][1] = -INFINITY, l[n][0] = l[n][1] = 0.f;
#pragma unroll
                for (int d = 0; d < D / 16; ++d) o[d][n][0] = o[d][n][1] = o[d][n][2] = o[d][n][3] = 0.f;
            }
            for (int i = from; i < from + run; ++i) {
                if (!failed && !wait_warp(full0 + 8 * s, parity)) failed = true;
                const uint32_t stage = smem0 + s * S::STAGE;
                const int key0 = c.s.tile(i) * DC_TILE, kw = key0 + key_w;
                // every row sees every key of the tile, or the tile needs its masks
                const bool plain = key0 + DC_TILE <= min(c.s.first + 1, p.cap) && (!p.window || key0 > c.s.last - p.window);
                float x[NT][4];
#pragma unroll
                for (int n = 0; n < NT; ++n) x[n][0] = x[n][1] = x[n][2] = x[n][3] = 0.f;
#pragma unroll
                for (int k = 0; k < D / 16; ++k) {
                    uint32_t a[4];
                    const int ch = 2 * k + (lane >> 4);
                    ldsm4(a, stage + k_off + (ch >> 3) * half_step + (uint32_t)(((ch & 7) ^ (k_row & 7)) << 4));
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<T>(x[n], a[0], a[1], a[2], a[3], qf[n][k][0], qf[n][k][1]);
                }
                uint32_t live[2] = {0xffffffffu, 0xffffffffu};
                if (plain) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) x[n][e] *= p.scale2;
                } else {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 4; ++e) {
                            const int j = kw + g + (e >> 1) * 8, at = pos[n][e & 1];
                            const bool see = j <= at && j < p.cap && (!p.window || j > at - p.window || j < p.sinks);
                            x[n][e] = see ? x[n][e] * p.scale2 : -INFINITY;
                        }
#pragma unroll
                    for (int e = 0; e < 2; ++e) {
                        const int j = kw + 2 * t + 8 * e;
                        live[e] = (c.s.alive(j, p.sinks) ? 0xffffu : 0u) | (c.s.alive(j + 1, p.sinks) ? 0xffff0000u : 0u);
                    }
                }
                bool over = false;
#pragma unroll
                for (int n = 0; n < NT; ++n)
#pragma unroll
                    for (int e = 0; e < 2; ++e) over |= fmaxf(x[n][e], x[n][2 + e]) > m[n][e] + Weights<T>::move;
                if (__any_sync(0xffffffffu, over)) {
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int e = 0; e < 2; ++e) {
                            float top = fmaxf(fmaxf(x[n][e], x[n][2 + e]), m[n][e]);
#pragma unroll
                            for (int d = 4; d < 32; d <<= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
                            const float f = m[n][e] == -INFINITY ? 0.f : exp2_fast(m[n][e] - top);
                            m[n][e] = top, l[n][e] *= f;
#pragma unroll
                            for (int d = 0; d < D / 16; ++d) o[d][n][e] *= f, o[d][n][2 + e] *= f;
                        }
                }
                uint32_t pf[NT][2];
#pragma unroll
                for (int n = 0; n < NT; ++n) {
                    const float m0 = m[n][0] == -INFINITY ? 0.f : m[n][0] - Weights<T>::below, m1 = m[n][1] == -INFINITY ? 0.f : m[n][1] - Weights<T>::below;
                    const float a = exp2_fast(x[n][0] - m0), b = exp2_fast(x[n][1] - m1), u = exp2_fast(x[n][2] - m0), w = exp2_fast(x[n][3] - m1);
                    l[n][0] += a + u, l[n][1] += b + w;
                    pf[n][0] = turn8x8(pack2<T>(a, b)), pf[n][1] = turn8x8(pack2<T>(u, w));
                }
#pragma unroll
                for (int d = 0; d < D / 16; ++d) {
                    uint32_t a[4];
                    const int ch = 2 * d + ((lane >> 3) & 1);
                    ldsm4_t(a, stage + v_off + (ch >> 3) * half_step + (uint32_t)(((ch & 7) ^ (v_row & 7)) << 4));
                    if (!plain) a[0] &= live[0], a[1] &= live[0], a[2] &= live[1], a[3] &= live[1];
#pragma unroll
                    for (int n = 0; n < NT; ++n) mma_16816<T>(o[d][n], a[0], a[1], a[2], a[3], pf[n][0], pf[n][1]);
                }
                __syncwarp();
                if (lane == 0) mbar_arrive_a(empty0 + 8 * s);
                if (++s == S::STAGES) s = 0, parity ^= 1u;
            }
            // ---- the warps' sums meet in shared memory, in warp order
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
#pragma unroll
                    for (int d = 4; d < 32; d <<= 1) l[n][e] += __shfl_xor_sync(0xffffffffu, l[n][e], d);
                    if (g == 0) sm[warp * S::ROWS + 8 * n + 2 * t + e] = m[n][e], sl[warp * S::ROWS + 8 * n + 2 * t + e] = l[n][e];
                }
            consumer_barrier();
            float f[NT][2];
#pragma unroll
            for (int n = 0; n < NT; ++n)
#pragma unroll
                for (int e = 0; e < 2; ++e) {
                    const int row = 8 * n + 2 * t + e;
                    float top = -INFINITY, sum = 0.f;
#pragma unroll
                    for (int w = 0; w < DC_WARPS; ++w) top = fmaxf(top, sm[w * S::ROWS + row]);
#pragma unroll
                    for (int w = 0; w < DC_WARPS; ++w) sum += sm[w * S::ROWS + row] == -INFINITY ? 0.f : sl[w * S::ROWS + row] * exp2_fast(sm[w * S::ROWS + row] - top);
                    f[n][e] = m[n][e] == -INFINITY ? 0.f : exp2_fast(m[n][e] - top);
                    if (warp == 0 && g == 0) sml[row] = top, sml[S::ROWS + row] = sum;
                }
            for (int w = 0; w < DC_WARPS; ++w) {
                if (w == warp)
#pragma unroll
                    for (int n = 0; n < NT; ++n)
#pragma unroll
                        for (int d = 0; d < D / 16; ++d)
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                float* const at = so + (8 * n + 2 * t + (e & 1)) * S::O_LD + 16 * d + g + 8 * (e >> 1);
                                const float v = o[d][n][e] * f[n][e & 1];
                                *at = w ? *at + v : v;
                            }
                consumer_barrier();
            }
            const bool whole = from == 0 && run == c.s.n;
            if (whole) {
                for (int x = threadIdx.x; x < c.s.rows * (D / 8); x += 32 * DC_WARPS) {
                    const int rr = x / (D / 8), col = (x % (D / 8)) * 8, row = c.s.row0 + rr, tok = row / p.group;
                    const float sum = sml[S::ROWS + rr], inv = sum > 0.f ? 1.f / sum : 0.f;
                    const float4 a = *reinterpret_cast<const float4*>(so + rr * S::O_LD + col), b = *reinterpret_cast<const float4*>(so + rr * S::O_LD + col + 4);
                    uint4 w;
                    w.x = pack2<T>(a.x * inv, a.y * inv), w.y = pack2<T>(a.z * inv, a.w * inv), w.z = pack2<T>(b.x * inv, b.y * inv), w.w = pack2<T>(b.z * inv, b.w * inv);
                    if (!failed)
                        *reinterpret_cast<uint4*>(reinterpret_cast<T*>(p.o) + (int64_t)(c.row_base + tok) * p.o_t + (int64_t)(c.h * p.group + row - tok * p.group) * p.o_h + col) = w;
                }
            } else {
                float* const part = p.parts + ((size_t)blockIdx.x * 2 + (from == 0)) * S::PART;
                for (int x = threadIdx.x; x < S::ROWS * (D / 4); x += 32 * DC_WARPS) {
                    const int rr = x / (D / 4), col = (x % (D / 4)) * 4;
                    *reinterpret_cast<float4*>(part + rr * D + col) = *reinterpret_cast<const float4*>(so + rr * S::O_LD + col);
                }
                for (int x = threadIdx.x; x < 2 * S::ROWS; x += 32 * DC_WARPS) part[S::ROWS * D + x] = sml[x];
                flags |= from == 0 ? NOTE_BEGINS : NOTE_CONTINUES | (from + run == c.s.n ? NOTE_ENDS : 0);
            }
            if (!whole && from == 0) begun = make_int4(c.r, c.rb, c.h, 0);   // the last item of the run
            c.advance<DecodeRuns>(p, S::ROWS, DC_TILE, run);
            consumer_barrier();                                              // the buffers are read
        }
        if (threadIdx.x == 0) p.notes[blockIdx.x] = make_int4(begun.x, begun.y, begun.z, flags);
    }
    if (failed) atomicExch(p.status, KYB_DEV_TIMEOUT_ATTN);
}

// The parts of the items that begin in run blockIdx.x and end in a later one: o = sum_i 2^(m_i - m) o_i / sum_i 2^(m_i - m) l_i, in a fixed order. PER_ROW warps a row,
// each with every PER_ROW-th part; a lane holds D / 32 of the row's values, the parts' maxima and sums are read 32 at a time. After the decode kernel a row may have a part from
// each of 296 runs (one long context, one key-value head): a block of four warps per row then, so that several SMs read the parts' megabyte (125 000 keys of one head 44 -> 31 us
// in all; eight warps 25, but 1 to 2 us more for every call with little to join). After the prefill kernel it has a few, and a block takes eight of up to 256 rows: many blocks
// that find nothing cost more.
template <typename T, int D, int JOIN_WARPS, int PER_ROW>
__global__ void __launch_bounds__(32 * JOIN_WARPS) paged_attn_join_kernel(const AttnParams p, const int ctas, const int block) {
    constexpr int E = D / 32;
    __shared__ float meet[PER_ROW > 1 ? JOIN_WARPS : 1][D + 1];
    pdl_launch_dependents();
    pdl_wait();
    const int first = blockIdx.x, lane = threadIdx.x & 31, warp = threadIdx.x >> 5, share = warp % PER_ROW;
    const int4 note = p.notes[first];
    const int rr = blockIdx.y * (JOIN_WARPS / PER_ROW) + warp / PER_ROW;
    if (!(note.w & NOTE_BEGINS) || rr >= block) return;
    int row_base;
    const int tokens = request_rows(p, note.x, row_base), row = note.y * block + rr, tok = row / p.group;
    if (tok >= tokens) return;
    const size_t size = (size_t)block * (D + 2);
    int n = 1;                                                               // parts: up to the run that ends the item
    for (bool more = true; more && first + n < ctas;) {
        const int i = first + n + lane;
        const uint32_t ends = __ballot_sync(0xffffffffu, i >= ctas || (p.notes[i].w & NOTE_ENDS));
        n += ends ? __ffs(ends) : 32, more = !ends;
    }
    n = min(n, ctas - first);
    auto part = [&](int i) { return p.parts + ((size_t)(first + i) * 2 + (i == 0)) * size; };
    float top = -INFINITY;
    for (int i = lane; i < n; i += 32) top = fmaxf(top, part(i)[(size_t)block * D + rr]);
#pragma unroll
    for (int d = 16; d; d >>= 1) top = fmaxf(top, __shfl_xor_sync(0xffffffffu, top, d));
    float o[E] = {}, sum = 0.f;
    const int mine = (n - share + PER_ROW - 1) / PER_ROW;                    // parts share, share + PER_ROW, ...
    for (int i0 = 0; i0 < mine; i0 += 32) {
        const int i = share + (i0 + lane) * PER_ROW;
        float w = 0.f;
        if (i0 + lane < mine) {
            const float* const x = part(i) + (size_t)block * D + rr;
            w = x[0] == -INFINITY ? 0.f : exp2f(x[0] - top);
            sum += w * x[block];
        }
        const int k = min(32, mine - i0);
#pragma unroll 4
        for (int j = 0; j < k; ++j) {
            const float* const x = part(share + (i0 + j) * PER_ROW) + (size_t)rr * D + lane * E;
            const float wj = __shfl_sync(0xffffffffu, w, j);
            if constexpr (E == 4) {
                const float4 v = *reinterpret_cast<const float4*>(x);
                o[0] += wj * v.x, o[1] += wj * v.y, o[2] += wj * v.z, o[3] += wj * v.w;
            } else {
                const float2 v = *reinterpret_cast<const float2*>(x);
                o[0] += wj * v.x, o[1] += wj * v.y;
            }
        }
    }
#pragma unroll
    for (int d = 16; d; d >>= 1) sum += __shfl_xor_sync(0xffffffffu, sum, d);
    if constexpr (PER_ROW > 1) {                                             // (all warps of a row's block come here or none)
#pragma unroll
        for (int e = 0; e < E; ++e) meet[warp][lane * E + e] = o[e];
        if (lane == 0) meet[warp][D] = sum;
        __syncthreads();
        if (share) return;
        for (int w = 1; w < PER_ROW; ++w) {
#pragma unroll
            for (int e = 0; e < E; ++e) o[e] += meet[warp + w][lane * E + e];
            sum += meet[warp + w][D];
        }
    }
    const float inv = sum > 0.f ? 1.f / sum : 0.f;
    T* const out = reinterpret_cast<T*>(p.o) + (int64_t)(row_base + tok) * p.o_t + (int64_t)(note.z * p.group + row - tok * p.group) * p.o_h + lane * E;
#pragma unroll
    for (int e = 0; e < E; e += 2) reinterpret_cast<uint32_t*>(out)[e / 2] = pack2<T>(o[e] * inv, o[e + 1] * inv);
}

}  // namespace kyb

namespace {

constexpr int DC_PER_SM = 2;

template <typename T, int D, int NT>
int launch_decode(KybAttnCall& c, void* ws) {
    using S = kyb::DecodeShape<D, NT>;
    auto kern = kyb::paged_attn_decode_kernel<T, D, NT>;
    if (int rc = kyb_allow_smem((const void*)kern)) return rc;
    const int64_t units = kyb_attn_units(c, S::ROWS, kyb::DC_TILE);
    KYB_REQUIRE(units, "more than 2^31 key tiles in one call: split it");
    const int ctas = (int)std::min<int64_t>(DC_PER_SM * c.sms, units), piece = std::min(c.page, kyb::DC_TILE);
    CUtensorMap mk, mv;
    if (int rc = kyb_make_cache_map(&mk, c.k, c.dtype, c.p.pages, c.p.hkv, c.page, D, c.k_p, c.k_h, piece, D / 64)) return rc;
    if (int rc = kyb_make_cache_map(&mv, c.v, c.dtype, c.p.pages, c.p.hkv, c.page, D, c.v_p, c.v_h, piece, D / 64)) return rc;
    c.p.notes = (int4*)ws, c.p.parts = (float*)((char*)ws + (size_t)ctas * sizeof(int4));
    if (int rc = kyb_launch_chained(kern, ctas, kyb::DC_THREADS, S::SMEM + 1024, c.st, mk, mv, c.p)) return rc;
    return kyb_attn_join(c, ctas, S::ROWS);
}

}  // namespace

size_t kyb_attn_decode_scratch(int d, int rows, int sms) {
    const size_t block = rows <= 8 ? 8 : 16;
    return (size_t)DC_PER_SM * sms * (sizeof(int4) + 2 * block * (d + 2) * sizeof(float));
}

int kyb_attn_decode(KybAttnCall& c, int rows, void* ws) {
    const bool wide = rows > 8;
    if (c.dtype == 1) {
        if (c.d == 64) return wide ? launch_decode<__half, 64, 2>(c, ws) : launch_decode<__half, 64, 1>(c, ws);
        return wide ? launch_decode<__half, 128, 2>(c, ws) : launch_decode<__half, 128, 1>(c, ws);
    }
    if (c.d == 64) return wide ? launch_decode<__nv_bfloat16, 64, 2>(c, ws) : launch_decode<__nv_bfloat16, 64, 1>(c, ws);
    return wide ? launch_decode<__nv_bfloat16, 128, 2>(c, ws) : launch_decode<__nv_bfloat16, 128, 1>(c, ws);
}

template <typename T, int D>
static int launch_join(const KybAttnCall& c, int ctas, int block) {
    cudaLaunchConfig_t cfg = {};
    const bool few = block <= KYB_DECODE_ROWS;
    cfg.gridDim = dim3((unsigned)ctas, (unsigned)(few ? block : (block + 7) / 8)), cfg.blockDim = dim3(few ? 128 : 256), cfg.stream = c.st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    if (few) KYB_CUDA(cudaLaunchKernelEx(&cfg, kyb::paged_attn_join_kernel<T, D, 4, 4>, c.p, ctas, block));
    else KYB_CUDA(cudaLaunchKernelEx(&cfg, kyb::paged_attn_join_kernel<T, D, 8, 1>, c.p, ctas, block));
    return kyb_launch_check("paged_attn_join");
}

int kyb_attn_join(const KybAttnCall& c, int ctas, int block) {
    if (c.dtype == 1) return c.d == 64 ? launch_join<__half, 64>(c, ctas, block) : launch_join<__half, 128>(c, ctas, block);
    return c.d == 64 ? launch_join<__nv_bfloat16, 64>(c, ctas, block) : launch_join<__nv_bfloat16, 128>(c, ctas, block);
}
