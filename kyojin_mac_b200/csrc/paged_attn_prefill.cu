// Attention over a paged cache for many rows a request and head (chunks of prompts, whole prompts), bound by the tensor cores and the exponentials.
//
// One persistent CTA an SM. A row block is two query tiles of 128 / G tokens (G query heads each: up to 128 rows, so the heads of a group share every key). Warps:
//   0-3, 4-7   softmax of the first and the second query tile, one row a thread
//   8          producer: query tiles, and a ring of 128-key tiles of K and V by tiled copies (one per page piece and half of the values)
//   9          tcgen05.mma issuer
//   10         clears values in places that no row sees (11 is idle: registers move between groups of four warps, from these four to the softmax)
// Tensor memory: S0 | S1 | O0 | O1, 128 columns each; the weights P (16 bits) take the place of their scores S. S = Q K^T with both operands in shared memory; O += P V with
// P in tensor memory and V as it lies in the cache (MN-major operand). The issuer's order S0(j+1) behind O0(j), S1(j+1) behind O1(j) keeps the tensor cores busy
// with one query tile while the softmax of the other runs; S(j+1) may overwrite P(j) without a wait in between, since one thread issues both products to the SM's one tensor
// core, which runs them in that order. An item's last O has a barrier of its own: on the scores' one the next item's first scores, which wait for nothing of the softmax, could end
// a second phase before a late softmax warp has seen the first, and a wait by parity would not pass any more. A row's reference maximum moves only when a score passes it by
// 2^8 (bf16: 2^15), so O is rescaled (by the softmax warps themselves, in tensor memory) hardly ever; sums are of the unrounded weights, in 32 bits.
// Measured, 64 / 8 heads of 128: 1024 tokens on 8192 cached ones 241 to 250 us, a prompt of 8192 tokens 910 us = 1210 TFLOP/s; 3200 clocks a pair of tiles, of which the tensor
// cores and the special-function units are busy 2050 each.
// Keys that a row does not see are masked by selection in the tiles at the borders; values in places that no row of the block sees are cleared in shared memory, since such
// places may hold anything and 0 times NaN is NaN.
#include <algorithm>
#include <type_traits>

#include "paged_attn.cuh"

namespace kyb {

constexpr int PF_TILE = 128, PF_THREADS = 384;

// An item costs about two tiles beyond its own (query load, the first scores, the last values, the output). Measured over nine shapes from 20 to 4001 new tokens: two and a
// snap of one on average 1 % faster than three, with eight prompts of 2048 tokens take 96 instead of 85 us.
using PrefillRuns = Runs<2, 1>;

template <int D>
struct PrefillShape {
    static constexpr uint32_t HALVES = D / 64, HALF = 128 * 128, TILE = HALVES * HALF;       // a tile of 128 rows: halves of 64 values, 128-byte rows
    static constexpr int SLOTS = 4 * 128 / D;                                // an even number: K in the even ones, V in the odd ones
    static constexpr uint32_t OFF_KV = 2 * TILE, OFF_OUT = OFF_KV + SLOTS * TILE, OFF_BAR = OFF_OUT + 8 * 4096, OFF_CUR = OFF_BAR + 24 * SLOTS + 96, SMEM = OFF_CUR + 8 * sizeof(Cursor);
};

__device__ __forceinline__ void tmem_st_16(uint32_t taddr, const uint32_t (&v)[16]) {
    asm volatile("tcgen05.st.sync.aligned.32x32b.x16.b32 [%0], {%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15,%16};" ::"r"(taddr), "r"(v[0]), "r"(v[1]), "r"(v[2]), "r"(v[3]), "r"(v[4]),
                 "r"(v[5]), "r"(v[6]), "r"(v[7]), "r"(v[8]), "r"(v[9]), "r"(v[10]), "r"(v[11]), "r"(v[12]), "r"(v[13]), "r"(v[14]), "r"(v[15])
                 : "memory");
}
__device__ __forceinline__ void tmem_ld_16(uint32_t taddr, uint32_t (&v)[16]) {
    asm volatile("tcgen05.ld.sync.aligned.32x32b.x16.b32 {%0,%1,%2,%3,%4,%5,%6,%7,%8,%9,%10,%11,%12,%13,%14,%15}, [%16];"
                 : "=r"(v[0]), "=r"(v[1]), "=r"(v[2]), "=r"(v[3]), "=r"(v[4]), "=r"(v[5]), "=r"(v[6]), "=r"(v[7]), "=r"(v[8]), "=r"(v[9]), "=r"(v[10]), "=r"(v[11]), "=r"(v[12]), "=r"(v[13]),
                   "=r"(v[14]), "=r"(v[15])
                 : "r"(taddr)
                 : "memory");
}
__device__ __forceinline__ void tmem_st_wait_all() { asm volatile("tcgen05.wait::st.sync.aligned;" ::: "memory"); }

// O[tmem] (+)= P[tmem] * V[smem], issued by one thread
__device__ __forceinline__ void umma_f16_ts(uint32_t tmem_d, uint32_t tmem_a, uint64_t bdesc, uint32_t idesc, uint32_t accumulate) {
    asm volatile(
        "{\n\t.reg .pred p;\n\tsetp.ne.b32 p, %4, 0;\n\t"
        "tcgen05.mma.cta_group::1.kind::f16 [%0], [%1], %2, %3, p;\n\t}" ::"r"(tmem_d),
        "r"(tmem_a), "l"(bdesc), "r"(idesc), "r"(accumulate)
        : "memory");
}
// MN-major operand (V: [key][value], 128-byte swizzle): 64-value column blocks HALF bytes apart (leading offset), groups of 8 keys 1024 bytes apart (stride offset)
__device__ __forceinline__ uint64_t umma_desc_mn128(uint32_t smem_addr, uint32_t half) {
    return (uint64_t)((smem_addr & 0x3FFFFu) >> 4) | ((uint64_t)(half >> 4) << 16) | ((uint64_t)(1024 >> 4) << 32) | ((uint64_t)1 << 46) | ((uint64_t)2 << 61);
}

// The bounded wait of this kernel, inline: a call would bind the caller to a calling convention's registers, which do not go with registers that move between warps.
__device__ __forceinline__ bool wait_here(uint32_t bar, uint32_t parity) {
    uint32_t ok = 0;
#pragma unroll 1
    for (uint32_t i = 0; i < (1u << 22); ++i) {
        asm volatile("{\n\t.reg .pred p;\n\tmbarrier.try_wait.parity.shared::cta.b64 p, [%1], %2;\n\tselp.u32 %0, 1, 0, p;\n\t}" : "=r"(ok) : "r"(bar), "r"(parity) : "memory");
        if (ok) break;
        if (i > 64) __nanosleep(64);
    }
    return __all_sync(0xffffffffu, ok);
}

struct RunFinder {
    unsigned long long rows;
    int tokens[PF_THREADS], kv[PF_THREADS], blocks_end[PF_THREADS], units[PF_THREADS], sums[2][PF_THREADS / 32];
    Cursor run;
    int at, request;
};
// inclusive sum over the block; two calls in a row use two places for the warps' sums, so that one barrier a call is enough
__device__ __forceinline__ int scan_block(int v, int* sums, int& total) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const int x = __shfl_up_sync(0xffffffffu, v, d);
        if (lane >= d) v += x;
    }
    if (lane == 31) sums[warp] = v;
    __syncthreads();
    total = 0;
#pragma unroll
    for (int w = 0; w < PF_THREADS / 32; ++w) {
        if (w < warp) v += sums[w];
        total += sums[w];
    }
    return v;
}
// rows, keys and (scanned) row blocks of up to PF_THREADS requests from r0 on, for all threads; gives the number of their row blocks (-1: the requests own more rows than there are)
__device__ __forceinline__ int load_chunk(const AttnParams& p, int block, int r0, RunFinder& f) {
    const int tid = threadIdx.x, n = min(PF_THREADS, p.batch - r0);
    int nb = 0;
    bool falls = false;
    if (tid < n) {
        falls = offsets_fall(p, r0 + tid);
        int base;
        f.tokens[tid] = request_rows(p, r0 + tid, base), f.kv[tid] = request_keys(p, r0 + tid);
        nb = row_blocks(p, f.tokens[tid], block);
    }
    int all;
    f.blocks_end[tid] = scan_block(nb, f.sums[0], all);
    return __syncthreads_or(falls) && !rows_hold(p, &f.rows) ? -1 : all;
}
// their units, of all heads: the row blocks of all of them are shared among the threads (-1 as above)
__device__ __forceinline__ int count_chunk(const AttnParams& p, int block, int r0, RunFinder& f, int& end) {
    const int tid = threadIdx.x, n = min(PF_THREADS, p.batch - r0);
    f.units[tid] = 0;
    const int all = load_chunk(p, block, r0, f);
    if (all < 0) return -1;
    for (int i0 = tid & ~31; i0 < all; i0 += PF_THREADS) {                   // whole numbers: the order of the additions does not matter
        const int i = min(i0 + (tid & 31), all - 1), r = first_above(f.blocks_end, n, i), rb = i - (r ? f.blocks_end[r - 1] : 0);
        const int u = i0 + (tid & 31) < all ? PrefillRuns::units(key_span(p, f.tokens[r], f.kv[r], block, rb, PF_TILE)) * p.hkv : 0;
        const int r_first = __shfl_sync(0xffffffffu, r, 0);
        if (__all_sync(0xffffffffu, r == r_first)) {                         // one request's blocks, as usual: one addition for the warp
            const int sum = __reduce_add_sync(0xffffffffu, u);
            if ((tid & 31) == 0) atomicAdd(&f.units[r], sum);
        } else if (u) atomicAdd(&f.units[r], u);
    }
    __syncthreads();
    int total;
    end = scan_block(f.units[tid], f.sums[1], total);
    return total;
}
// a run that starts x units into row block rb of request r (whose items have `one` units each) and has `length` units
__device__ __forceinline__ void enter_run(const AttnParams& p, int block, Cursor& k, int r, int rb, int x, int one, int length) {
    k.r = r, k.rb = rb, k.left = length;
    k.load(p, block, PF_TILE);
    k.h = x / one;
    k.at = PrefillRuns::enter(k.s, x - k.h * one, k.left);
    if (k.at == k.s.n) k.next(p, block, PF_TILE);
}
// The run of tiles of CTA blockIdx.x, into f.run. FEW: with the short way for few row blocks (32 tokens 15.3 -> 13.9 us). The kernel for heads of 64 does without: with it there
// the compiler orders the softmax loop so that it runs 6 % slower (1024 tokens on 8192: 206 -> 219 us; 32 tokens 14.2 -> 12.7).
template <bool FEW>
__device__ __forceinline__ void find_run_wide(const AttnParams& p, int block, RunFinder& f) {
    const int tid = threadIdx.x, c = blockIdx.x;
    if (tid == 0) f.run.left = 0, f.request = 0, f.at = 0;
    if (FEW && p.batch <= PF_THREADS) {
        const int all = load_chunk(p, block, 0, f);
        if (all < 0) return;
        if (all <= PF_THREADS) {                                             // a row block a thread: one more scan gives the sums and the place
            const int r = tid < all ? first_above(f.blocks_end, p.batch, tid) : 0, rb = tid - (r ? f.blocks_end[r - 1] : 0);
            const int one = tid < all ? PrefillRuns::units(key_span(p, f.tokens[r], f.kv[r], block, rb, PF_TILE)) : 0, n = one * p.hkv;
            int total;
            const int e = scan_block(n, f.sums[1], total), ctas = min((int)gridDim.x, total);
            if (c >= ctas) return;
            const int u0 = run_border(total, ctas, c);
            if (n && u0 >= e - n && u0 < e) enter_run(p, block, f.run, r, rb, u0 - (e - n), one, run_border(total, ctas, c + 1) - u0);
            return;
        }
        __syncthreads();
    }
    int total = 0, end = 0, mine = 0;
    for (int r0 = 0; r0 < p.batch; r0 += PF_THREADS) {
        if (r0) __syncthreads();
        mine = count_chunk(p, block, r0, f, end), total += mine;
        if (mine < 0) return;
    }
    const int ctas = min((int)gridDim.x, total);
    const int u0 = c < ctas ? run_border(total, ctas, c) : 0, u1 = c < ctas ? run_border(total, ctas, c + 1) : 0;
    if (u1 == u0) return;
    __syncthreads();
    int before = 0;
    for (int r0 = 0; r0 < p.batch && before <= u0; r0 += PF_THREADS) {
        if (p.batch > PF_THREADS) {
            __syncthreads();
            mine = count_chunk(p, block, r0, f, end);
        }
        const int e = before + end, n = f.units[tid];
        if (n && u0 >= e - n && u0 < e) f.request = r0 + tid, f.at = u0 - (e - n);
        before += mine;
    }
    __syncthreads();
    const int r = f.request, at = f.at;
    int base;
    const int tokens = request_rows(p, r, base), kv = request_keys(p, r), nb = row_blocks(p, tokens, block);
    before = 0;
    for (int b0 = 0; b0 < nb && before <= at; b0 += PF_THREADS) {
        const int rb = b0 + tid, one = rb < nb ? PrefillRuns::units(key_span(p, tokens, kv, block, rb, PF_TILE)) : 0, n = one * p.hkv;
        int all;
        const int e = before + scan_block(n, f.sums[b0 / PF_THREADS & 1], all);
        if (n && at >= e - n && at < e) enter_run(p, block, f.run, r, rb, at - (e - n), one, u1 - u0);
        before += all;
    }
}

// pairs of 32-bit values in one register pair
__device__ __forceinline__ uint64_t pair_of(float a, float b) {
    uint64_t d;
    asm("mov.b64 %0, {%1, %2};" : "=l"(d) : "f"(a), "f"(b));
    return d;
}
__device__ __forceinline__ void split_pair(uint64_t v, float& a, float& b) { asm("mov.b64 {%0, %1}, %2;" : "=f"(a), "=f"(b) : "l"(v)); }
__device__ __forceinline__ uint64_t fma_pair(uint64_t a, uint64_t b, uint64_t c) {
    uint64_t d;
    asm("fma.rn.f32x2 %0, %1, %2, %3;" : "=l"(d) : "l"(a), "l"(b), "l"(c));
    return d;
}
__device__ __forceinline__ uint64_t add_pair(uint64_t a, uint64_t b) {
    uint64_t d;
    asm("add.rn.f32x2 %0, %1, %2;" : "=l"(d) : "l"(a), "l"(b));
    return d;
}
__device__ __forceinline__ float max3(float a, float b, float c) {
    float d;
    asm("max.f32 %0, %1, %2, %3;" : "=f"(d) : "f"(a), "f"(b), "f"(c));
    return d;
}

template <typename T, int D>
__global__ void __launch_bounds__(PF_THREADS, 1) paged_attn_prefill_kernel(const __grid_constant__ CUtensorMap map_q, const __grid_constant__ CUtensorMap map_k,
                                                                           const __grid_constant__ CUtensorMap map_v, const AttnParams p, const int qtoks) {
    using S = PrefillShape<D>;
    extern __shared__ __align__(1024) uint8_t smem_raw[];
    const uint32_t smem0 = (smem_u32(smem_raw) + 1023u) & ~1023u, kv0 = smem0 + S::OFF_KV;
    const uint32_t full0 = smem0 + S::OFF_BAR, empty0 = full0 + 8 * S::SLOTS, clean0 = empty0 + 8 * S::SLOTS, qfull = clean0 + 8 * S::SLOTS, qempty = qfull + 8, sfull0 = qfull + 16,
                   pfull0 = qfull + 32, phalf0 = qfull + 48, ofull0 = qfull + 64, tmem_slot = qfull + 80;      // pfull, phalf: the weights of a tile's first and second 64 keys
    const int warp = threadIdx.x >> 5, lane = threadIdx.x & 31;
    const int qrows = qtoks * p.group, block = 2 * qrows;                    // rows of a query tile, of a row block
    if (threadIdx.x == 0) {
        for (int s = 0; s < S::SLOTS; ++s) mbar_init_a(full0 + 8 * s, 1), mbar_init_a(empty0 + 8 * s, 1), mbar_init_a(clean0 + 8 * s, 1);
        mbar_init_a(qfull, 1), mbar_init_a(qempty, 1);
        for (int w = 0; w < 2; ++w) mbar_init_a(sfull0 + 8 * w, 1), mbar_init_a(pfull0 + 8 * w, 4), mbar_init_a(phalf0 + 8 * w, 4), mbar_init_a(ofull0 + 8 * w, 1);
        mbar_fence_init();
        prefetch_tmap(&map_q), prefetch_tmap(&map_k), prefetch_tmap(&map_v);
    }
    if (warp == 9) tmem_alloc(tmem_slot, 512);
    tc_fence_before();
    __syncthreads();
    tc_fence_after();
    const uint32_t tmem = lds32(tmem_slot);
    RunFinder& finder = *reinterpret_cast<RunFinder*>(smem_raw + (kv0 - smem_u32(smem_raw)));       // where the ring will be
    find_run_wide<D != 64>(p, block, finder);
    __syncthreads();
    const Cursor c0 = finder.run;
    asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
    __syncthreads();
    pdl_launch_dependents();
    bool failed = false;

    // registers move from the producer's group of four warps to the softmax groups: 72 + 2 x 216 = 3 x 168, what the block was launched with
    if (warp >= 8) {
        asm volatile("setmaxnreg.dec.sync.aligned.u32 72;");
        Cursor c = c0;
        auto wait = [&](uint32_t bar, uint32_t par) {
            if (!failed && !wait_here(bar, par)) failed = true;
        };
        if (warp == 8) {
            // ---- producer: lane i looks up the page of the run's piece `base + i`; lanes issue the copies of a tile's pieces and halves
            const int page = 1 << p.page_log2, piece = min(page, PF_TILE), piece_log2 = min(p.page_log2, 7), pieces = PF_TILE >> piece_log2, per_load = 32 / pieces;
            const int j = lane / (int)S::HALVES, half = lane % (int)S::HALVES;
            int s = 0, issued = 0;
            uint32_t parity = 1, qparity = 1;                                // a fresh barrier passes a wait on the previous phase
            for (int run; (run = c.run<PrefillRuns>()) > 0;) {
                auto lookup = [&](int i) {                                   // the pages of the pieces of tiles i, i + 1, ...
                    const int tl = i + lane / pieces, key = tl < c.s.n ? c.s.tile(tl) * PF_TILE + ((lane & (pieces - 1)) << piece_log2) : p.cap;
                    const bool seen = key < c.s.end && (key + piece > c.s.lo || key < p.sinks);
                    const int id = seen ? p.table[c.r * p.ld_table + (key >> p.page_log2)] : p.pages;      // a piece that no row sees is read as if it lay behind the cache: zeros
                    return (unsigned)id >= (unsigned)p.pages ? p.pages : id;
                };
                int base = c.at, ids = lookup(base), ids_next = lookup(base + per_load);
                for (int i = c.at; i < c.at + run; ++i) {
                    if (i - base == per_load) base = i, ids = ids_next, ids_next = lookup(base + per_load);
                    const int id = __shfl_sync(0xffffffffu, ids, (i - base) * pieces + (j & (pieces - 1)));
                    const int y = (c.s.tile(i) * PF_TILE + (j << piece_log2)) & (page - 1);
#pragma unroll
                    for (int kv = 0; kv < 2; ++kv) {
                        wait(empty0 + 8 * s, parity);
                        if (!failed) {
                            if (lane == 0) mbar_expect_tx_a(full0 + 8 * s, S::TILE);
                            __syncwarp();
                            if (j < pieces) tma_load_5d(kv0 + s * S::TILE + half * S::HALF + j * (piece * 128), kv ? &map_v : &map_k, 0, y, half, c.h, id, full0 + 8 * s);
                            ++issued;
                        }
                        if (++s == S::SLOTS) s = 0, parity ^= 1u;
                        if (kv == 0 && i == c.at) {                          // the queries, behind the first keys: their place is free only when the last scores are there
                            const int tiles_q = c.s.rows > qrows ? 2 : 1;
                            wait(qempty, qparity);
                            qparity ^= 1u;
                            if (!failed) {
                                if (lane == 0) mbar_expect_tx_a(qfull, (uint32_t)tiles_q * S::HALVES * (uint32_t)qrows * 128u);
                                __syncwarp();
                                if (j < tiles_q) tma_load_5d(smem0 + j * S::TILE + half * S::HALF, &map_q, 0, half, 0, c.h, c.row_base + c.rb * 2 * qtoks + j * qtoks, qfull);
                            }
                        }
                    }
                }
                c.advance<PrefillRuns>(p, block, PF_TILE, run);
            }
            if (failed)                                                      // copies in flight end before the block does
                for (int k = 0; k < min(issued, S::SLOTS); ++k) {
                    const int at = issued - 1 - k;
                    wait_here(full0 + 8 * (at % S::SLOTS), (uint32_t)(at / S::SLOTS) & 1u);
                }
        } else if (warp == 9) {
            // ---- issuer. The whole warp runs this, its conditions are votes and reductions and one elected lane issues, so that addresses and descriptors stay in uniform
            // registers: with operands in vector registers an MMA took 75 clocks to issue, more than it runs.
            constexpr uint32_t fmt = std::is_same<T, __nv_bfloat16>::value ? (1u << 7) | (1u << 10) : 0u;
            constexpr uint32_t idesc_s = umma_idesc_f16(128, 128) | fmt, idesc_o = umma_idesc_f16(128, D) | fmt | (1u << 16);      // V: MN-major
            const bool lead = elect_one();
            const uint32_t td = __reduce_max_sync(0xffffffffu, tmem);
            const uint64_t desc_q = umma_desc_sw128(smem0), desc_k = umma_desc_sw128(kv0), desc_v = umma_desc_mn128(kv0, S::HALF);
            uint32_t n = 0, items = 0, p0 = 0, p1 = 0;                       // slots, items and weights of either query tile so far
            bool ok = true;
            auto scores = [&](uint32_t w, uint32_t slot) {                   // S_w = Q_w K^T
#pragma unroll
                for (uint32_t h = 0; h < S::HALVES; ++h)
#pragma unroll
                    for (uint32_t k = 0; k < 4; ++k)
                        umma_f16(td + 128 * w, desc_q + (w * S::TILE + h * S::HALF) / 16 + 2 * k, desc_k + slot * (S::TILE / 16) + h * (S::HALF / 16) + 2 * k, idesc_s, (h | k) != 0);
            };
            auto values = [&](uint32_t w, uint32_t slot, uint32_t half, uint32_t acc) {       // O_w += P_w V for 64 keys
#pragma unroll
                for (uint32_t k = 0; k < 4; ++k)
                    umma_f16_ts(td + 256 + 128 * w, td + 128 * w + 32 * half + 8 * k, desc_v + slot * (S::TILE / 16) + 512 * half + 128 * k, idesc_o, half || k ? 1u : acc);
            };
            auto wait = [&](uint32_t bar, uint32_t par) {
                if (ok) ok = wait_here(bar, par);
            };
            for (int taken; (taken = c.run<PrefillRuns>()) > 0;) {
                const uint32_t run = __reduce_max_sync(0xffffffffu, (uint32_t)taken), two = __reduce_max_sync(0xffffffffu, c.s.rows > qrows ? 1u : 0u);
                wait(full0 + 8 * (n % S::SLOTS), (n / S::SLOTS) & 1u);
                wait(qfull, items & 1u);
                tc_fence_after();
                if (!ok) break;
                if (lead) {
                    scores(0, n % S::SLOTS);
                    umma_commit(sfull0);
                    if (two) scores(1, n % S::SLOTS), umma_commit(sfull0 + 8);
                    umma_commit(empty0 + 8 * (n % S::SLOTS));
                    if (run == 1) umma_commit(qempty);
                }
                __syncwarp();
                ++n, ++items;
                for (uint32_t i = 0; i < run && ok; ++i) {
                    const uint32_t sv = n % S::SLOTS, sk = (n + 1) % S::SLOTS, pv = (n / S::SLOTS) & 1u, pk = ((n + 1) / S::SLOTS) & 1u, more = i + 1 < run, acc = i != 0;
                    wait(full0 + 8 * sv, pv);
                    wait(clean0 + 8 * sv, pv);
                    wait(pfull0, p0);
                    tc_fence_after();
                    if (lead && ok) values(0, sv, 0, acc);
                    __syncwarp();
                    if (more) wait(full0 + 8 * sk, pk);
                    wait(phalf0, p0);
                    tc_fence_after();
                    p0 ^= 1u;
                    if (lead && ok) {
                        values(0, sv, 1, acc);
                        if (more) scores(0, sk);
                        umma_commit(more ? sfull0 : ofull0);                 // S0 of the next tile is there, O0 of this one too
                    }
                    __syncwarp();
                    if (two) {
                        wait(pfull0 + 8, p1);
                        tc_fence_after();
                        if (lead && ok) values(1, sv, 0, acc);
                        __syncwarp();
                        wait(phalf0 + 8, p1);
                        tc_fence_after();
                        p1 ^= 1u;
                    }
                    if (lead && ok) {
                        if (two) values(1, sv, 1, acc);
                        umma_commit(empty0 + 8 * sv);
                        if (two && more) scores(1, sk);
                        if (two) umma_commit((more ? sfull0 : ofull0) + 8);
                        if (more) umma_commit(empty0 + 8 * sk);
                        if (i + 2 == run) umma_commit(qempty);
                    }
                    __syncwarp();
                    n += 1 + more;
                }
                c.advance<PrefillRuns>(p, block, PF_TILE, taken);
            }
            failed = !ok;
        } else if (warp == 10) {
            // ---- between producer and issuer: values in places that no row sees become 0 (the first and last tiles of an item)
            int s = 1;
            uint32_t parity = 0;
            for (int run; (run = c.run<PrefillRuns>()) > 0;) {
                for (int i = 0; i < run; ++i) {
                    wait(full0 + 8 * s, parity);
                    const int key0 = c.s.tile(c.at + i) * PF_TILE;
                    // dead keys of the tile: [a0, a1) between the sinks and the window, [a2, 128) behind the last
                    const int a1 = min(max(c.s.lo - key0, 0), PF_TILE), a0 = min(max(p.sinks - key0, 0), a1), a2 = max(min(c.s.end - key0, PF_TILE), 0);
                    if ((a0 < a1 || a2 < PF_TILE) && !failed) {
                        const uint32_t v = kv0 + s * S::TILE + (lane >> 3 & (S::HALVES - 1)) * S::HALF + (lane & 7) * 16;
                        for (int k = a0 + lane / (8 * (int)S::HALVES); k < PF_TILE; k += 32 / (8 * (int)S::HALVES)) {
                            if (k >= a1 && k < a2) continue;
                            asm volatile("st.shared.v4.b32 [%0], {%1, %1, %1, %1};" ::"r"(v + k * 128), "r"(0) : "memory");
                        }
                        asm volatile("fence.proxy.async.shared::cta;" ::: "memory");
                        __syncwarp();
                    }
                    if (lane == 0) mbar_arrive_a(clean0 + 8 * s);
                    s += 2;
                    if (s > S::SLOTS) s = 1, parity ^= 1u;
                }
                c.advance<PrefillRuns>(p, block, PF_TILE, run);
            }
        }
    } else {
        asm volatile("setmaxnreg.inc.sync.aligned.u32 216;");
        // ---- softmax: one row a thread
        const int w = warp >> 2, rl = (warp & 3) * 32 + lane;
        const uint32_t lane_base = (uint32_t)((warp & 3) * 32) << 16, ts = tmem + lane_base + 128u * w, to = ts + 256u, sfull = sfull0 + 8 * w, ofull = ofull0 + 8 * w, pfull = pfull0 + 8 * w, phalf = phalf0 + 8 * w;
        const uint32_t stage = smem0 + S::OFF_OUT + warp * 4096;             // 32 rows x 128 bytes on their way to memory
        const float scale2 = fabsf(p.scale2);
        const uint64_t scale_pair = pair_of(scale2, scale2);
        const bool flip = p.scale2 < 0.f;
        uint32_t sparity = 0, oparity = 0;
        int flags = 0;
        // the warp's place in its run lies in shared memory: a row's 128 scores take the registers
        Cursor& c = *reinterpret_cast<Cursor*>(smem_raw + (smem0 - smem_u32(smem_raw)) + S::OFF_CUR + warp * sizeof(Cursor));
        if (lane == 0) c = c0;
        if (threadIdx.x == 0) p.notes[blockIdx.x] = make_int4(0, 0, 0, 0);
        __syncwarp();
        for (int run; (run = c.run<PrefillRuns>()) > 0;) {
            const int from = c.at;
            const int row = w * qrows + rl;                                  // row of the block
            const bool on = rl < qrows && row < c.s.rows;
            float m = -INFINITY, l = 0.f;
            if (w == 0 || c.s.rows > qrows) {                                // the second tile may be empty: then nothing of it is issued
                const int pos = on ? c.kv - c.tokens + (c.s.row0 + row) / p.group : -1, sink_tiles = c.s.sink_tiles, main_tile = c.s.main_tile - sink_tiles;
                // tiles from key plain_lo to plain_hi need no masks for any row of the query tile
                const int plain_hi = min(c.s.first + w * qtoks + 1, p.cap) - PF_TILE, plain_lo = p.window ? min(c.s.last, c.s.first + (w + 1) * qtoks - 1) - p.window + 1 : 0;
                for (int i = 0; i < run; ++i) {
                    if (!failed && !wait_here(sfull, sparity)) failed = true;
                    sparity ^= 1u;
                    tc_fence_after();
                    uint32_t v[4][32];
                    tmem_ld_32x32(ts, v[0]);
                    tmem_ld_32x32(ts + 32, v[1]);
                    tmem_ld_32x32(ts + 64, v[2]);
                    tmem_ld_32x32(ts + 96, v[3]);
                    tmem_ld_wait();
                    const int key0 = (from + i + (from + i < sink_tiles ? 0 : main_tile)) * PF_TILE;
                    if (flip)
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int e = 0; e < 32; ++e) v[q][e] ^= 0x80000000u;
                    if (key0 > plain_hi || key0 < plain_lo) {
                        // keys up to hi, from lo on or below sk are seen: 32 of them a mask word
                        const int hi = min(pos, p.cap - 1) - key0, lo = p.window ? pos - p.window + 1 - key0 : 0, sk = p.sinks - key0;
                        auto below = [](int n) { return n <= 0 ? 0u : n >= 32 ? 0xffffffffu : (1u << n) - 1u; };
#pragma unroll
                        for (int q = 0; q < 4; ++q) {
                            const uint32_t see = below(hi + 1 - 32 * q) & (~below(lo - 32 * q) | below(sk - 32 * q));
#pragma unroll
                            for (int e = 0; e < 32; ++e)
                                if (!(see >> e & 1u)) v[q][e] = 0xff800000u;
                        }
                    }
                    // weights of 32 keys to tensor memory, their sum added to `sum`
                    uint64_t m_pair, sum[2];
                    auto reference = [&]() {
                        const float m0 = m == -INFINITY ? 0.f : Weights<T>::below - m;
                        m_pair = pair_of(m0, m0), sum[0] = sum[1] = 0;
                    };
                    float t[4];
#pragma unroll
                    for (int q = 0; q < 4; ++q) t[q] = fmaxf(__uint_as_float(v[q][0]), __uint_as_float(v[q][1]));
                    auto weights = [&](int q, bool find_top) {
                        uint32_t pk[16];
#pragma unroll
                        for (int e = 0; e < 32; e += 2) {
                            float a, b;
                            split_pair(fma_pair(pair_of(__uint_as_float(v[q][e]), __uint_as_float(v[q][e + 1])), scale_pair, m_pair), a, b);
                            a = exp2_fast(a), b = exp2_fast(b);
                            sum[(e >> 1) & 1] = add_pair(sum[(e >> 1) & 1], pair_of(a, b));
                            pk[e / 2] = pack2<T>(a, b);
                            if (find_top && e) {
                                t[q] = max3(t[q], __uint_as_float(v[q][e]), __uint_as_float(v[q][e + 1]));
                                t[q + 2 & 3] = max3(t[q + 2 & 3], __uint_as_float(v[q + 2 & 3][e]), __uint_as_float(v[q + 2 & 3][e + 1]));
                            }
                        }
                        tmem_st_16(ts + 16 * q, pk);
                    };
                    // With heads of 64 the first half's weights are made with the reference as it is while the maximum is found, and again in the rare tile where a score
                    // passes the reference too far: 219 -> 208 us for 1024 tokens on 8192. With heads of 128, where the wait for the
                    // products is the longer part, it gained nothing (252 -> 255 us): there, as in the first tile of an item, the maximum comes first.
                    if (D == 64 && i) {
                        reference();
                        weights(0, true), weights(1, true);
                    } else {
#pragma unroll
                        for (int q = 0; q < 4; ++q)
#pragma unroll
                            for (int e = 2; e < 32; e += 2) t[q] = max3(t[q], __uint_as_float(v[q][e]), __uint_as_float(v[q][e + 1]));
                    }
                    const float top = fmaxf(max3(t[0], t[1], t[2]), t[3]) * scale2;
                    const bool over = top > m + Weights<T>::move;            // false where nothing is seen yet (-inf on both sides)
                    const bool move = __any_sync(0xffffffffu, over);
                    if (move || D != 64 || i == 0) {
                        const float f = !over ? 1.f : m == -INFINITY ? 0.f : exp2_fast(m - top);
                        if (over) m = top;
                        l *= f;
                        if (i && (D == 64 || move)) {
#pragma unroll 1
                            for (int q = 0; q < D; q += 16) {
                                uint32_t x[16];
                                tmem_ld_16(to + q, x);
                                tmem_ld_wait();
#pragma unroll
                                for (int e = 0; e < 16; ++e) x[e] = __float_as_uint(__uint_as_float(x[e]) * f);
                                tmem_st_16(to + q, x);
                            }
                        }
                        reference();
                        weights(0, false), weights(1, false);
                    }
                    auto hand_over = [&](uint32_t bar) {
                        tmem_st_wait_all();
                        tc_fence_before();
                        __syncwarp();
                        if (lane == 0) mbar_arrive_a(bar);
                    };
                    hand_over(pfull);
                    weights(2, false), weights(3, false);
                    hand_over(phalf);
                    float a, b;
                    split_pair(add_pair(sum[0], sum[1]), a, b);
                    l += a + b;
                }
                if (!failed && !wait_here(ofull, oparity)) failed = true;    // the last O
                oparity ^= 1u;
                tc_fence_after();
                // ---- output: 128 bytes of each of the warp's rows at a time through shared memory (16-byte pieces, swizzled), so that eight lanes store one row's
                const bool whole = from == 0 && run == c.s.n;
                const float inv = !whole ? 1.f : l > 0.f ? 1.f / l : 0.f;
                const int tok = (c.s.row0 + row) / p.group;
                const uint32_t row_bytes = whole ? D * 2 : D * 4;
                uint8_t* mine = whole ? p.o + 2 * ((int64_t)(c.row_base + tok) * p.o_t + (int64_t)(c.h * p.group + c.s.row0 + row - tok * p.group) * p.o_h)
                                      : reinterpret_cast<uint8_t*>(p.parts + ((size_t)blockIdx.x * 2 + (from == 0)) * ((size_t)block * (D + 2)) + (size_t)row * D);
                if (on && !whole && !failed) {
                    float* const ml = p.parts + ((size_t)blockIdx.x * 2 + (from == 0)) * ((size_t)block * (D + 2)) + (size_t)block * D + row;
                    ml[0] = m, ml[block] = l;
                }
                if (!on || failed) mine = nullptr;
#pragma unroll 1
                for (uint32_t off = 0; off < row_bytes; off += 128) {
                    __syncwarp();
                    if (whole) {
#pragma unroll
                        for (int h = 0; h < 2; ++h) {
                            uint32_t x[32];
                            tmem_ld_32x32(to + off / 2 + 32 * h, x);
                            tmem_ld_wait();
#pragma unroll
                            for (int e = 0; e < 4; ++e) {
                                uint32_t y[4];
#pragma unroll
                                for (int u = 0; u < 4; ++u) y[u] = pack2<T>(__uint_as_float(x[8 * e + 2 * u]) * inv, __uint_as_float(x[8 * e + 2 * u + 1]) * inv);
                                asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + (((4 * h + e) ^ (lane & 7)) << 4)), "r"(y[0]), "r"(y[1]), "r"(y[2]), "r"(y[3]) : "memory");
                            }
                        }
                    } else {
                        uint32_t x[32];
                        tmem_ld_32x32(to + off / 4, x);
                        tmem_ld_wait();
#pragma unroll
                        for (int e = 0; e < 8; ++e)
                            asm volatile("st.shared.v4.b32 [%0], {%1, %2, %3, %4};" ::"r"(stage + lane * 128 + ((e ^ (lane & 7)) << 4)), "r"(x[4 * e]), "r"(x[4 * e + 1]), "r"(x[4 * e + 2]), "r"(x[4 * e + 3])
                                         : "memory");
                    }
                    __syncwarp();
                    uint4 y[8];
#pragma unroll
                    for (int k = 0; k < 8; ++k) y[k] = lds128(stage + (4 * k + (lane >> 3)) * 128 + (((lane & 7) ^ ((4 * k + (lane >> 3)) & 7)) << 4));
#pragma unroll
                    for (int k = 0; k < 8; ++k) {
                        uint8_t* const to_row = reinterpret_cast<uint8_t*>(__shfl_sync(0xffffffffu, reinterpret_cast<unsigned long long>(mine), 4 * k + (lane >> 3)));
                        if (to_row) *reinterpret_cast<uint4*>(to_row + off + (lane & 7) * 16) = y[k];
                    }
                }
                tc_fence_before();
            }
            __syncwarp();
            if (lane == 0) {
                if (from != 0 || run != c.s.n) {
                    flags |= from == 0 ? NOTE_BEGINS : NOTE_CONTINUES | (from + run == c.s.n ? NOTE_ENDS : 0);
                    if (warp == 0) p.notes[blockIdx.x] = make_int4(c.r, c.rb, c.h, flags);
                }
                c.advance<PrefillRuns>(p, block, PF_TILE, run);
            }
            __syncwarp();
        }
    }
    if (failed) atomicExch(p.status, KYB_DEV_TIMEOUT_ATTN);
    tc_fence_before();
    __syncthreads();
    if (warp == 9) {
        tc_fence_after();
        tmem_dealloc(tmem, 512);
    }
}

}  // namespace kyb

namespace {

// queries [tokens][kv heads][group][d]: {64 values, half, head of the group, kv head, token}, boxes of all heads of a group and `qtoks` tokens
int make_query_map(CUtensorMap* tm, const KybAttnCall& c, int qtoks) {
    const kyb::AttnParams& p = c.p;
    const int64_t head = p.hq == 1 ? c.d : p.q_h, token = c.tokens == 1 ? (int64_t)c.d * p.hq : p.q_t;       // the stride of a dimension of one is never used: any valid one
    const cuuint64_t dims[5] = {64, (cuuint64_t)(c.d / 64), (cuuint64_t)p.group, (cuuint64_t)p.hkv, (cuuint64_t)c.tokens};
    const cuuint64_t strides[4] = {128, (cuuint64_t)head * 2, (cuuint64_t)head * 2 * (cuuint64_t)p.group, (cuuint64_t)token * 2};
    const cuuint32_t box[5] = {64, 1, (cuuint32_t)p.group, 1, (cuuint32_t)qtoks};
    const CUresult r = kyb_encode_map(tm, c.dtype == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, p.q, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != CUDA_SUCCESS) {
        kyb_set_error("%s CUresult %d (queries %p: %lld tokens, %d x %d heads of %d, strides %lld, %lld)", kyb_encode_problem(r), (int)r, (const void*)p.q, (long long)c.tokens, p.hkv,
                      p.group, c.d, (long long)token, (long long)head);
        return KYB_ECUDA;
    }
    return KYB_OK;
}

template <typename T, int D>
int launch_prefill(KybAttnCall& c, void* ws) {
    using S = kyb::PrefillShape<D>;
    auto kern = kyb::paged_attn_prefill_kernel<T, D>;
    if (int rc = kyb_allow_smem((const void*)kern)) return rc;
    const int piece = std::min(c.page, kyb::PF_TILE), qtoks = 128 / c.p.group;
    const int64_t units = kyb_attn_units(c, 2 * qtoks * c.p.group, kyb::PF_TILE);
    KYB_REQUIRE(units, "more than 2^31 key tiles in one call: split it");
    const int ctas = (int)std::min<int64_t>(c.sms, units);
    CUtensorMap mq, mk, mv;
    if (int rc = make_query_map(&mq, c, qtoks)) return rc;
    if (int rc = kyb_make_cache_map(&mk, c.k, c.dtype, c.p.pages, c.p.hkv, c.page, D, c.k_p, c.k_h, piece, 1)) return rc;
    if (int rc = kyb_make_cache_map(&mv, c.v, c.dtype, c.p.pages, c.p.hkv, c.page, D, c.v_p, c.v_h, piece, 1)) return rc;
    c.p.block_tokens = 2 * qtoks;
    c.p.notes = (int4*)ws, c.p.parts = (float*)((char*)ws + (size_t)ctas * sizeof(int4));
    kern<<<(unsigned)ctas, kyb::PF_THREADS, S::SMEM + 1024, c.st>>>(mq, mk, mv, c.p, qtoks);
    if (int rc = kyb_launch_check("paged_attn_prefill")) return rc;
    return kyb_attn_join(c, ctas, 2 * qtoks * c.p.group);
}

}  // namespace

size_t kyb_attn_prefill_scratch(int d, int group, int sms) {
    const size_t block = 2 * (size_t)(128 / group) * (size_t)group;
    return (size_t)sms * (sizeof(int4) + 2 * block * (d + 2) * sizeof(float));
}

int kyb_attn_prefill(KybAttnCall& c, void* ws) {
    if (c.dtype == 1) return c.d == 64 ? launch_prefill<__half, 64>(c, ws) : launch_prefill<__half, 128>(c, ws);
    return c.d == 64 ? launch_prefill<__nv_bfloat16, 64>(c, ws) : launch_prefill<__nv_bfloat16, 128>(c, ws);
}
