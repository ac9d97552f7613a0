// Attention over a paged cache: what the decode and the prefill kernel share (parameters, the keys that a block of rows sees, tensor maps of the cache, the split of the
// work over the CTAs and the sum of the parts).
//
// Rows: the (token, query head) pairs of one request and one key-value head, token by token, G = hq / hkv rows a token: all of them read the same keys. A row block
// is `block` consecutive ones. An item is (request, row block, key-value head); its work is cut along the keys into tiles of `tile` keys. The tiles of all items, in
// order (request, then row block, then head), are dealt to the CTAs in contiguous runs of equal cost, so ragged lengths and few long ones balance alike; an item that a run's
// border cuts leaves parts in the scratch, unnormalised and in 32 bits, which a second launch adds in their order. Nothing depends on timing.
#pragma once

#include <cuda_bf16.h>

#include "tc_common.cuh"

namespace kyb {

struct AttnParams {
    const uint8_t* q;                                         // 16-bit elements
    uint8_t* o;
    int64_t q_t, q_h, o_t, o_h;                               // strides in elements (token, head)
    const int* table;
    const int* kv_lens;
    const int* cu_q;
    int64_t ld_table;
    int batch, tokens, hq, hkv, group, page_log2, pages, cap; // tokens: rows of q; cap: tokens that a row of the table can hold
    int block_tokens;                                         // tokens of a row block, where it is made of whole ones (0: it is not)
    int window, sinks;                                        // window 0: none
    float scale2;                                             // scale log2(e)
    unsigned int* status;
    float* parts;                                             // scratch: parts[cta][2][block * (d + 2)]
    int4* notes;                                              // scratch: notes[cta] = {request, row block, head, flags}
};
// flags of a CTA's note: its first run continues an item (and ends it), its last run begins an item that the next CTA continues
constexpr int NOTE_CONTINUES = 1, NOTE_ENDS = 2, NOTE_BEGINS = 4;

// A row's weights are 2^(below + score - m), rounded to the inputs' type for the product with V; the reference m is the largest score when it is set and moves when a score
// passes it by `move`. The factor 2^below is in all parts of a row alike and leaves with the division by their sum. It is there for fp16, which has steps of 2^-24: under a
// largest weight of 1, those below 2^-25 would be gone, and where one key takes nearly all of the mass (a first token, say) the many small ones add up to something all the
// same. With the largest between 2^7 and 2^15 what is lost is 2^-32 of it. (2^15 keeps fp16 finite; the sums are in 32 bits. A smaller `move` would leave room for a larger
// factor, but scores pass the first tile's largest by 2^4 now and then, by 2^8 hardly ever.) bf16 has the exponents of 32 bits and needs no factor.
template <typename T> struct Weights { static constexpr float below = 7.f, move = 8.f; };
template <> struct Weights<__nv_bfloat16> { static constexpr float below = 0.f, move = 15.f; };

#ifdef __CUDACC__
// The keys that a block of rows sees: tiles of `tile` keys, first those of the sinks, then those of the window (or of the whole context).
struct KeySpan {
    int row0, rows;            // first row of the block in its request, rows of the block
    int first, last;           // positions of its first and last token
    int lo, end;               // keys [lo, end) and [0, min(sinks, lo)) are seen by some row
    int sink_tiles, main_tile, n;
    __device__ __forceinline__ int tile(int i) const { return i < sink_tiles ? i : main_tile + (i - sink_tiles); }
    __device__ __forceinline__ bool alive(int key, int sinks) const { return key < end && (key >= lo || key < sinks); }
};

// block: rows of a row block; p.block_tokens: its tokens when it is made of whole ones (no division by the group then), else 0
__device__ __forceinline__ KeySpan key_span(const AttnParams& p, int tokens, int kv, int block, int rb, int tile) {
    KeySpan s;
    s.row0 = rb * block, s.rows = min(block, tokens * p.group - s.row0);
    if (p.block_tokens) s.first = rb * p.block_tokens, s.last = min(s.first + p.block_tokens, tokens) - 1;
    else s.first = s.row0 / p.group, s.last = (s.row0 + s.rows - 1) / p.group;
    s.first += kv - tokens, s.last += kv - tokens;
    s.end = max(0, min(s.last + 1, p.cap));
    s.lo = p.window ? max(0, s.first - p.window + 1) : 0;
    s.main_tile = s.lo / tile;
    const int main_end = (s.end + tile - 1) / tile;
    s.sink_tiles = min((min(p.sinks, s.end) + tile - 1) / tile, min(s.main_tile, main_end));
    s.n = max(1, s.sink_tiles + max(0, main_end - s.main_tile));            // a block that sees nothing still has its zeros to write: one tile, masked throughout
    return s;
}
// a request's first row and its rows, whatever cu_q holds: inside [0, tokens)
__device__ __forceinline__ int request_rows(const AttnParams& p, int r, int& base) {
    base = min(max(p.cu_q[r], 0), p.tokens);
    return min(max(p.cu_q[r + 1], base), p.tokens) - base;
}
// Whether a request's offsets fall. Where none do, the requests own no more rows than there are, and the host's bound of the units (fewer than 2^31 in all) rests on that.
__device__ __forceinline__ bool offsets_fall(const AttnParams& p, int r) { return max(p.cu_q[r + 1], 0) < min(max(p.cu_q[r], 0), p.tokens); }
// Where some do (0, T, 0, T, ... would give every second request all rows): whether the requests together still own no more than there are. If not, the sums of units could pass
// 32 bits and the runs be anything, so nothing is done and the status word says why. All threads of the block call it; `sum` is a word of shared memory.
__device__ __forceinline__ bool rows_hold(const AttnParams& p, unsigned long long* sum) {
    __syncthreads();
    if (threadIdx.x == 0) {                                                  // one thread: a shared sum here cost the prefill kernel for heads of 64 1 % (206 -> 208 us) by its softmax loop's code
        int base;
        *sum = 0;
#pragma unroll 1
        for (int r = 0; r < p.batch; ++r) *sum += (unsigned)request_rows(p, r, base);
    }
    __syncthreads();
    if (*sum <= (unsigned long long)p.tokens) return true;
    if (blockIdx.x == 0 && threadIdx.x == 0) atomicExch(p.status, KYB_DEV_ROWS_ATTN);
    return false;
}
__device__ __forceinline__ int request_keys(const AttnParams& p, int r) { return min(max(p.kv_lens[r], 0), 1 << 30); }
__device__ __forceinline__ int row_blocks(const AttnParams& p, int tokens, int block) { return (tokens * p.group + block - 1) / block; }

// The work is dealt in units: an item counts its tiles and OVER more, what beginning and ending it costs (measured, in tiles), in front of them. A border between runs that
// falls into those, or so that SNAP tiles or fewer of the item would be left, moves to the item's begin or end: items are not cut for nothing.
template <int OVER, int SNAP>
struct Runs {
    static __device__ __forceinline__ int units(const KeySpan& s) { return s.n + OVER; }
    // a run that starts `x` units into an item: the tile it starts with (n: with the next item), and what changes in its number of units
    static __device__ __forceinline__ int enter(const KeySpan& s, int x, int& left) {
        if (x > OVER && s.n + OVER - x <= SNAP) {
            left -= s.n + OVER - x;
            return s.n;
        }
        if (x <= OVER) {
            left += x;
            return 0;
        }
        return x - OVER;
    }
    // tiles of the item that a run with `left` units takes from tile `at` on (0: the run ends in front of it)
    static __device__ __forceinline__ int take(const KeySpan& s, int at, int left) {
        const int n = left - (at ? 0 : OVER);
        return n <= 0 ? 0 : n + SNAP >= s.n - at ? s.n - at : n;
    }
    static __device__ __forceinline__ int cost(int at, int taken) { return taken + (at ? 0 : OVER); }
};

// border c of `runs` equal runs over `total` units (fewer than 2^31: the host sees to it for requests side by side, rows_hold to those)
__device__ __forceinline__ int run_border(int total, int runs, int c) {
    const int each = total / runs;
    return each * c + min(c, total - each * runs);
}

// Where a CTA's run is
struct Cursor {
    int r, rb, h, at;          // request, row block, head, next tile of the item
    int left;                  // units left in the run
    int tokens, kv, blocks, row_base;
    KeySpan s;
    __device__ __forceinline__ void load(const AttnParams& p, int block, int tile) {
        tokens = request_rows(p, r, row_base), kv = request_keys(p, r), blocks = row_blocks(p, tokens, block);
        if (rb < blocks) s = key_span(p, tokens, kv, block, rb, tile);
    }
    // to the next item
    __device__ __forceinline__ void next(const AttnParams& p, int block, int tile) {
        at = 0;
        if (++h < p.hkv) return;
        h = 0, ++rb;
        while (rb >= blocks) {
            rb = 0;
            if (++r >= p.batch) {
                r = p.batch - 1, left = 0;
                return;
            }
            load(p, block, tile);
        }
        s = key_span(p, tokens, kv, block, rb, tile);
    }
    // behind `taken` tiles
    template <typename RUNS> __device__ __forceinline__ void advance(const AttnParams& p, int block, int tile, int taken) {
        left -= RUNS::cost(at, taken), at += taken;
        if (at == s.n) next(p, block, tile);
    }
    template <typename RUNS> __device__ __forceinline__ int run() const { return left > 0 ? RUNS::take(s, at, left) : 0; }
};

// 5-D copy of a piece of one page and head into shared memory: [half of the values][token][128 bytes], 128-byte swizzle
__device__ __forceinline__ void tma_load_5d(uint32_t dst, const CUtensorMap* tm, int x, int y, int z, int h, int page, uint32_t bar) {
    asm volatile("cp.async.bulk.tensor.5d.shared::cluster.global.mbarrier::complete_tx::bytes [%0], [%1, {%2, %3, %4, %5, %6}], [%7];" ::"r"(dst), "l"(tm), "r"(x), "r"(y), "r"(z), "r"(h),
                 "r"(page), "r"(bar)
                 : "memory");
}
// a wait whose answer is the warp's: what follows stands warp-wide instructions that a part of the warp must not meet alone
__device__ __forceinline__ bool wait_warp(uint32_t bar, uint32_t parity) { return __all_sync(0xffffffffu, mbar_wait_fast(bar, parity)); }
__device__ __forceinline__ float exp2_fast(float x) {
    float y;
    asm("ex2.approx.ftz.f32 %0, %1;" : "=f"(y) : "f"(x));
    return y;
}
__device__ __forceinline__ void pdl_launch_dependents() { asm volatile("griddepcontrol.launch_dependents;" ::: "memory"); }
__device__ __forceinline__ void pdl_wait() { asm volatile("griddepcontrol.wait;" ::: "memory"); }

template <typename T> __device__ __forceinline__ uint32_t pack2(float a, float b);
template <> __device__ __forceinline__ uint32_t pack2<__half>(float a, float b) {
    uint32_t d;
    asm("cvt.rn.f16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}
template <> __device__ __forceinline__ uint32_t pack2<__nv_bfloat16>(float a, float b) {
    uint32_t d;
    asm("cvt.rn.bf16x2.f32 %0, %1, %2;" : "=r"(d) : "f"(b), "f"(a));
    return d;
}
#endif

}  // namespace kyb

// tensor map of a cache [pages][heads][page][d] of 16-bit values: {64 values, token, half, head, page}, boxes of `box_tokens` tokens and `box_halves` halves
static inline int kyb_make_cache_map(CUtensorMap* tm, const void* base, int dtype, int64_t pages, int heads, int page, int d, int64_t page_stride, int64_t head_stride, int box_tokens,
                                     int box_halves) {
    if (heads == 1) head_stride = (int64_t)page * d;                        // the stride of a dimension of one is never used: any valid one
    if (pages == 1) page_stride = head_stride * heads;
    const cuuint64_t dims[5] = {64, (cuuint64_t)page, (cuuint64_t)(d / 64), (cuuint64_t)heads, (cuuint64_t)pages};
    const cuuint64_t strides[4] = {(cuuint64_t)d * 2, 128, (cuuint64_t)head_stride * 2, (cuuint64_t)page_stride * 2};
    const cuuint32_t box[5] = {64, (cuuint32_t)box_tokens, (cuuint32_t)box_halves, 1, 1};
    const CUresult r = kyb_encode_map(tm, dtype == 2 ? CU_TENSOR_MAP_DATA_TYPE_BFLOAT16 : CU_TENSOR_MAP_DATA_TYPE_FLOAT16, 5, base, dims, strides, box, CU_TENSOR_MAP_SWIZZLE_128B);
    if (r != CUDA_SUCCESS) {
        kyb_set_error("%s CUresult %d (cache %p: %lld pages, %d heads, %d tokens of %d values, strides %lld, %lld)", kyb_encode_problem(r), (int)r, base, (long long)pages, heads, page,
                      d, (long long)page_stride, (long long)head_stride);
        return KYB_ECUDA;
    }
    return KYB_OK;
}

#ifdef __CUDACC__
// launch whose beginning may overlap the end of the kernel before it on the stream (the kernel waits for that one before it reads or writes memory)
template <typename K, typename... A>
static inline int kyb_launch_chained(K kern, int ctas, int threads, size_t smem, cudaStream_t st, const A&... args) {
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3((unsigned)threads), cfg.dynamicSmemBytes = smem, cfg.stream = st;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeProgrammaticStreamSerialization;
    at[0].val.programmaticStreamSerializationAllowed = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    KYB_CUDA(cudaLaunchKernelEx(&cfg, kern, args...));
    return KYB_OK;
}
#endif

// The call as the C entry hands it to a kernel's launcher
struct KybAttnCall {
    kyb::AttnParams p;
    const void *k, *v;
    int64_t k_p, k_h, v_p, v_h, tokens;
    int d, dtype, page, sms;
    cudaStream_t st;
};
// an upper bound of the units that the kernels deal out: row blocks (each request's last may be a part) x heads x tiles of a full table row and an item's extra; 0 from 2^31 on
static inline int64_t kyb_attn_units(const KybAttnCall& c, int block, int tile) {
    const int64_t blocks = c.tokens * c.p.group / block + c.p.batch, tiles = (int64_t)c.p.cap / tile + 8;
    return blocks * c.p.hkv < (1ll << 31) / tiles ? blocks * c.p.hkv * tiles : 0;
}
// rows a request may bring for the decode kernel; beyond, the prefill kernel
constexpr int KYB_DECODE_ROWS = 16;
size_t kyb_attn_decode_scratch(int d, int rows, int sms);
int kyb_attn_decode(KybAttnCall& c, int rows, void* ws);
size_t kyb_attn_prefill_scratch(int d, int group, int sms);
int kyb_attn_prefill(KybAttnCall& c, void* ws);
// second launch: adds the parts of the items that were cut (ctas runs, blocks of `block` rows)
int kyb_attn_join(const KybAttnCall& c, int ctas, int block);
