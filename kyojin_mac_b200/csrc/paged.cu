// A paged key/value cache in device memory: the step's slots from request lengths (paged_step, paged_release) and rotary positions with the cache append
// (rope_append). Cache layout: [page][kv head][token of the page][value], so the tokens of one (page, head) are one contiguous block that attention loads with a
// tiled copy.
#include <algorithm>

#include <cuda_bf16.h>

#include "kyb_common.cuh"

namespace kyb {

// ------------------------------------------------------------------------------------------------ slots of a step
// Requests r = 0 .. batch - 1 hold len_r cached tokens and bring new_r: with P tokens a page, need_r = ceil((len_r + new_r) / P) - ceil(len_r / P) pages come from
// the top of the free list, in request order (the k-th page of r is free[count - 1 - (sum of the needs before r) - k]). A request is served when its pages fit the
// table's columns, its tokens fit the step's rows and the needs up to and including its own fit the free list; a request that needs no page is not held up by
// others. Everything is whole numbers, so the result does not depend on the launch.
//
// Every CTA makes the prefix sums of all requests for itself (chunks of one request per thread, two scans), then the CTAs share the tokens and the table entries among
// their threads, each found by a binary search in the chunk's sums in shared memory. The state (lengths, free count) is written by one CTA behind a cluster barrier, when
// every CTA has read it, where it is updated in place (one cluster of up to 8 CTAs then, else up to 64 without one). Bound by latency: loads, scans, search, stores;
// 64 requests of one token 5.0 us, 1000 requests with 60 000 rows 7.2 us (in place, by eight CTAs,
// 12.6).
constexpr int PS_THREADS = 1024;

struct StepParams {
    const int* lens;
    const int* news;
    const int* free_pages;
    const int* free_count;
    int* table;
    int64_t ld_table;
    int64_t batch, cols, rows, free_cap;
    int page_log2;
    int* cu_q;
    int* kv_lens;
    int* positions;
    int* slots;
    int* lens_out;
    int* count_out;
    int* refused;
};

struct StepShared {
    int cu[PS_THREADS + 1];          // first row of each request of the chunk (clipped to the rows)
    int len[PS_THREADS];
    int first[PS_THREADS];           // pages taken before this request
    int need_end[PS_THREADS];        // pages taken by the served requests of the chunk up to and including this one (counted from the chunk's start)
    uint8_t served[PS_THREADS];
    long long warp_sum[2][32];
};

// inclusive sum over the CTA; two calls in a row use two places for the warps' sums, so that two barriers a call are enough
__device__ __forceinline__ long long block_scan(long long a, long long* sums) {
    const int lane = threadIdx.x & 31, warp = threadIdx.x >> 5;
#pragma unroll
    for (int d = 1; d < 32; d <<= 1) {
        const long long x = __shfl_up_sync(0xffffffffu, a, d);
        if (lane >= d) a += x;
    }
    if (lane == 31) sums[warp] = a;
    __syncthreads();
    if (warp == 0) {
        long long x = sums[lane];
#pragma unroll
        for (int d = 1; d < 32; d <<= 1) {
            const long long u = __shfl_up_sync(0xffffffffu, x, d);
            if (lane >= d) x += u;
        }
        sums[lane] = x;
    }
    __syncthreads();
    return warp ? a + sums[warp - 1] : a;
}

__global__ void __launch_bounds__(PS_THREADS, 1) paged_step_kernel(const StepParams p, const int ctas) {
    __shared__ StepShared s;
    __shared__ long long total[2];                                      // sums up to the end of the chunk
    __shared__ int taken_s;
    const int tid = threadIdx.x, cta = blockIdx.x, log2 = p.page_log2, low = (1 << log2) - 1;
    const long long count = max(0ll, min((long long)*p.free_count, (long long)p.free_cap));
    long long rows0 = 0, need0 = 0, taken = 0, refused = 0;             // sums over the chunks before this one
    for (int64_t c0 = 0; c0 < p.batch; c0 += PS_THREADS) {
        const int n = (int)min((int64_t)PS_THREADS, p.batch - c0);
        const bool on = tid < n;
        const unsigned len = on ? (unsigned)max(0, p.lens[c0 + tid]) : 0u, add = on ? (unsigned)max(0, p.news[c0 + tid]) : 0u;
        const long long have = ((long long)len + low) >> log2, want = ((long long)len + add + low) >> log2;
        const long long row_end = rows0 + block_scan(add, s.warp_sum[0]);
        const bool fits = want <= p.cols && row_end <= p.rows && (long long)len + add <= 0x7fffffffll;
        const long long need = on && fits ? want - have : 0;
        if (tid == 0) taken_s = 0;
        const long long need_end = need0 + block_scan(need, s.warp_sum[1]);
        const bool served = on && fits && (need == 0 || need_end <= count);
        // the sums of the needs grow, so those within the free list are a first part of them: what is taken up to here is that part's sum
        if (served && need) atomicMax(&taken_s, (int)(need_end - taken));
        const int missed = __syncthreads_count(on && !served);
        if (on) {
            s.cu[tid + 1] = (int)min(row_end, (long long)p.rows);
            s.len[tid] = (int)len, s.first[tid] = (int)(need_end - need), s.need_end[tid] = (int)min(max(need_end - taken, 0ll), (long long)taken_s), s.served[tid] = served;
        }
        if (tid == 0) s.cu[0] = (int)min(rows0, (long long)p.rows);
        if (tid == PS_THREADS - 1) total[0] = row_end, total[1] = need_end;
        __syncthreads();
        if (cta == 0 && on) {
            if (c0 == 0 && tid == 0) p.cu_q[0] = 0;
            p.cu_q[c0 + tid + 1] = s.cu[tid + 1];
            p.kv_lens[c0 + tid] = served ? (int)(len + add) : 0;
        }
        // table entries of the chunk's served requests
        const int pages = taken_s;
        for (int j = cta * PS_THREADS + tid; j < pages; j += ctas * PS_THREADS) {
            const int r = first_above(s.need_end, n, j), k = j - (r ? s.need_end[r - 1] : 0);
            const int col = (int)(((unsigned)s.len[r] + low) >> log2) + k;
            p.table[(c0 + r) * p.ld_table + col] = p.free_pages[count - 1 - (s.first[r] + k)];
        }
        // tokens of the chunk
        for (int64_t t = s.cu[0] + (int64_t)cta * PS_THREADS + tid; t < s.cu[n]; t += (int64_t)ctas * PS_THREADS) {
            const int r = first_above(s.cu + 1, n, (int)t);
            int pos = -1, slot = -1;
            if (s.served[r]) {
                pos = s.len[r] + (int)(t - s.cu[r]);
                const int held = (int)(((unsigned)s.len[r] + low) >> log2), col = pos >> log2;
                const int id = col < held ? p.table[(c0 + r) * p.ld_table + col] : p.free_pages[count - 1 - (s.first[r] + (col - held))];
                slot = (int)(((unsigned)id << log2) + (unsigned)(pos & low));
            }
            p.positions[t] = pos, p.slots[t] = slot;
        }
        taken += pages, rows0 = total[0], need0 = total[1], refused += missed;
        __syncthreads();                                                // the chunk's arrays are read
    }
    // rows behind the last request
    for (int64_t t = min(rows0, (long long)p.rows) + (int64_t)cta * PS_THREADS + tid; t < p.rows; t += (int64_t)ctas * PS_THREADS) p.positions[t] = -1, p.slots[t] = -1;
    // every CTA has read the state (not the .aligned form: the threads of a warp come out of the loop above at their own times)
    asm volatile("barrier.cluster.arrive.release;\n\tbarrier.cluster.wait.acquire;" ::: "memory");
    if (cta) return;
    if (tid == 0) *p.count_out = (int)(count - taken), *p.refused = (int)refused;
    // a request that was not served keeps its length; one that was has it in kv_lens (0 there: it holds and brings nothing)
    for (int64_t r = tid; r < p.batch; r += PS_THREADS) {
        const int kv = p.kv_lens[r];
        p.lens_out[r] = kv ? kv : max(0, p.lens[r]);
    }
}

// Pages of the requests with which[r] != 0 go back to the free list, in request order; their table entries read -1 and their lengths 0 afterwards. A request whose pages, behind
// those of all of them before it, would overflow the list (a page freed twice) keeps them and is counted in *refused; one that holds no page is not held up. One CTA, bound by
// dependent loads: 64 requests of 250 pages 13 us, one request's pages 3 us.
__global__ void __launch_bounds__(PS_THREADS, 1) paged_release_kernel(int* lens, const uint8_t* which, int* table, int64_t ld_table, int64_t batch, int64_t cols, int page,
                                                                      int* free_pages, int* free_count, int64_t free_cap, int* refused) {
    __shared__ StepShared s;
    __shared__ long long total, asked;                                  // pages that go back, and that would, of the chunk
    const int tid = threadIdx.x;
    long long count = max(0ll, min((long long)*free_count, (long long)free_cap)), room = free_cap - count, missed = 0;
    for (int64_t c0 = 0; c0 < batch; c0 += PS_THREADS) {
        const int n = (int)min((int64_t)PS_THREADS, batch - c0);
        const bool on = tid < n && which[c0 + tid];
        const long long len = on ? max(0, lens[c0 + tid]) : 0, pages = min((len + page - 1) / page, (long long)cols);
        const long long end = block_scan(on ? pages : 0, s.warp_sum[0]);
        const bool fits = on && (pages == 0 || end <= room);            // sums grow, so the requests that fit are the first ones, over all chunks
        const long long kept = block_scan(fits ? pages : 0, s.warp_sum[1]);
        const int miss = __syncthreads_count(on && !fits);
        if (tid < n) s.need_end[tid] = (int)kept;
        if (tid == PS_THREADS - 1) total = kept, asked = end;
        __syncthreads();
        for (int j = tid; j < (int)total; j += PS_THREADS) {
            const int r = first_above(s.need_end, n, j), k = j - (r ? s.need_end[r - 1] : 0);
            int* e = table + (c0 + r) * ld_table + k;
            free_pages[count + j] = *e;
            *e = -1;
        }
        if (fits) lens[c0 + tid] = 0;
        count += total, room -= asked, missed += miss;
        __syncthreads();
    }
    if (tid == 0) *free_count = (int)count, *refused = (int)missed;
}

// ------------------------------------------------------------------------------------------------ rotary positions and cache append
// Token t at position m: each pair (a, b) of a query or key head's first `rot` values becomes s (a cos f - b sin f, b cos f + a sin f) with f = m inv_freq[i]; pairs
// are (2 i, 2 i + 1) or (i, i + rot / 2). Keys (turned) and values go to the cache at the token's slot; queries to q_out. Far positions: f reaches 10^6 and more,
// where 32 bits hold it to 0.06 only, so the product and its reduction to [-pi, pi] are made in 64 bits, sine and cosine of the rest in 32.
// Bound by HBM: every element is read and written once, 16 bytes at a time (8191 tokens of 64 / 8 heads of 128: 57 us = 5.9 TB/s, 55 with neighbours paired; 64 tokens 2.8 us).
// A CTA makes the rot / 2 pairs of sine and cosine of its token once in shared memory and serves all of the token's heads with them; few tokens are cut into parts of the
// heads so that every SM has a CTA. Loads made before the angles (57 -> 66 us) and angles laid out without bank conflicts (57 -> 64) were slower.
constexpr int RP_THREADS = 256;                                          // at most

struct RopeParams {
    const uint8_t *q, *k, *v;                // 16-bit elements
    uint8_t *qo, *kc, *vc;
    int64_t q_t, q_h, k_t, k_h, v_t, v_h, qo_t, qo_h;     // strides in bytes (token, head)
    int64_t kc_p, kc_h, vc_p, vc_h;                       // strides in bytes (page, head); tokens of a page are dense
    const int* positions;
    const int* slots;
    const float* inv;
    int64_t pages;
    int page_log2, hq, hkv, d, rot, parts;
    float mscale;
};

template <typename T> struct Pair;
template <> struct Pair<__half> {
    static __device__ __forceinline__ float2 get(uint32_t w) { return __half22float2(*reinterpret_cast<__half2*>(&w)); }
    static __device__ __forceinline__ uint32_t put(float a, float b) { __half2 h = __floats2half2_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};
template <> struct Pair<__nv_bfloat16> {
    static __device__ __forceinline__ float2 get(uint32_t w) { return __bfloat1622float2(*reinterpret_cast<__nv_bfloat162*>(&w)); }
    static __device__ __forceinline__ uint32_t put(float a, float b) { __nv_bfloat162 h = __floats2bfloat162_rn(a, b); return *reinterpret_cast<uint32_t*>(&h); }
};

__device__ __forceinline__ void turn(float& a, float& b, float c, float s) {
    const float u = a * c - b * s, w = b * c + a * s;
    a = u, b = w;
}

template <typename T, bool INTER>
__global__ void __launch_bounds__(RP_THREADS) rope_append_kernel(const RopeParams p) {
    __shared__ float2 cs[128];
    const int64_t t = blockIdx.x;
    const int pos = p.positions[t], slot = p.hkv ? p.slots[t] : -1;
    if (pos < 0) return;                                                  // a row behind the last request: nothing of it is read or written
    for (int i = threadIdx.x; i < p.rot / 2; i += blockDim.x) {
        const double f = (double)pos * (double)p.inv[i], turns = rint(f * 0.15915494309189533577);
        const double r = fma(-turns, 2.4492935982947064e-16, fma(-turns, 6.283185307179586477, f));
        float s, c;
        sincosf((float)r, &s, &c);
        cs[i] = make_float2(c * p.mscale, s * p.mscale);
    }
    __syncthreads();
    const int half = p.rot / 2;
    const bool stored = slot >= 0 && (slot >> p.page_log2) < p.pages;
    const int64_t at = stored ? slot >> p.page_log2 : 0, off = stored ? (int64_t)(slot & ((1 << p.page_log2) - 1)) * p.d * 2 : 0;
    // a unit is two 16-byte pieces, half of the turned part, of the plain part or of the values apart (the last one of an odd number is alone)
    const int turned = p.rot / 16, plain = (p.d - p.rot) / 8, per_head = turned + (plain + 1) / 2, all = p.d / 8, per_v = (all + 1) / 2;
    const int units_t = (p.hq + p.hkv) * per_head, units = units_t + p.hkv * per_v;
    for (int u = blockIdx.y * blockDim.x + threadIdx.x; u < units; u += p.parts * blockDim.x) {
        const bool value = u >= units_t;
        const int h = value ? (u - units_t) / per_v : u / per_head, e = value ? u - units_t - h * per_v : u - h * per_head;
        const bool query = !value && h < p.hq;
        if (!query && !stored) continue;
        const uint8_t* src = value ? p.v + t * p.v_t + h * p.v_h : query ? p.q + t * p.q_t + h * p.q_h : p.k + t * p.k_t + (h - p.hq) * p.k_h;
        uint8_t* dst = value ? p.vc + at * p.vc_p + h * p.vc_h + off : query ? p.qo + t * p.qo_t + h * p.qo_h : p.kc + at * p.kc_p + (h - p.hq) * p.kc_h + off;
        if (value || e >= turned) {
            const int n = value ? all : plain, far = (n + 1) / 2, i = value ? e : e - turned, x = (value ? 0 : p.rot * 2) + i * 16, y = x + far * 16;
            const bool two = i + far < n;
            const uint4 w = *reinterpret_cast<const uint4*>(src + x);
            uint4 z = w;
            if (two) z = *reinterpret_cast<const uint4*>(src + y);
            *reinterpret_cast<uint4*>(dst + x) = w;
            if (two) *reinterpret_cast<uint4*>(dst + y) = z;
            continue;
        }
        const int x = e * 16, y = half * 2 + x;
        uint4 w = *reinterpret_cast<const uint4*>(src + x), z = *reinterpret_cast<const uint4*>(src + y);
        uint32_t *q = reinterpret_cast<uint32_t*>(&w), *r = reinterpret_cast<uint32_t*>(&z);
#pragma unroll
        for (int j = 0; j < 4; ++j) {
            float2 a = Pair<T>::get(q[j]), b = Pair<T>::get(r[j]);
            const float2 c0 = cs[INTER ? e * 4 + j : e * 8 + 2 * j], c1 = cs[INTER ? half / 2 + e * 4 + j : e * 8 + 2 * j + 1];
            if (INTER) turn(a.x, a.y, c0.x, c0.y), turn(b.x, b.y, c1.x, c1.y);
            else turn(a.x, b.x, c0.x, c0.y), turn(a.y, b.y, c1.x, c1.y);
            q[j] = Pair<T>::put(a.x, a.y), r[j] = Pair<T>::put(b.x, b.y);
        }
        *reinterpret_cast<uint4*>(dst + x) = w;
        *reinterpret_cast<uint4*>(dst + y) = z;
    }
}

}  // namespace kyb

extern "C" int kyb_paged_step(const kyb_paged_step_args* a, void* stream) {
    KYB_REQUIRE(a, "null pointer");
    const void *lens = a->lens, *new_lens = a->new_lens, *free_pages = a->free_pages, *free_count = a->free_count;
    void *table = a->table, *cu_q = a->cu_q, *kv_lens = a->kv_lens, *positions = a->positions, *slots = a->slots, *lens_out = a->lens_out, *free_count_out = a->free_count_out,
         *refused = a->refused;
    const int64_t free_cap = a->free_cap, ld_table = a->ld_table, batch = a->batch, cols = a->cols, rows = a->rows;
    const int page = (int)std::min<int64_t>(std::max<int64_t>(a->page, 0), 1 << 20);
    KYB_REQUIRE(lens && new_lens && free_pages && free_count && table && cu_q && kv_lens && lens_out && free_count_out && refused && (rows == 0 || (positions && slots)), "null pointer");
    KYB_REQUIRE(batch > 0 && batch < (1ll << 24) && cols > 0 && ld_table >= cols && rows >= 0 && rows < (1ll << 31) && free_cap > 0 && free_cap < (1ll << 31),
                "batch=%lld cols=%lld (row stride %lld) rows=%lld free list of %lld: out of range", (long long)batch, (long long)cols, (long long)ld_table, (long long)rows,
                (long long)free_cap);
    KYB_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page=%d: a power of two from 16 to 256", page);
    kyb::StepParams p;
    p.lens = (const int*)lens, p.news = (const int*)new_lens, p.free_pages = (const int*)free_pages, p.free_count = (const int*)free_count, p.table = (int*)table;
    p.ld_table = ld_table, p.batch = batch, p.cols = cols, p.rows = rows, p.free_cap = free_cap, p.page_log2 = 0;
    while ((1 << p.page_log2) < page) ++p.page_log2;
    p.cu_q = (int*)cu_q, p.kv_lens = (int*)kv_lens, p.positions = (int*)positions, p.slots = (int*)slots;
    p.lens_out = (int*)lens_out, p.count_out = (int*)free_count_out, p.refused = (int*)refused;
    // one CTA for few rows; more share them, as one cluster where the state is updated in place, else as many as there are thousands of rows
    const bool in_place = lens_out == lens || free_count_out == free_count;
    const int ctas = rows <= 4 * kyb::PS_THREADS ? 1 : in_place ? 8 : (int)std::min<int64_t>(64, rows / kyb::PS_THREADS);
    cudaLaunchConfig_t cfg = {};
    cfg.gridDim = dim3((unsigned)ctas), cfg.blockDim = dim3(kyb::PS_THREADS), cfg.stream = (cudaStream_t)stream;
    cudaLaunchAttribute at[1];
    at[0].id = cudaLaunchAttributeClusterDimension;
    at[0].val.clusterDim.x = in_place ? (unsigned)ctas : 1, at[0].val.clusterDim.y = 1, at[0].val.clusterDim.z = 1;
    cfg.attrs = at, cfg.numAttrs = 1;
    KYB_CUDA(cudaLaunchKernelEx(&cfg, kyb::paged_step_kernel, p, ctas));
    return kyb_launch_check("paged_step");
}

extern "C" int kyb_paged_release(void* lens, const void* which, void* table, int64_t ld_table, int64_t batch, int64_t cols, int page, void* free_pages, int64_t free_cap,
                                 void* free_count, void* refused, void* stream) {
    KYB_REQUIRE(lens && which && table && free_pages && free_count && refused, "null pointer");
    KYB_REQUIRE(batch > 0 && batch < (1ll << 24) && cols > 0 && ld_table >= cols && free_cap > 0 && free_cap < (1ll << 31),
                "batch=%lld cols=%lld (row stride %lld) free list of %lld: out of range", (long long)batch, (long long)cols, (long long)ld_table, (long long)free_cap);
    KYB_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0, "page=%d: a power of two from 16 to 256", page);
    kyb::paged_release_kernel<<<1, kyb::PS_THREADS, 0, (cudaStream_t)stream>>>((int*)lens, (const uint8_t*)which, (int*)table, ld_table, batch, cols, page, (int*)free_pages,
                                                                               (int*)free_count, free_cap, (int*)refused);
    return kyb_launch_check("paged_release");
}

extern "C" int kyb_rope_append(const kyb_rope_append_args* a, void* stream) {
    KYB_REQUIRE(a, "null pointer");
    const void *q = a->q, *k = a->k, *v = a->v, *positions = a->positions, *slots = a->slots, *inv_freq = a->inv_freq;
    void *q_out = a->q_out, *k_cache = a->k_cache, *v_cache = a->v_cache;
    const int64_t tokens = a->tokens, pages = a->pages;
    for (int64_t n : {a->hq, a->hkv, a->d, a->rot, a->dtype, a->page}) KYB_REQUIRE(n >= 0 && n <= 65536, "a size of %lld: out of range", (long long)n);
    const int hq = (int)a->hq, hkv = (int)a->hkv, d = (int)a->d, rot = (int)a->rot, dtype = (int)a->dtype, page = (int)a->page;
    const bool interleaved = a->interleaved != 0;
    const float mscale = (float)a->mscale;
    KYB_REQUIRE(tokens >= 0 && tokens < (1ll << 31) && hq + hkv > 0, "tokens=%lld heads %d + %d: out of range", (long long)tokens,
                hq, hkv);
    KYB_REQUIRE(d >= 16 && d <= 256 && d % 8 == 0 && rot >= 16 && rot <= d && rot % 16 == 0, "d=%d rot=%d: d a multiple of 8 up to 256, rot a multiple of 16 from 16 to d", d, rot);
    KYB_REQUIRE(dtype == 1 || dtype == 2, "dtype=%d: 1 (fp16) or 2 (bf16)", dtype);
    if (tokens == 0) return KYB_OK;
    KYB_REQUIRE(positions && inv_freq && (hq == 0 || (q && q_out)) && (hkv == 0 || (k && v && slots && k_cache && v_cache)), "null pointer");
    for (int64_t s : {a->q_token, a->q_head, a->k_token, a->k_head, a->v_token, a->v_head, a->q_out_token, a->q_out_head, a->k_cache_page, a->k_cache_head, a->v_cache_page, a->v_cache_head})
        KYB_REQUIRE(s % 8 == 0, "a stride of %lld elements: strides are multiples of 8 elements (16 bytes)", (long long)s);
    KYB_REQUIRE((((uintptr_t)q | (uintptr_t)k | (uintptr_t)v | (uintptr_t)q_out | (uintptr_t)k_cache | (uintptr_t)v_cache) & 15) == 0, "pointers must be 16-byte aligned");
    KYB_REQUIRE(hkv == 0 || (page >= 16 && page <= 256 && (page & (page - 1)) == 0 && pages > 0 && pages < (1ll << 31)), "page=%d pages=%lld: a power of two from 16 to 256, at least one page",
                page, (long long)pages);
    kyb::RopeParams p;
    p.q = (const uint8_t*)q, p.k = (const uint8_t*)k, p.v = (const uint8_t*)v, p.qo = (uint8_t*)q_out, p.kc = (uint8_t*)k_cache, p.vc = (uint8_t*)v_cache;
    p.q_t = a->q_token * 2, p.q_h = a->q_head * 2, p.k_t = a->k_token * 2, p.k_h = a->k_head * 2, p.v_t = a->v_token * 2, p.v_h = a->v_head * 2;
    p.qo_t = a->q_out_token * 2, p.qo_h = a->q_out_head * 2;
    p.kc_p = a->k_cache_page * 2, p.kc_h = a->k_cache_head * 2, p.vc_p = a->v_cache_page * 2, p.vc_h = a->v_cache_head * 2;
    p.positions = (const int*)positions, p.slots = (const int*)slots, p.inv = (const float*)inv_freq, p.pages = pages;
    p.page_log2 = 0;
    while (hkv && (1 << p.page_log2) < page) ++p.page_log2;
    p.hq = hq, p.hkv = hkv, p.d = d, p.rot = rot, p.mscale = mscale;
    const int units = (hq + hkv) * (rot / 16 + ((d - rot) / 8 + 1) / 2) + hkv * ((d / 8 + 1) / 2);
    int parts = 1;                                                        // parts of a token's heads: until every SM has two CTAs or a thread has one unit
    while (tokens * parts < 2 * kyb_sm_count() && parts * kyb::RP_THREADS < units) parts *= 2;
    p.parts = parts;
    // as many threads as a CTA's units fill in equal turns (8191 tokens of 8 / 1 heads of 128, 80 units: 18 us by 256 threads, 12.3 by 96)
    const int share = (units + parts - 1) / parts, turns = (share + kyb::RP_THREADS - 1) / kyb::RP_THREADS;
    const int threads = std::max(64, ((share + turns - 1) / turns + 31) / 32 * 32);
    const dim3 grid((unsigned)tokens, (unsigned)parts);
    cudaStream_t st = (cudaStream_t)stream;
    if (dtype == 1) {
        if (interleaved) kyb::rope_append_kernel<__half, true><<<grid, threads, 0, st>>>(p);
        else kyb::rope_append_kernel<__half, false><<<grid, threads, 0, st>>>(p);
    } else {
        if (interleaved) kyb::rope_append_kernel<__nv_bfloat16, true><<<grid, threads, 0, st>>>(p);
        else kyb::rope_append_kernel<__nv_bfloat16, false><<<grid, threads, 0, st>>>(p);
    }
    return kyb_launch_check("rope_append");
}
