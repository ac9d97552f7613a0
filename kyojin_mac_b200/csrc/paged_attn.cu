// Attention of a step's new tokens over a paged cache: o = softmax(scale q K^T) V per query head, where the token at position p of its request sees key j when j <= p,
// and with a window W only when j > p - W or j < sinks. Tokens of all requests are packed (cu_q), a request's last token is its last cached one.
#include <float.h>

#include <algorithm>

#include "paged_attn.cuh"

extern "C" size_t kyb_paged_attention_workspace_bytes(int64_t batch, int64_t tokens, int64_t max_q, int64_t cols, int page, int hq, int hkv, int d) {
    (void)batch, (void)cols, (void)page;
    if (tokens <= 0 || hkv <= 0 || hq < hkv || hq / hkv > 128) return 0;
    const int64_t rows = std::max<int64_t>(max_q, 1) * (hq / hkv);
    return rows <= KYB_DECODE_ROWS ? kyb_attn_decode_scratch(d, (int)rows, kyb_sm_count()) : kyb_attn_prefill_scratch(d, hq / hkv, kyb_sm_count());
}

extern "C" int kyb_paged_attention(const kyb_paged_attention_args* a, void* stream) {
    KYB_REQUIRE(a, "null pointer");
    const void *q = a->q, *k_cache = a->k_cache, *v_cache = a->v_cache, *table = a->table, *kv_lens = a->kv_lens, *cu_q = a->cu_q;
    void *out = a->out, *ws = a->ws;
    const int64_t pages = a->pages, ld_table = a->ld_table, cols = a->cols, batch = a->batch, tokens = a->tokens, max_q = a->max_q, window = a->window, sinks = a->sinks;
    for (int64_t n : {a->page, a->hq, a->hkv, a->d, a->dtype}) KYB_REQUIRE(n >= 0 && n <= 65535, "a size of %lld: out of range", (long long)n);
    const int page = (int)a->page, hq = (int)a->hq, hkv = (int)a->hkv, d = (int)a->d, dtype = (int)a->dtype;
    const float scale2 = (float)a->scale * 1.4426950408889634f;          // what the kernels multiply with
    const size_t ws_bytes = a->ws_bytes < 0 ? 0 : (size_t)a->ws_bytes;
    KYB_REQUIRE(batch > 0 && batch < (1ll << 24) && tokens >= 0 && tokens < (1ll << 30) && max_q >= 0 && max_q <= (1 << 30), "batch=%lld tokens=%lld max_q=%lld: out of range", (long long)batch, (long long)tokens,
                (long long)max_q);
    KYB_REQUIRE(hkv > 0 && hq > 0 && hq % hkv == 0 && hq / hkv <= 128, "heads %d / %d: query heads are a multiple (up to 128) of the key-value heads", hq, hkv);
    KYB_REQUIRE(tokens * (hq / hkv) < (1ll << 30), "%lld tokens of %d heads a group: out of range", (long long)tokens, hq / hkv);
    KYB_REQUIRE(d == 64 || d == 128, "d=%d: heads of 64 or 128", d);
    KYB_REQUIRE(dtype == 1 || dtype == 2, "dtype=%d: 1 (fp16) or 2 (bf16)", dtype);
    KYB_REQUIRE(page >= 16 && page <= 256 && (page & (page - 1)) == 0 && pages > 0 && pages < (1ll << 31) - 1, "page=%d pages=%lld: a power of two from 16 to 256, at least one page", page,
                (long long)pages);
    KYB_REQUIRE(cols > 0 && ld_table >= cols && cols <= (1 << 30) / page, "table of %lld columns (row stride %lld), %d tokens a page: out of range", (long long)cols, (long long)ld_table, page);
    KYB_REQUIRE(window >= 0 && sinks >= 0 && (window > 0 || sinks == 0), "window=%lld sinks=%lld: not negative, sinks only with a window", (long long)window, (long long)sinks);
    KYB_REQUIRE(scale2 - scale2 == 0.f, "scale=%g: a finite number, and so times log2(e) in 32 bits", a->scale);
    if (tokens == 0) return KYB_OK;
    KYB_REQUIRE(q && k_cache && v_cache && table && kv_lens && cu_q && out, "null pointer");
    for (int64_t s : {a->q_token, a->q_head, a->k_page, a->k_head, a->v_page, a->v_head, a->out_token, a->out_head})
        KYB_REQUIRE(s % 8 == 0 && s >= 0, "a stride of %lld elements: strides are multiples of 8 elements (16 bytes)", (long long)s);
    KYB_REQUIRE((((uintptr_t)q | (uintptr_t)k_cache | (uintptr_t)v_cache | (uintptr_t)out) & 15) == 0, "pointers must be 16-byte aligned");
    unsigned int* status = kyb_device_status_word();
    KYB_REQUIRE(status, "could not set up the device status word");
    KybAttnCall c;
    kyb::AttnParams& p = c.p;
    p.q = (const uint8_t*)q, p.o = (uint8_t*)out, p.q_t = a->q_token, p.q_h = a->q_head, p.o_t = a->out_token, p.o_h = a->out_head;
    p.table = (const int*)table, p.ld_table = ld_table, p.kv_lens = (const int*)kv_lens, p.cu_q = (const int*)cu_q;
    p.batch = (int)batch, p.tokens = (int)tokens, p.hq = hq, p.hkv = hkv, p.group = hq / hkv, p.pages = (int)pages, p.cap = (int)(cols * page);
    p.window = (int)std::min<int64_t>(window, 1 << 30), p.sinks = (int)std::min<int64_t>(sinks, 1 << 30), p.scale2 = scale2, p.status = status;
    // a hidden score is -inf and stays so times the scale: 0 would make it NaN, the smallest normal number gives the same weights
    if (!(p.scale2 >= FLT_MIN || p.scale2 <= -FLT_MIN)) p.scale2 = FLT_MIN;
    p.page_log2 = 0, p.block_tokens = 0, p.parts = nullptr, p.notes = nullptr;
    while ((1 << p.page_log2) < page) ++p.page_log2;
    c.k = k_cache, c.v = v_cache, c.k_p = a->k_page, c.k_h = a->k_head, c.v_p = a->v_page, c.v_h = a->v_head, c.tokens = tokens, c.d = d, c.dtype = dtype, c.page = page, c.sms = kyb_sm_count();
    c.st = (cudaStream_t)stream;
    KYB_REQUIRE(c.sms > 0, "no CUDA device");
    const size_t need = kyb_paged_attention_workspace_bytes(batch, tokens, max_q, cols, page, hq, hkv, d);
    if (ws_bytes < need || (need && !ws)) {
        kyb_set_error("workspace of %zu bytes, %zu needed", ws_bytes, need);
        return KYB_EWORKSPACE;
    }
    KYB_REQUIRE(!need || ((uintptr_t)ws & 15) == 0, "the workspace must be 16-byte aligned");
    const int64_t rows = std::max<int64_t>(max_q, 1) * p.group;
    if (rows <= KYB_DECODE_ROWS) return kyb_attn_decode(c, (int)rows, ws);
    return kyb_attn_prefill(c, ws);
}
