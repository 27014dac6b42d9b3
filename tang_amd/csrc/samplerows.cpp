// th_sample_rows: checks of arguments (samplerows.hpp).
#include "samplerows.hpp"
#include "capi_util.hpp"
#include "kvcache.hpp"

using namespace th;

extern "C" {

int th_sample_rows(th_device* dev, const th_buffer* logits, size_t n_rows, size_t vocab, const th_buffer* u, const th_buffer* temperature,
                   const th_buffer* top_k, const th_buffer* top_p, const th_buffer* min_p, th_buffer* tokens, th_buffer* prob) {
    TH_API_BEGIN
    TH_REQUIRE(dev && logits && u && tokens, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    for (const th_buffer* b : {logits, u, temperature, top_k, top_p, min_p, (const th_buffer*)tokens, (const th_buffer*)prob})
        TH_REQUIRE(!b || b->dev == dev, "a buffer is on another device handle");
    TH_REQUIRE(vocab > 0, "empty row");
    TH_REQUIRE(vocab <= SAMPLE_MAX_VOCAB && n_rows < (size_t)1 << 31, "sizes out of range");
    TH_REQUIRE(logits->dtype == TH_F32 || logits->dtype == TH_F16 || logits->dtype == TH_BF16, "logits must be f32, f16 or bf16");
    require_len_any(logits, n_rows * vocab, "logits");
    require_len(u, TH_F32, n_rows, "u");
    if (temperature) require_len(temperature, TH_F32, n_rows, "temperature");
    if (top_p) require_len(top_p, TH_F32, n_rows, "top_p");
    if (min_p) require_len(min_p, TH_F32, n_rows, "min_p");
    if (prob) require_len(prob, TH_F32, n_rows, "prob");
    TH_REQUIRE(!top_k || top_k->dtype == TH_U32 || top_k->dtype == TH_I32, "top_k must be u32");
    if (top_k) require_len_any(top_k, n_rows, "top_k");
    TH_REQUIRE(tokens->dtype == TH_U32 || tokens->dtype == TH_I32, "tokens must be u32");
    require_len_any(tokens, n_rows, "tokens");
    for (const th_buffer* b : {logits, u, temperature, top_k, top_p, min_p})
        TH_REQUIRE(!b || (b != tokens && b != prob), "a result must not be an input");
    SampleArgs a = {};
    a.x = logits->ptr;
    a.xdt = logits->dtype;
    a.u = (const float*)u->ptr;
    a.temp = temperature ? (const float*)temperature->ptr : nullptr;
    a.top_k = top_k ? (const uint32_t*)top_k->ptr : nullptr;
    a.top_p = top_p ? (const float*)top_p->ptr : nullptr;
    a.min_p = min_p ? (const float*)min_p->ptr : nullptr;
    a.token = (uint32_t*)tokens->ptr;
    a.prob = prob ? (float*)prob->ptr : nullptr;
    a.rows = (int)n_rows;
    a.vocab = (int)vocab;
    DeviceScope scope(dev);
    launch_sample_rows(a, dev->stream);
    TH_API_END
}

}  // extern "C"
