// The host side of the operators around the paged cache (i8gemm.cpp, samplerows.cpp), over the runtime of kvcache_host.cpp and
// launchers that only check what they are handed.
#include "kvcache_host.cpp"

#include "../../tang_amd/csrc/i8gemm.cpp"
#include "../../tang_amd/csrc/samplerows.cpp"

namespace th {

static size_t g_m, g_k;  // of the last launch
void launch_quantize_rows(const void* x, th_dtype, size_t m, size_t K, int8_t* q, float* scale, bool, hipStream_t) {
    CHECK(x && q && scale);
    g_m = m;
    g_k = K;
}
void launch_q8_pack(const int8_t* q, const float* scale, const th_qweight* w, hipStream_t) {
    CHECK(q && scale && w->data && w->scales && w->data_bytes == w->Np * w->Kp && w->scale_bytes == w->Np * 4);
}
void launch_i8_linear(th_device*, const th_qweight* w, const int8_t* xq, const I8Out& out, size_t m) {
    CHECK(xq && out.y && out.xs && out.ws == w->scales && out.N == (int)w->rows);
    g_m = m;
    g_k = w->cols;
}

void launch_sample_rows(const SampleArgs& a, hipStream_t) {
    CHECK(a.x && a.u && a.token);
    g_m = a.rows;
    g_k = a.vocab;
}

}  // namespace th

extern "C" {
// (as device.cpp's; a weight whose rows have `per_row` scales or one for each group)
int th_qweight_free(th_qweight* w) {
    device_release(w->dev);
    (void)hipFree(w->data);
    (void)hipFree(w->scales);
    delete w;
    return TH_OK;
}
void host_grouped(th_qweight* w, int bits, int per_row) {
    w->bits = bits;
    w->per_row = per_row != 0;
}
int host_i8_form(size_t m, size_t n, size_t k, size_t cus) { return (int)i8_form(m, n, k, cus); }
size_t host_i8_rows(size_t n) { return i8_rows_at_once(n); }
void host_rows(th_qweight* w, size_t rows) { w->rows = rows; }
void host_last(size_t* v) {
    v[0] = g_m;
    v[1] = g_k;
}
}
