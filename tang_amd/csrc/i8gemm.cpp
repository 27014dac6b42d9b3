// The 8-bit products' entry points: checks of arguments (i8gemm.hpp).
#include <algorithm>

#include "capi_util.hpp"
#include "i8gemm.hpp"
#include "kvcache.hpp"

namespace th {

static void require_weight(const th_device* dev, size_t rows, size_t cols) {
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    TH_REQUIRE(rows > 0 && cols > 0, "empty matrix");
    TH_REQUIRE(rows <= I8_MAX_ROWS && cols <= I8_MAX_K, "sizes out of range");
    TH_REQUIRE(!dev->capturing, "makes a new weight: not while a graph is captured");
}

// A q8 weight with one scale a row, whose memory `fill` enqueues the contents of.
template <typename F>
static th_qweight* new_weight(th_device* dev, size_t rows, size_t cols, F&& fill) {
    DeviceScope scope(dev);
    th_qweight* w = new th_qweight();
    w->dev = dev;
    w->bits = 8;
    w->rows = rows;
    w->cols = cols;
    w->Np = round_up(rows, 16);
    w->Kp = round_up(cols, 64);
    w->scale_dtype = TH_F32;
    w->per_row = true;
    w->data_bytes = w->Np * w->Kp;
    w->scale_bytes = w->Np * 4;
    try {
        TH_HIP(hipMalloc(&w->data, w->data_bytes));
        TH_HIP(hipMalloc(&w->scales, w->scale_bytes));
        fill(w);
    } catch (...) {
        (void)hipStreamSynchronize(dev->stream);
        if (w->data) (void)hipFree(w->data);
        if (w->scales) (void)hipFree(w->scales);
        delete w;
        throw;
    }
    device_retain(dev);
    return w;
}

// Up to 64 rows the weights' stream bounds a product, and each workgroup takes all
// rows and one to three tiles of 16 channels, so many that there is one workgroup a CU:
// 61 rows, 4096 x 11008: one tile 29.2 us, two 23.2, three 16.8.  (Up to 16 rows one tile is best: 12.3 against 12.4 us with
// two, 4096 x 4096 at one row 4.7 against 5.4.)  Beyond 768 tiles, 12288 channels on 256 CUs, there are more workgroups than
// CUs, and of those with three tiles (96 KiB) a CU holds one, so that a last round may be nearly empty: 61 rows of 4096, 12288 channels 12.9 us, 12304
// 20.4, 14336 23.0, 24576 26.3.
static I8Form i8_few_rows(size_t m, size_t n, size_t cus) {
    const size_t tiles = ceil_div(ceil_div(n, (size_t)16), cus);
    if (m <= 16) return I8Form::ROWS_1X1;
    if (m <= 32) return tiles == 1 ? I8Form::ROWS_1X2 : I8Form::ROWS_2X2;
    return tiles == 1 ? I8Form::ROWS_1X4 : tiles == 2 ? I8Form::ROWS_2X4 : I8Form::ROWS_3X4;
}

// Beyond: the tile whose rounds over the chip take least, by what one costs a CU (us, measured at K = 64 and 4096; workgroups that
// share a CU take as long as one after the other).  512 x 4096 x 4096: 64 x 64 tiles 26.3 us, 64 x 128 18.3 to 19.6, 128 x 128 25.9;
// 2048 x 4096 x 4096: 128 x 128 52.8, 128 x 256 41.6, 256 x 256 63.9; 8192 x 8192 x 8192: 128 x 256 547, 256 x 256 499.
// A 64 x 128 tile alone on its CU has two groups of waves (100 x 4096 x 11008: 18.9 against 24.4 us; 509 x 2047 x 5631, where
// two share a CU: 20.7 against 17.9).  A round counts as one however few CUs work in it: k is not split over workgroups.
I8Form i8_form(size_t m, size_t n, size_t k, size_t cus) {
    if (m <= 64) return i8_few_rows(m, n, cus);
    const double steps = (double)ceil_div(k, (size_t)64);
    struct Tile { size_t rows, cols; double fixed, step; I8Form form; };
    const Tile tiles[] = {{64, 64, 1.0, 0.175, I8Form::TILE_64X64}, {64, 128, 2.2, 0.23, I8Form::TILE_64X128},
                          {128, 128, 4.0, 0.304, I8Form::TILE_128X128}, {128, 256, 7.0, 0.47, I8Form::TILE_128X256},
                          {256, 256, 14.5, 0.8, I8Form::TILE_256X256}};
    const Tile* best = nullptr;
    double least = 0.0;
    size_t count = 0;
    for (const Tile& tile : tiles) {
        const size_t c = ceil_div(m, tile.rows) * ceil_div(n, tile.cols);
        const double t = (double)ceil_div(c, cus) * (tile.fixed + tile.step * steps);
        if (!best || t < least) {
            best = &tile;
            least = t;
            count = c;
        }
    }
    return best->form == I8Form::TILE_64X128 && count <= cus ? I8Form::TILE_64X128_TWO : best->form;
}

// A launch has below 2^32 threads (16 for each 16 x 16 results of a tile; of few rows see I8_MAX_ROWS) and 2^16 tiles of rows; whole
// blocks of quantized rows.
size_t i8_rows_at_once(size_t n) {
    return std::min<size_t>((size_t)1 << 21, std::max<size_t>(16, ((size_t)1 << 28) / ceil_div(n, (size_t)16) / 16 * 16));
}

}  // namespace th

using namespace th;

extern "C" {

int th_quantize_rows(th_device* dev, const th_buffer* x, size_t m, size_t k, th_buffer* q, th_buffer* scale) {
    TH_API_BEGIN
    TH_REQUIRE(dev && x && q && scale, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    TH_REQUIRE(x->dev == dev && q->dev == dev && scale->dev == dev, "a buffer is on another device handle");
    TH_REQUIRE(x->dtype == TH_F32 || x->dtype == TH_F16 || x->dtype == TH_BF16, "x must be f32, f16 or bf16");
    TH_REQUIRE(k > 0 && k <= I8_MAX_K, "k must be from 1 to 2^17 - 1");
    TH_REQUIRE(m < (size_t)1 << 31, "too many rows");
    const size_t kp = round_up(k, 64);
    require_len_any(x, m * k, "x");
    require_len(q, TH_I8, m * kp, "q");
    require_len(scale, TH_F32, m, "scale");
    TH_REQUIRE(scale != x, "scale must not be x");
    DeviceScope scope(dev);
    launch_quantize_rows(x->ptr, x->dtype, m, k, (int8_t*)q->ptr, (float*)scale->ptr, false, dev->stream);
    TH_API_END
}

int th_q8_pack_rows(th_device* dev, const th_buffer* q, const th_buffer* scale, size_t rows, size_t cols, th_qweight** out) {
    TH_API_BEGIN
    TH_REQUIRE(dev && q && scale && out, "null argument");
    TH_REQUIRE(q->dev == dev && scale->dev == dev, "a buffer is on another device handle");
    require_weight(dev, rows, cols);
    require_len(q, TH_I8, rows * round_up(cols, 64), "q");
    require_len(scale, TH_F32, rows, "scale");
    *out = new_weight(dev, rows, cols, [&](const th_qweight* w) { launch_q8_pack((const int8_t*)q->ptr, (const float*)scale->ptr, w, dev->stream); });
    TH_API_END
}

int th_q8_quantize(th_device* dev, const th_buffer* x, size_t rows, size_t cols, th_qweight** out) {
    TH_API_BEGIN
    TH_REQUIRE(dev && x && out, "null argument");
    TH_REQUIRE(x->dev == dev, "a buffer is on another device handle");
    TH_REQUIRE(x->dtype == TH_F32 || x->dtype == TH_F16 || x->dtype == TH_BF16, "x must be f32, f16 or bf16");
    require_weight(dev, rows, cols);
    require_len_any(x, rows * cols, "x");
    *out = new_weight(dev, rows, cols, [&](const th_qweight* w) {
        launch_quantize_rows(x->ptr, x->dtype, rows, cols, (int8_t*)w->data, (float*)w->scales, true, dev->stream);
    });
    TH_API_END
}

int th_gemm_i8(th_device* dev, const th_buffer* xq, const th_buffer* x_scale, size_t m, const th_qweight* w, const th_buffer* bias, th_buffer* y) {
    TH_API_BEGIN
    TH_REQUIRE(dev && xq && x_scale && w && y, "null argument");
    TH_REQUIRE(!dev->closed, "the device was destroyed");
    TH_REQUIRE(xq->dev == dev && x_scale->dev == dev && w->dev == dev && y->dev == dev && (!bias || bias->dev == dev),
               "a buffer or the weight is on another device handle");
    TH_REQUIRE(w->bits == 8, "weight is not q8");
    if (!w->per_row) throw Error(TH_ERR_UNSUPPORTED, "th_gemm_i8: the weight has a scale for each group of 32 (th_gemv_q8 takes those): needs one a row");
    TH_REQUIRE(w->cols <= I8_MAX_K, "sums of 2^17 products and more leave 32 bits");
    TH_REQUIRE(y->dtype == TH_F32 || y->dtype == TH_F16 || y->dtype == TH_BF16, "y must be f32, f16 or bf16");
    TH_REQUIRE(m < (size_t)1 << 31 && w->rows <= I8_MAX_ROWS, "sizes out of range");
    require_len(xq, TH_I8, m * w->Kp, "xq");
    require_len(x_scale, TH_F32, m, "x_scale");
    if (bias) require_len(bias, TH_F32, w->rows, "bias");
    require_len_any(y, m * w->rows, "y");
    TH_REQUIRE(y != x_scale && y != bias, "y must not be an input");
    DeviceScope scope(dev);
    const I8Out out{y->ptr, (const float*)x_scale->ptr, (const float*)w->scales, bias ? (const float*)bias->ptr : nullptr, y->dtype, (int)w->rows};
    launch_i8_linear(dev, w, (const int8_t*)xq->ptr, out, m);
    TH_API_END
}

}  // extern "C"
