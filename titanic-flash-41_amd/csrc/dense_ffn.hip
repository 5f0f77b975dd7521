// The dense feed-forward operators of the C ABI (include/titanic_moe.h): residual addition + RMS norm + MXFP8 codes, quantization to
// MXFP4 and back, products with MXFP4 weights.  Nothing here allocates, frees or synchronizes.
#include "context.hpp"
#include "add_norm.cuh"
#include "mxfp4_gemm.cuh"

namespace {

bool aligned(const void* p, size_t to) { return (size_t)p % to == 0; }
// The kernels run on the device that the context was opened on: -1 where another one is current.
int check_device(const Context& c) {
    int device = 0;
    const hipError_t e = hipGetDevice(&device);
    return e != hipSuccess ? (int)e : device != c.device ? -1 : 0;
}
int type_bytes(int type) { return type == CA_TYPE_FP32 ? 4 : 2; }
// The byte-work kernels' items of eight values, one a thread.
constexpr long long kMaxItems = 0x7fffffffll;
unsigned byte_work_grid(long long items) { return (unsigned)((items + 255) / 256); }
// Sizes whose launches stay below 2^32 threads.
constexpr int kMaxRows = 1 << 22;
int check_weights(int n, int k) { return n < 1 || n > (1 << 24) || k < 32 || k > 65536 || k % 32 || (long long)n * k > 1ll << 36 ? -1 : 0; }
int check_rows(const Context& c, int rows, int k, const void* a, const void* a_scales, int a_type) {
    if (rows < 0 || rows > kMaxRows || (a_type != CA_MX_E4M3 && a_type != CA_MX_E2M1) || (a_type == CA_MX_E4M3 && k % c.g.act_block)) return -1;
    if (rows > 0 && (!a || !a_scales || !aligned(a, 16))) return -1;
    return 0;
}

}  // namespace

extern "C" {

int ca_ffn_add_norm_quant(void* context, int rows, int cols, const void* x, int64_t x_stride, const void* residual, int64_t residual_stride,
                          const void* weight, float eps, void* residual_out, int64_t residual_out_stride, void* normed, void* codes, void* scales,
                          void* codes_min, void* scales_min, void* stream) {
    if (!context || rows < 0 || rows > kMaxRows || (!codes != !scales) || (!codes_min != !scales_min) || !(eps >= 0.f)) return -1;
    const Context& c = *(const Context*)context;
    if (cols < c.g.act_block || cols > 8192 || cols % c.g.act_block) return -4;
    if (rows == 0) return 0;
    if (!x || !weight || (!normed && !codes && !codes_min && !residual_out)) return -1;
    if (x_stride < cols || x_stride % 8 || (residual && (residual_stride < cols || residual_stride % 8)) ||
        (residual_out && (residual_out_stride < cols || residual_out_stride % 8)))
        return -1;
    if (!aligned(x, 16) || !aligned(residual, 16) || !aligned(weight, 16) || !aligned(residual_out, 16) || !aligned(normed, 16) || !aligned(codes, 8) ||
        !aligned(codes_min, 8))
        return -1;
    const int device = check_device(c);
    if (device) return device;
    AddNormArgs p{(const uint16_t*)x, (const uint16_t*)residual, (const uint16_t*)weight, (uint16_t*)residual_out, (uint16_t*)normed, (uint8_t*)codes,
                  (uint8_t*)scales, (uint8_t*)codes_min, (uint8_t*)scales_min, x_stride, residual_stride, residual_out_stride, rows, cols, c.g.act_block, eps};
    tf_launch_add_norm(p, c.cus, (hipStream_t)stream);
    return (int)hipGetLastError();
}

int ca_mxfp4_quant(void* context, int rows, int cols, const void* x, int64_t x_stride, int x_type, void* words, void* scales, void* stream) {
    if (!context || rows < 0 || cols < 32 || cols % 32 || x_type < CA_TYPE_BF16 || x_type > CA_TYPE_FP32) return -1;
    if (rows == 0) return 0;
    const long long items = (long long)rows * (cols >> 3), pitch = x_stride * type_bytes(x_type);
    if (!x || !words || !scales || x_stride < cols || pitch % 16 || !aligned(x, 16) || !aligned(words, 4) || items > kMaxItems) return -1;
    const Context& c = *(const Context*)context;
    const int device = check_device(c);
    if (device) return device;
    const unsigned grid = byte_work_grid(items), count = (uint32_t)items, per_row = (uint32_t)cols >> 3, inverse = (uint32_t)((1ull << 32) / per_row);
    const hipStream_t s = (hipStream_t)stream;
    const uint8_t* from = (const uint8_t*)x;
    if (x_type == CA_TYPE_BF16) tf_mxfp4_quant<TF_TYPE_BF16><<<grid, 256, 0, s>>>(from, pitch, (uint32_t*)words, (uint8_t*)scales, count, per_row, inverse);
    else if (x_type == CA_TYPE_FP16) tf_mxfp4_quant<TF_TYPE_FP16><<<grid, 256, 0, s>>>(from, pitch, (uint32_t*)words, (uint8_t*)scales, count, per_row, inverse);
    else tf_mxfp4_quant<TF_TYPE_FP32><<<grid, 256, 0, s>>>(from, pitch, (uint32_t*)words, (uint8_t*)scales, count, per_row, inverse);
    return (int)hipGetLastError();
}
int ca_mxfp4_dequant(void* context, int rows, int cols, const void* words, const void* scales, void* out, int64_t out_stride, int out_type, void* stream) {
    if (!context || rows < 0 || cols < 32 || cols % 32 || out_type < CA_TYPE_BF16 || out_type > CA_TYPE_FP32) return -1;
    if (rows == 0) return 0;
    const long long items = (long long)rows * (cols >> 3), pitch = out_stride * type_bytes(out_type);
    if (!out || !words || !scales || out_stride < cols || pitch % 16 || !aligned(out, 16) || !aligned(words, 4) || items > kMaxItems) return -1;
    const Context& c = *(const Context*)context;
    const int device = check_device(c);
    if (device) return device;
    const unsigned grid = byte_work_grid(items), count = (uint32_t)items, per_row = (uint32_t)cols >> 3, inverse = (uint32_t)((1ull << 32) / per_row);
    const hipStream_t s = (hipStream_t)stream;
    uint8_t* to = (uint8_t*)out;
    if (out_type == CA_TYPE_BF16) tf_mxfp4_dequant<TF_TYPE_BF16><<<grid, 256, 0, s>>>((const uint32_t*)words, (const uint8_t*)scales, to, pitch, count, per_row, inverse);
    else if (out_type == CA_TYPE_FP16) tf_mxfp4_dequant<TF_TYPE_FP16><<<grid, 256, 0, s>>>((const uint32_t*)words, (const uint8_t*)scales, to, pitch, count, per_row, inverse);
    else tf_mxfp4_dequant<TF_TYPE_FP32><<<grid, 256, 0, s>>>((const uint32_t*)words, (const uint8_t*)scales, to, pitch, count, per_row, inverse);
    return (int)hipGetLastError();
}

int64_t ca_mxfp4_words_bytes(int n, int k) { return check_weights(n, k) ? -1 : (int64_t)((n + 15) / 16) * ((k + 127) / 128) * 1024; }
int64_t ca_mxfp4_scales_bytes(int n, int k) { return check_weights(n, k) ? -1 : (int64_t)((n + 15) / 16) * ((k + 511) / 512) * 256; }
int ca_mxfp4_prepare(void* context, int n, int k, const void* words, const void* scales, void* prepared_words, void* prepared_scales, void* stream) {
    if (!context || check_weights(n, k) || !words || !scales || !prepared_words || !prepared_scales || words == prepared_words || scales == prepared_scales ||
        !aligned(words, 16) || !aligned(prepared_words, 16) || !aligned(prepared_scales, 16))
        return -1;
    const int device = check_device(*(const Context*)context);
    if (device) return device;
    const long long chunks = ca_mxfp4_words_bytes(n, k) / 16, scale_words = ca_mxfp4_scales_bytes(n, k) / 4;
    tf_mxfp4_prepare_words<<<(unsigned)((chunks + 255) / 256), 256, 0, (hipStream_t)stream>>>((const u4v*)words, (u4v*)prepared_words, n, k, chunks);
    tf_mxfp4_prepare_scales<<<(unsigned)((scale_words + 255) / 256), 256, 0, (hipStream_t)stream>>>((const uint8_t*)scales, (uint32_t*)prepared_scales, n, k, scale_words);
    return (int)hipGetLastError();
}

int ca_mxfp4_linear(void* context, int rows, int n, int k, const void* a, const void* a_scales, int a_type, const void* w, const void* w_scales, void* out,
                    int64_t out_stride, void* stream) {
    if (!context || check_weights(n, k)) return -1;
    const Context& c = *(const Context*)context;
    const int bad = check_rows(c, rows, k, a, a_scales, a_type);
    if (bad) return bad;
    if (rows == 0) return 0;
    if (!w || !w_scales || !out || out_stride < n || !aligned(w, 16) || !aligned(w_scales, 16) || !aligned(out, 2)) return -1;
    const int device = check_device(c);
    if (device) return device;
    MxArgs p{};
    p.a = (const uint8_t*)a; p.a_scales = (const uint8_t*)a_scales; p.w = (const u4v*)w; p.ws = (const uint32_t*)w_scales;
    p.rows = rows; p.n = n; p.k = k; p.block_shift = a_type == CA_MX_E4M3 && c.g.act_block == 128 ? 7 : 5;
    p.out = (uint16_t*)out; p.out_stride = out_stride; p.wide = out_stride % 8 == 0 && aligned(out, 16) ? 2 : out_stride % 4 == 0 && aligned(out, 8) ? 1 : 0;
    return tf_launch_mx(p, false, a_type == CA_MX_E2M1, c.cus, (hipStream_t)stream);
}

int ca_mxfp4_swiglu(void* context, int rows, int inter, int k, const void* a, const void* a_scales, int a_type, const void* up, const void* up_scales,
                    const void* gate, const void* gate_scales, void* act, void* codes, void* scales, int out_type, void* stream) {
    if (!context || check_weights(inter, k) || (!codes != !scales) || (out_type != CA_MX_E4M3 && out_type != CA_MX_E2M1)) return -1;
    const Context& c = *(const Context*)context;
    const int bad = check_rows(c, rows, k, a, a_scales, a_type), block = out_type == CA_MX_E4M3 ? c.g.act_block : 32;
    if (bad || inter % block) return -1;
    if (rows == 0) return 0;
    if (!up || !up_scales || !gate || !gate_scales || (!act && !codes) || !aligned(up, 16) || !aligned(gate, 16) || !aligned(up_scales, 16) ||
        !aligned(gate_scales, 16) || !aligned(act, 16) || !aligned(codes, 8))
        return -1;
    const int device = check_device(c);
    if (device) return device;
    MxArgs p{};
    p.a = (const uint8_t*)a; p.a_scales = (const uint8_t*)a_scales;
    p.w = (const u4v*)up; p.ws = (const uint32_t*)up_scales; p.w2 = (const u4v*)gate; p.ws2 = (const uint32_t*)gate_scales;
    p.rows = rows; p.n = inter; p.k = k; p.block_shift = a_type == CA_MX_E4M3 && c.g.act_block == 128 ? 7 : 5;
    p.act = (uint16_t*)act; p.codes = (uint8_t*)codes; p.scales = (uint8_t*)scales; p.out_block = block; p.out_fp4 = out_type == CA_MX_E2M1;
    p.limit = c.g.swiglu_limit;
    return tf_launch_mx(p, true, a_type == CA_MX_E2M1, c.cus, (hipStream_t)stream);
}

}  // extern "C"
