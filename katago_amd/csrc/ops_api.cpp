// ops_api.cpp — the C ABI of include/katamx_ops.h: checks of the arguments, the caller's device around the launch. Nothing here computes.
#include <algorithm>
#include <functional>
#include <string>

#include "../../include/katamx_ops.h"
#include "engine.h"
#include "ops.h"

using namespace kmx;

namespace kmx {
int apiGuarded(const std::function<void()>& f);  // kmx_api.cpp
}

static_assert((int)KMX_SCALES_NONE == (int)SCALES_NONE && (int)KMX_SCALES_ROW == (int)SCALES_ROW && (int)KMX_SCALES_MX == (int)SCALES_MX, "scale kinds");

namespace {

[[noreturn]] void refuse(const char* entry, const std::string& why) { throw Error(KMX_ERR_INVALID_ARG, std::string(entry) + ": " + why); }

int dtypeOf(const char* entry, int type) {
  if(type == KMX_PREC_FP16) return DT_F16;
  if(type == KMX_PREC_BF16) return DT_BF16;
  if(type == KMX_PREC_FP32) return DT_F32;
  refuse(entry, "the type is KMX_PREC_FP16, KMX_PREC_BF16 or KMX_PREC_FP32");
}
void aligned(const char* entry, const char* name, const void* p, size_t to) {
  if((size_t)p % to != 0) refuse(entry, std::string(name) + " must be aligned to " + std::to_string(to) + " bytes");
}

// The calling thread's device is `device` while this lives
class OnDevice {
 public:
  explicit OnDevice(int device) {
    static const int n = [] {
      int c = 0;
      return hipGetDeviceCount(&c) == hipSuccess ? c : 0;
    }();
    if(n <= 0) throw Error(KMX_ERR_DEVICE, "no usable HIP device (katamx has no CPU fallback)");
    if(device < 0 || device >= n) throw Error(KMX_ERR_INVALID_ARG, "there is no device " + std::to_string(device));
    hipCheck(hipGetDevice(&before_), "hipGetDevice");
    if(before_ != device) {
      hipCheck(hipSetDevice(device), "hipSetDevice");
      changed_ = true;
    }
  }
  ~OnDevice() {
    if(changed_) (void)hipSetDevice(before_);
  }
  OnDevice(const OnDevice&) = delete;
  OnDevice& operator=(const OnDevice&) = delete;

 private:
  int before_ = 0;
  bool changed_ = false;
};

// Rows of bytes: [rows][width] with a stride, what an output must not share with another tensor
struct Rows {
  const char* p;
  int64_t rows, stride, width;  // bytes
  const char* end() const { return p + (rows > 0 ? (rows - 1) * stride + width : 0); }
};
bool meet(const Rows& a, const Rows& b) {
  if(a.p == nullptr || b.p == nullptr || a.rows == 0 || b.rows == 0) return false;
  if(a.end() <= b.p || b.end() <= a.p) return false;
  if(a.stride == b.stride && a.stride > 0) {  // columns of one matrix: apart where the columns are
    const int64_t d = ((b.p - a.p) % a.stride + a.stride) % a.stride;
    return d < a.width || d + b.width > a.stride;
  }
  return true;
}
bool same(const Rows& a, const Rows& b) { return a.p == b.p && (a.stride == b.stride || a.rows <= 1); }

// A strided tensor of batch x seq x heads rows of head_dim elements, in bytes
struct Box {
  const char* p;
  int64_t len[3], stride[3], width;
  int64_t span() const { return (len[0] - 1) * stride[0] + (len[1] - 1) * stride[1] + (len[2] - 1) * stride[2] + width; }
};
bool tooFar(int64_t stride, int64_t len) { return stride >= (int64_t)1 << 40 || (len > 1 && stride > ((int64_t)1 << 57) / len); }
// What a box covers of every period of `period` bytes, 0 where it has no such period
int64_t within(const Box& b, int64_t period) {
  int64_t w = b.width;
  for(int d = 0; d < 3; d++) {
    if(b.len[d] <= 1 || b.stride[d] % period == 0) continue;
    if(b.stride[d] > period) return 0;
    w += (b.len[d] - 1) * b.stride[d];
  }
  return w;
}
// Do two tensors share bytes? Apart are those whose spans are, and columns of one buffer: q and k of a fused projection's output, side by side in a
// token, in a sequence or in a head. (Stranger interleavings count as shared.)
bool meet(const Box& a, const Box& b) {
  if(a.p + a.span() <= b.p || b.p + b.span() <= a.p) return false;
  for(const Box* of : {&a, &b})
    for(int d = 0; d < 3; d++) {
      const int64_t period = of->stride[d];
      if(of->len[d] <= 1 || period <= 0) continue;
      const int64_t wa = within(a, period), wb = within(b, period), at = ((b.p - a.p) % period + period) % period;
      if(wa > 0 && wb > 0 && at >= wa && at + wb <= period) return false;
    }
  return true;
}

int64_t elements(const char* entry, const char* name, int64_t rows, int64_t stride, int64_t width, bool output) {
  if(stride < 0 || (output && rows > 1 && stride < width)) refuse(entry, std::string(name) + ": rows overlap (stride " + std::to_string(stride) + ")");
  if(rows > 0 && stride > ((int64_t)1 << 58) / rows) refuse(entry, std::string(name) + ": the stride is out of range");
  return stride;
}

void checkRows(const char* entry, int64_t rows, int channels, int scaleKind, const void* codes, const void* scales) {
  if(rows < 0 || rows > 0x7fffffff) refuse(entry, "rows must be 0 .. 2^31 - 1");
  if(channels < 1 || channels > (1 << 28)) refuse(entry, "channels must be 1 .. 2^28");
  if(scaleKind != SCALES_NONE && scaleKind != SCALES_ROW && scaleKind != SCALES_MX) refuse(entry, "unknown kind of scales");
  if((codes != nullptr) != (scaleKind != SCALES_NONE) || (scales != nullptr) != (scaleKind != SCALES_NONE))
    refuse(entry, "codes and scales are given exactly where a kind of scales is");
  if(scaleKind == SCALES_MX && channels % MX_BLOCK != 0) refuse(entry, "scales for 32 channels each need a multiple of 32 channels");
  if(scaleKind == SCALES_ROW) aligned(entry, "scales", scales, 4);
}

}  // namespace

extern "C" {

int kmx_ops_version(void) { return KMX_OPS_VERSION; }

int kmx_rmsnorm(int device, void* stream, const kmx_rmsnorm_args* p) {
  return apiGuarded([&] {
    const char* const me = "kmx_rmsnorm";
    if(p == nullptr) refuse(me, "null argument");
    const int dtype = dtypeOf(me, p->type);
    const size_t es = (size_t)dtSize(dtype);
    checkRows(me, p->rows, p->channels, p->scale_kind, p->codes, p->scales);
    if(p->x == nullptr) refuse(me, "x is null");
    if((p->residual != nullptr) != (p->sum != nullptr)) refuse(me, "residual and sum are both given or both null");
    if(p->y == nullptr && p->codes == nullptr) refuse(me, "neither y nor codes is wanted");
    if(!(p->epsilon >= 0.0f) || p->epsilon > 3.0e38f) refuse(me, "epsilon must be a finite number, not negative");
    aligned(me, "x", p->x, es);
    aligned(me, "residual", p->residual, es);
    aligned(me, "sum", p->sum, es);
    aligned(me, "y", p->y, es);
    aligned(me, "weight", p->weight, 4);
    aligned(me, "beta", p->beta, 4);
    aligned(me, "mask", p->mask, 4);
    const int64_t n = p->rows, C = p->channels;
    auto rowsOf = [&](const char* name, const void* ptr, int64_t stride, size_t size, bool output) {
      if(ptr == nullptr) return Rows{nullptr, 0, 0, 0};
      return Rows{(const char*)ptr, n, elements(me, name, n, stride, C, output) * (int64_t)size, C * (int64_t)size};
    };
    const Rows x = rowsOf("x", p->x, p->x_stride, es, false), r = rowsOf("residual", p->residual, p->residual_stride, es, false);
    const Rows sum = rowsOf("sum", p->sum, p->sum_stride, es, true), y = rowsOf("y", p->y, p->y_stride, es, true);
    const Rows codes = rowsOf("codes", p->codes, p->codes_stride, 1, true);
    const int64_t scaleBytes = p->scale_kind == SCALES_ROW ? 4 * n : n * (C / MX_BLOCK);
    const Rows scales{(const char*)p->scales, p->scales != nullptr && n > 0 ? 1 : 0, scaleBytes, scaleBytes};
    const Rows w{(const char*)p->weight, 1, 4 * C, 4 * C}, beta{(const char*)p->beta, 1, 4 * C, 4 * C}, mask{(const char*)p->mask, n > 0 ? 1 : 0, 4 * n, 4 * n};
    const Rows* const in[] = {&x, &r, &w, &beta, &mask};
    const Rows* const out[] = {&sum, &y, &codes, &scales};
    for(int i = 0; i < 4; i++) {
      for(int j = 0; j < 5; j++)
        if(meet(*out[i], *in[j]) && !(i < 2 && j < 2 && same(*out[i], *in[j]))) refuse(me, "an output overlaps an input (sum and y may be x or residual itself)");
      for(int j = 0; j < i; j++)
        if(meet(*out[i], *out[j])) refuse(me, "two outputs overlap");
    }
    NormQuantArgs a;
    a.x = p->x; a.residual = p->residual; a.sum = p->sum; a.weight = p->weight; a.beta = p->beta; a.mask = p->mask; a.y = p->y;
    a.codes = (uint8_t*)p->codes; a.scales = p->scales;
    a.xStride = p->x_stride; a.residualStride = p->residual_stride; a.sumStride = p->sum_stride; a.yStride = p->y_stride; a.codesStride = p->codes_stride;
    a.rows = n; a.C = p->channels; a.scaleKind = p->scale_kind; a.normed = 1; a.eps = p->epsilon; a.perChannel = 1.0 / p->channels;
    OnDevice on(device);
    hipCheck(launchNormQuant(dtype, a, (hipStream_t)stream), "rmsnorm launch");
  });
}

int kmx_quantize(int device, void* stream, int type, int scale_kind, int64_t rows, int channels, const void* x, int64_t x_stride, void* codes,
                 int64_t codes_stride, void* scales) {
  return apiGuarded([&] {
    const char* const me = "kmx_quantize";
    const int dtype = dtypeOf(me, type);
    const int64_t es = dtSize(dtype), C = channels;
    if(scale_kind == SCALES_NONE) refuse(me, "a kind of scales is needed");
    checkRows(me, rows, channels, scale_kind, codes, scales);
    if(x == nullptr) refuse(me, "x is null");
    aligned(me, "x", x, (size_t)es);
    const int64_t scaleBytes = scale_kind == SCALES_ROW ? 4 * rows : rows * (C / MX_BLOCK);
    const Rows in{(const char*)x, rows, elements(me, "x", rows, x_stride, C, false) * es, C * es};
    const Rows out{(const char*)codes, rows, elements(me, "codes", rows, codes_stride, C, true), C};
    const Rows sc{(const char*)scales, rows > 0 ? 1 : 0, scaleBytes, scaleBytes};
    if(meet(out, in) || meet(sc, in) || meet(out, sc)) refuse(me, "codes or scales overlap another tensor");
    NormQuantArgs a = {};
    a.x = x; a.xStride = x_stride; a.codes = (uint8_t*)codes; a.codesStride = codes_stride; a.scales = scales;
    a.rows = rows; a.C = channels; a.scaleKind = scale_kind;
    OnDevice on(device);
    hipCheck(launchNormQuant(dtype, a, (hipStream_t)stream), "quantize launch");
  });
}

int kmx_linear8(int device, void* stream, const kmx_linear8_args* p) {
  return apiGuarded([&] {
    const char* const me = "kmx_linear8";
    if(p == nullptr) refuse(me, "null argument");
    const int dtype = dtypeOf(me, p->out_type);
    const int64_t es = dtSize(dtype), M = p->rows, N = p->n, K = p->k;
    if(M < 0 || M > 0x7fffffff) refuse(me, "rows must be 0 .. 2^31 - 1");
    if(N < 1 || N >= (1 << 23)) refuse(me, "n must be 1 .. 2^23 - 1");
    if(p->scale_kind != SCALES_ROW && p->scale_kind != SCALES_MX) refuse(me, "the scales are KMX_SCALES_ROW or KMX_SCALES_MX");
    const int step = p->scale_kind == SCALES_MX ? MX_BLOCK : 16;
    if(K < step || K % step != 0 || K >= (1 << 23)) refuse(me, "k must be a multiple of " + std::to_string(step) + " below 2^23");
    if(p->a == nullptr || p->w == nullptr || p->a_scales == nullptr || p->w_scales == nullptr || p->out == nullptr) refuse(me, "a, w, their scales and out are needed");
    aligned(me, "a", p->a, 16);
    aligned(me, "w", p->w, 16);
    if(p->scale_kind == SCALES_ROW) {
      aligned(me, "a_scales", p->a_scales, 4);
      aligned(me, "w_scales", p->w_scales, 4);
    }
    aligned(me, "bias", p->bias, 4);
    aligned(me, "out", p->out, (size_t)es);
    if(p->a_stride < 0 || p->w_stride < 0 || p->a_stride % 16 != 0 || p->w_stride % 16 != 0 || p->a_stride >= (1 << 23) || p->w_stride >= (1 << 23))
      refuse(me, "the strides of a and w must be multiples of 16 below 2^23");
    if(p->out_stride >= (1 << 23)) refuse(me, "out_stride must be below 2^23");
    const Rows out{(const char*)p->out, M, elements(me, "out", M, p->out_stride, N, true) * es, N * es};
    const int64_t perA = p->scale_kind == SCALES_ROW ? 4 : K / MX_BLOCK;
    const Rows in[] = {{(const char*)p->a, M, p->a_stride, K}, {(const char*)p->w, N, p->w_stride, K}, {(const char*)p->a_scales, 1, M * perA, M * perA},
                       {(const char*)p->w_scales, 1, N * perA, N * perA}, {(const char*)p->bias, 1, 4 * N, 4 * N}};
    for(const Rows& i : in)
      if(meet(out, i)) refuse(me, "out overlaps an input");
    Linear8Args a;
    a.a = (const uint8_t*)p->a; a.w = (const uint8_t*)p->w; a.aScales = p->a_scales; a.wScales = p->w_scales; a.bias = p->bias; a.out = p->out;
    a.aStride = p->a_stride; a.wStride = p->w_stride; a.outStride = p->out_stride; a.rows = M; a.N = p->n; a.K = p->k; a.scaleKind = p->scale_kind;
    OnDevice on(device);
    hipCheck(launchLinear8(dtype, a, (hipStream_t)stream), "linear8 launch");
  });
}

int kmx_rotary(int device, void* stream, const kmx_rotary_args* p) {
  return apiGuarded([&] {
    const char* const me = "kmx_rotary";
    if(p == nullptr) refuse(me, "null argument");
    const int dtype = dtypeOf(me, p->type);
    const int64_t es = dtSize(dtype);
    if(p->batch < 0 || p->seq < 0 || (p->seq > 0 && p->batch > 0x7fffffff / p->seq)) refuse(me, "batch * seq must be below 2^31");
    if(p->q_heads < 1 || p->k_heads < 0 || p->q_heads > (1 << 16) || p->k_heads > (1 << 16)) refuse(me, "q_heads must be 1 .. 65536, k_heads 0 .. 65536");
    if(p->head_dim < 2 || p->head_dim > (1 << 16) || p->pairs < 1 || 2 * p->pairs > p->head_dim) refuse(me, "2 <= 2 * pairs <= head_dim <= 65536");
    if(((int64_t)p->q_heads + p->k_heads) * p->head_dim > 0x7fffffff) refuse(me, "a token's heads must have fewer than 2^31 channels");
    if(p->axes != 1 && p->axes != 2) refuse(me, "axes must be 1 or 2");
    if(p->freq_heads < 1 || p->q_heads % p->freq_heads != 0 || p->k_heads % p->freq_heads != 0) refuse(me, "freq_heads must divide q_heads and k_heads");
    if(p->frequencies == nullptr || p->positions == nullptr) refuse(me, "frequencies and positions are needed");
    aligned(me, "frequencies", p->frequencies, 8);
    aligned(me, "positions", p->positions, p->positions_are_64bit ? 8 : 4);
    if(p->pos_batch_stride < 0 || p->pos_seq_stride < 0 || p->pos_axis_stride < 0) refuse(me, "negative strides");
    if(!(p->magnitude >= -3.0e38f && p->magnitude <= 3.0e38f)) refuse(me, "the magnitude must be finite");
    RotaryArgs a = {};
    Box in[2], out[2];
    const kmx_rotary_tensor* const t[2] = {&p->q, &p->k};
    const int heads[2] = {p->q_heads, p->k_heads};
    const bool any = p->batch > 0 && p->seq > 0;
    for(int i = 0; i < 2; i++) {
      const kmx_rotary_tensor& x = *t[i];
      a.side[i].heads = heads[i];
      if(heads[i] == 0) continue;
      const std::string name = i == 0 ? "q" : "k";
      if(x.in == nullptr || x.out == nullptr) refuse(me, name + " is null");
      aligned(me, name.c_str(), x.in, (size_t)es);
      aligned(me, name.c_str(), x.out, (size_t)es);
      const int64_t si[3] = {x.in_batch_stride, x.in_seq_stride, x.in_head_stride}, so[3] = {x.out_batch_stride, x.out_seq_stride, x.out_head_stride};
      const int64_t len[3] = {p->batch, p->seq, heads[i]};
      for(int d = 0; d < 3; d++) {
        if(si[d] < 0 || so[d] < 0) refuse(me, name + ": negative strides");
        if(tooFar(si[d], len[d]) || tooFar(so[d], len[d])) refuse(me, name + ": a stride is out of range");
      }
      // an output's elements are apart: sorted by stride, each dimension steps over all that the smaller ones span
      int order[3] = {0, 1, 2};
      for(int u = 0; u < 3; u++)
        for(int v = u + 1; v < 3; v++)
          if(so[order[v]] < so[order[u]]) std::swap(order[u], order[v]);
      int64_t inner = p->head_dim;
      for(int d : order) {
        if(len[d] <= 1) continue;
        if(so[d] < inner) refuse(me, name + ": the output's elements overlap");
        inner += (len[d] - 1) * so[d];
      }
      in[i] = Box{(const char*)x.in, {len[0], len[1], len[2]}, {si[0] * es, si[1] * es, si[2] * es}, p->head_dim * es};
      out[i] = Box{(const char*)x.out, {len[0], len[1], len[2]}, {so[0] * es, so[1] * es, so[2] * es}, p->head_dim * es};
      const bool inPlace = x.in == x.out && (len[0] <= 1 || si[0] == so[0]) && (len[1] <= 1 || si[1] == so[1]) && (len[2] <= 1 || si[2] == so[2]);
      if(!inPlace && any && meet(in[i], out[i])) refuse(me, name + ": out overlaps in and is not in itself");
      RotarySide& s = a.side[i];
      s.in = x.in; s.out = x.out;
      s.inBatch = si[0]; s.inToken = si[1]; s.inHead = si[2]; s.outBatch = so[0]; s.outToken = so[1]; s.outHead = so[2];
    }
    if(heads[1] > 0 && any && (meet(out[0], out[1]) || meet(out[0], in[1]) || meet(in[0], out[1]))) refuse(me, "q and k overlap");
    if(any) {
      const int64_t ps = p->positions_are_64bit ? 8 : 4;
      if(tooFar(p->pos_batch_stride, p->batch) || tooFar(p->pos_seq_stride, p->seq) || tooFar(p->pos_axis_stride, p->axes)) refuse(me, "positions: a stride is out of range");
      const Box pos{(const char*)p->positions, {p->batch, p->seq, p->axes}, {p->pos_batch_stride * ps, p->pos_seq_stride * ps, p->pos_axis_stride * ps}, ps};
      const int64_t freqBytes = (int64_t)p->freq_heads * p->axes * p->pairs * 8;
      const Box freq{(const char*)p->frequencies, {1, 1, 1}, {0, 0, 0}, freqBytes};
      for(int i = 0; i < (heads[1] > 0 ? 2 : 1); i++)
        if(meet(out[i], pos) || meet(out[i], freq)) refuse(me, "an output overlaps the positions or the frequencies");
    }
    a.positions = p->positions;
    a.posBatch = p->pos_batch_stride; a.posToken = p->pos_seq_stride; a.posAxis = p->pos_axis_stride; a.pos64 = p->positions_are_64bit != 0;
    a.freqs = p->frequencies; a.freqHeads = p->freq_heads; a.axes = p->axes; a.pairs = p->pairs; a.headDim = p->head_dim;
    a.seq = (int)p->seq; a.tokens = p->batch * p->seq; a.magnitude = p->magnitude; a.inverse = p->inverse != 0; a.half = p->half != 0;
    OnDevice on(device);
    hipCheck(launchRotary(dtype, a, (hipStream_t)stream), "rotary launch");
  });
}

}  // extern "C"
