// XLA FFI handlers for every entry point of libbux_amd (include/bux_amd.h): what bux
// binds as jax.ffi targets so that the kernels run inside jit on XLA's stream, with XLA
// owning every buffer. Each handler unpacks XLA's buffers, reads the shapes the C ABI
// takes from them, calls the entry point on XLA's stream and turns a nonzero status into
// an ffi::Error carrying bux_last_error().
//
// Conventions: an empty buffer (0 bytes) stands for a NULL argument (an absent index,
// `filled`, bias, copy not asked for); settings are attributes; in-place outputs
// (bux_expert_bias_add's x, bux_expert_bias_weight_grad's d_weights) are results the
// caller aliases to their input (jax.ffi.ffi_call's input_output_aliases). A listed
// GEMM's tile list is an argument: the kernels write it only to refuse a list made for
// other dimensions.
//
// Built only where the XLA FFI headers are (jax.ffi.include_dir(), or
// BUX_XLA_FFI_INCLUDE): `python -m bux_amd.build` makes libbux_amd_xla.so next to
// libbux_amd.so then, and skips it otherwise. Without the headers this file is empty.

#if __has_include("xla/ffi/api/ffi.h")

#include <hip/hip_runtime.h>

#include <cstdint>
#include <string>

#include "bux_amd.h"
#include "xla/ffi/api/ffi.h"

namespace ffi = xla::ffi;

namespace {

using Stream = ffi::PlatformStream<hipStream_t>;
using In = ffi::AnyBuffer;
using Out = ffi::Result<ffi::AnyBuffer>;

template <typename T>
T* at(const In& b) {
  return b.size_bytes() ? static_cast<T*>(b.untyped_data()) : nullptr;
}
template <typename T>
T* at(Out& b) {
  return b->size_bytes() ? static_cast<T*>(b->untyped_data()) : nullptr;
}
int64_t dim(const In& b, int i) {
  const auto d = b.dimensions();
  return d[i < 0 ? static_cast<int>(d.size()) + i : i];
}
int64_t dim(Out& b, int i) {
  const auto d = b->dimensions();
  return d[i < 0 ? static_cast<int>(d.size()) + i : i];
}
ffi::Error status(int rc) {
  if (rc == 0) return ffi::Error::Success();
  return ffi::Error(ffi::ErrorCode::kInternal, std::string(bux_last_error()));
}
// An operand the C ABI takes as a pointer alone, whose length it cannot check.
ffi::Error mismatch(const char* what) {
  return ffi::Error(ffi::ErrorCode::kInvalidArgument, std::string(what));
}
// Whether a buffer holds `count` elements of `type`; one that may be absent (an empty buffer) does.
bool holds(const In& b, ffi::DataType type, int64_t count) {
  return b.element_type() == type && static_cast<int64_t>(b.element_count()) == count;
}
bool absent_or(const In& b, ffi::DataType type, int64_t count) {
  return b.size_bytes() == 0 || holds(b, type, count);
}
bool holds(Out& b, ffi::DataType type, int64_t count) { return holds(*b, type, count); }
bool absent_or(Out& b, ffi::DataType type, int64_t count) { return absent_or(*b, type, count); }
// Codes: bytes, whatever XLA calls them.
bool holds_bytes(const In& b, int64_t count) {
  return static_cast<int64_t>(b.size_bytes()) == count;
}
bool holds_bytes(Out& b, int64_t count) { return holds_bytes(*b, count); }
bool ranked(const In& b, size_t rank) { return b.dimensions().size() == rank; }
bool ranked(Out& b, size_t rank) { return ranked(*b, rank); }
bool layer_type(const In& b) {
  return b.element_type() == ffi::DataType::BF16 || b.element_type() == ffi::DataType::F32;
}
// A row's bytes of 8-bit codes.
int64_t whole_128(int64_t k) { return (k + 127) / 128 * 128; }

int dtype_of(Out& y) { return y->element_type() == ffi::DataType::F32 ? BUX_F32 : BUX_BF16; }
bool f32(const In& b) { return b.element_type() == ffi::DataType::F32; }

bux_ffn ffn_of(int64_t activation, int64_t gated, int64_t clamped, float limit, int64_t capped,
               float up_softcap, float up_offset) {
  return bux_ffn{static_cast<int32_t>(activation), static_cast<int32_t>(gated),
                 static_cast<int32_t>(clamped), limit, static_cast<int32_t>(capped), up_softcap,
                 up_offset};
}

bux_norm norm_of(int64_t kind, int64_t affine, int64_t zero_centered, int64_t scale_input,
                 int64_t bias, float eps) {
  return bux_norm{static_cast<int32_t>(kind), static_cast<int32_t>(affine),
                  static_cast<int32_t>(zero_centered), static_cast<int32_t>(scale_input),
                  static_cast<int32_t>(bias), eps};
}

}  // namespace

// The activation's settings (bux_ffn), as attributes.
#define BUX_FFN_ATTRS                                                                      \
  .Attr<int64_t>("activation").Attr<int64_t>("gated").Attr<int64_t>("clamped")            \
      .Attr<float>("limit").Attr<int64_t>("capped").Attr<float>("up_softcap")              \
      .Attr<float>("up_offset")
#define BUX_FFN_PARAMS                                                                     \
  int64_t activation, int64_t gated, int64_t clamped, float limit, int64_t capped,        \
      float up_softcap, float up_offset
#define BUX_FFN ffn_of(activation, gated, clamped, limit, capped, up_softcap, up_offset)
#define BUX_NORM_ATTRS                                                                     \
  .Attr<int64_t>("kind").Attr<int64_t>("affine").Attr<int64_t>("zero_centered")           \
      .Attr<int64_t>("scale_input").Attr<int64_t>("norm_bias").Attr<float>("eps")
#define BUX_NORM_PARAMS                                                                    \
  int64_t kind, int64_t affine, int64_t zero_centered, int64_t scale_input,               \
      int64_t norm_bias, float eps
#define BUX_NORM norm_of(kind, affine, zero_centered, scale_input, norm_bias, eps)

// --- a-1: the sort by expert ---------------------------------------------------------

static ffi::Error MoePermute(hipStream_t s, In idx, int64_t num_experts, Out order, Out inverse,
                             Out sizes, Out offsets, Out ws) {
  return status(bux_moe_permute(at<const int32_t>(idx), static_cast<int64_t>(idx.element_count()),
                                static_cast<int32_t>(num_experts), at<int32_t>(order),
                                at<int32_t>(inverse), at<int32_t>(sizes), at<int32_t>(offsets),
                                at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMoePermute, MoePermute,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Attr<int64_t>("num_experts")
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// weights and row_weights: one a pick, bfloat16 or float32 both; list: bux_mx_grouped_tiles's
// buffer, or empty.
static ffi::Error MoePermuteLayer(hipStream_t s, In idx, In weights, int64_t num_experts,
                                  int64_t m, int64_t height, Out order, Out inverse, Out sizes,
                                  Out offsets, Out row_weights, Out list, Out ws) {
  if (!(f32(weights) || weights.element_type() == ffi::DataType::BF16) ||
      weights.element_count() != idx.element_count() ||
      row_weights->element_type() != weights.element_type() ||
      row_weights->element_count() != idx.element_count())
    return mismatch("BuxMoePermuteLayer: weights and row_weights are one bfloat16 or float32 a pick");
  return status(bux_moe_permute_layer(
      at<const int32_t>(idx), static_cast<int64_t>(idx.element_count()),
      static_cast<int32_t>(num_experts), at<const void>(weights),
      f32(weights) ? 4 : 2, at<int32_t>(order), at<int32_t>(inverse),
      at<int32_t>(sizes), at<int32_t>(offsets), at<void>(row_weights), at<void>(list),
      list->size_bytes(), m, height, at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMoePermuteLayer, MoePermuteLayer,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("num_experts").Attr<int64_t>("m")
                                  .Attr<int64_t>("height").Ret<In>().Ret<In>().Ret<In>().Ret<In>()
                                  .Ret<In>().Ret<In>().Ret<In>());

// --- a-4: MXFP8 quantization -----------------------------------------------------------

// x [groups, rows, cols] (or with an index the matrix read from), bfloat16 or float32;
// index and filled may be empty; a copy's results empty when not asked for.
static ffi::Error MxQuantize(hipStream_t s, In x, In index, In filled, int64_t index_div,
                             int64_t groups, int64_t rows, int64_t height, int64_t flags,
                             Out values, Out scales, Out t_values, Out t_scales) {
  if (f32(x))
    return status(bux_mx_quantize_f32(at<const float>(x), at<const int32_t>(index),
                                      static_cast<int32_t>(index_div), dim(x, 0), groups, rows,
                                      dim(x, -1), height, at<const int32_t>(filled),
                                      static_cast<int>(flags), at<uint8_t>(values),
                                      at<uint8_t>(scales), at<uint8_t>(t_values),
                                      at<uint8_t>(t_scales), s));
  return status(bux_mx_quantize(at<const uint16_t>(x), at<const int32_t>(index),
                                static_cast<int32_t>(index_div), dim(x, 0), groups, rows,
                                dim(x, -1), height,
                                at<const int32_t>(filled), static_cast<int>(flags),
                                at<uint8_t>(values), at<uint8_t>(scales), at<uint8_t>(t_values),
                                at<uint8_t>(t_scales), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxQuantize, MxQuantize,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("index_div").Attr<int64_t>("groups")
                                  .Attr<int64_t>("rows").Attr<int64_t>("height")
                                  .Attr<int64_t>("flags")
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// --- a-6, a-7: the grouped MXFP8 GEMMs -----------------------------------------------------
// Tiled operands: a values [K/64, m, 64]; b values [g, K/64, n, 64]; the contract's a
// [M/64, d, 64] and b [M/64, f, 64].

static ffi::Error MxRows(hipStream_t s, In av, In as, In bv, In bs, In sizes, Out y, Out ws) {
  return status(bux_mx_grouped_rows(at<const uint8_t>(av), at<const uint8_t>(as),
                                    at<const uint8_t>(bv), at<const uint8_t>(bs),
                                    at<const int32_t>(sizes), static_cast<int32_t>(dim(bv, 0)),
                                    dim(av, 1), dim(bv, 2), dim(av, 0) * 64, dim(y, 0),
                                    dtype_of(y), at<void>(y), at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxRows, MxRows,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Ret<In>().Ret<In>());

static ffi::Error MxRowsStarted(hipStream_t s, In av, In as, In bv, In bs, In sizes, In starts,
                                Out y, Out ws) {
  return status(bux_mx_grouped_rows_started(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<const int32_t>(sizes), at<const int32_t>(starts), static_cast<int32_t>(dim(bv, 0)),
      dim(av, 1), dim(bv, 2), dim(av, 0) * 64, dim(y, 0), dtype_of(y), at<void>(y),
      at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxRowsStarted, MxRowsStarted,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Ret<In>().Ret<In>());

static ffi::Error MxTiles(hipStream_t s, In sizes, int64_t m, int64_t height, Out list) {
  return status(bux_mx_grouped_tiles(at<const int32_t>(sizes),
                                     static_cast<int32_t>(sizes.element_count()), m, height,
                                     at<void>(list), list->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxTiles, MxTiles,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Attr<int64_t>("m")
                                  .Attr<int64_t>("height").Ret<In>());

static ffi::Error MxRowsListed(hipStream_t s, In av, In as, In bv, In bs, In list, Out y) {
  return status(bux_mx_grouped_rows_listed(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<void>(list), list.size_bytes(), static_cast<int32_t>(dim(bv, 0)), dim(av, 1), dim(bv, 2),
      dim(av, 0) * 64, dim(y, 0), dtype_of(y), at<void>(y), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxRowsListed, MxRowsListed,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Ret<In>());

// bias [groups, n] in y's dtype.
static ffi::Error MxRowsBiased(hipStream_t s, In av, In as, In bv, In bs, In list, In bias,
                               Out y) {
  if (bias.element_type() != y->element_type() ||
      static_cast<int64_t>(bias.element_count()) != dim(bv, 0) * dim(bv, 2))
    return mismatch("BuxMxRowsBiased: bias is [groups, n] of y's dtype");
  return status(bux_mx_grouped_rows_biased(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<void>(list), list.size_bytes(), static_cast<int32_t>(dim(bv, 0)), dim(av, 1), dim(bv, 2),
      dim(av, 0) * 64, dim(y, 0), dtype_of(y), at<const void>(bias), at<void>(y), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxRowsBiased, MxRowsBiased,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Ret<In>());

static ffi::Error MxContract(hipStream_t s, In av, In as, In bv, In bs, In sizes, Out dw,
                             Out ws) {
  return status(bux_mx_grouped_contract(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<const int32_t>(sizes), static_cast<int32_t>(sizes.element_count()), dim(av, 1),
      dim(bv, 1), dim(av, 0) * 64, dtype_of(dw), at<void>(dw), at<void>(ws), ws->size_bytes(),
      s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxContract, MxContract,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Ret<In>().Ret<In>());

static ffi::Error MxContractListed(hipStream_t s, In av, In as, In bv, In bs, In list,
                                   int64_t groups, Out dw) {
  return status(bux_mx_grouped_contract_listed(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<void>(list), list.size_bytes(), static_cast<int32_t>(groups), dim(av, 1), dim(bv, 1),
      dim(av, 0) * 64, dtype_of(dw), at<void>(dw), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxContractListed, MxContractListed,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Attr<int64_t>("groups").Ret<In>());

// --- a-10: the bfloat16 grouped GEMMs ----------------------------------------------------

// ws: a u8 result of bux_bf16_grouped_rows_workspace_size (_contract_) bytes.
// float32 x (a layer in float32): bux_bf16_grouped_rows_f32 (_contract_f32), the same
// workspace.
static ffi::Error Bf16Rows(hipStream_t s, In x, In w, In sizes, int64_t transposed, Out y,
                           Out ws) {
  if (f32(x))
    return status(bux_bf16_grouped_rows_f32(at<const float>(x), at<const float>(w),
                                            static_cast<int>(transposed), at<const int32_t>(sizes),
                                            static_cast<int32_t>(dim(w, 0)), dim(x, 0), dim(y, 1),
                                            dim(x, 1), at<float>(y), at<void>(ws),
                                            ws->size_bytes(), s));
  return status(bux_bf16_grouped_rows(at<const uint16_t>(x), at<const uint16_t>(w),
                                      static_cast<int>(transposed), at<const int32_t>(sizes),
                                      static_cast<int32_t>(dim(w, 0)), dim(x, 0), dim(y, 1),
                                      dim(x, 1), at<uint16_t>(y), at<void>(ws), ws->size_bytes(),
                                      s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxBf16Rows, Bf16Rows,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("transposed").Ret<In>().Ret<In>());

static ffi::Error Bf16Contract(hipStream_t s, In x, In dy, In sizes, Out dw, Out ws) {
  if (f32(x))
    return status(bux_bf16_grouped_contract_f32(at<const float>(x), at<const float>(dy),
                                                at<const int32_t>(sizes),
                                                static_cast<int32_t>(sizes.element_count()),
                                                dim(x, 0), dim(x, 1), dim(dy, 1), at<float>(dw),
                                                at<void>(ws), ws->size_bytes(), s));
  return status(bux_bf16_grouped_contract(at<const uint16_t>(x), at<const uint16_t>(dy),
                                          at<const int32_t>(sizes),
                                          static_cast<int32_t>(sizes.element_count()), dim(x, 0),
                                          dim(x, 1), dim(dy, 1), at<uint16_t>(dw), at<void>(ws),
                                          ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxBf16Contract, Bf16Contract,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Ret<In>().Ret<In>());

static ffi::Error Bf16RowsListed(hipStream_t s, In x, In w, In list, int64_t transposed, Out y) {
  if (f32(x))
    return status(bux_bf16_grouped_rows_listed_f32(
        at<const float>(x), at<const float>(w), static_cast<int>(transposed),
        static_cast<int32_t>(dim(w, 0)), dim(x, 0), dim(y, 1), dim(x, 1), at<float>(y),
        at<void>(list), list.size_bytes(), s));
  return status(bux_bf16_grouped_rows_listed(
      at<const uint16_t>(x), at<const uint16_t>(w), static_cast<int>(transposed),
      static_cast<int32_t>(dim(w, 0)), dim(x, 0), dim(y, 1), dim(x, 1), at<uint16_t>(y),
      at<void>(list), list.size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxBf16RowsListed, Bf16RowsListed,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("transposed").Ret<In>());

static ffi::Error Bf16ContractListed(hipStream_t s, In x, In dy, In list, Out dw) {
  if (f32(x))
    return status(bux_bf16_grouped_contract_listed_f32(
        at<const float>(x), at<const float>(dy), static_cast<int32_t>(dim(dw, 0)), dim(x, 0),
        dim(x, 1), dim(dy, 1), at<float>(dw), at<void>(list), list.size_bytes(), s));
  return status(bux_bf16_grouped_contract_listed(
      at<const uint16_t>(x), at<const uint16_t>(dy), static_cast<int32_t>(dim(dw, 0)), dim(x, 0),
      dim(x, 1), dim(dy, 1), at<uint16_t>(dw), at<void>(list), list.size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxBf16ContractListed, Bf16ContractListed,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Ret<In>());

// --- a-2, a-3: the token path's gathers and sums ---------------------------------------

static ffi::Error TokenRows(hipStream_t s, In z, In order, int64_t k, Out rows) {
  return status(bux_token_rows(at<const uint16_t>(z), dim(z, 0), at<const int32_t>(order),
                               dim(rows, 0), static_cast<int32_t>(k), dim(z, -1),
                               at<uint16_t>(rows), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxTokenRows, TokenRows,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("k").Ret<In>());

// inverse [t, k]; y and out bfloat16 or float32
static ffi::Error TokenSums(hipStream_t s, In y, In inverse, Out out) {
  if (f32(y))
    return status(bux_token_sums_f32(at<const float>(y), dim(y, 0), at<const int32_t>(inverse),
                                     dim(inverse, 0), static_cast<int32_t>(dim(inverse, 1)),
                                     dim(y, 1), at<float>(out), s));
  return status(bux_token_sums(at<const uint16_t>(y), dim(y, 0), at<const int32_t>(inverse),
                               dim(inverse, 0), static_cast<int32_t>(dim(inverse, 1)), dim(y, 1),
                               at<uint16_t>(out), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxTokenSums, TokenSums,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Ret<In>());

// --- a-8: the expert FFN's activation, biases and output norm ------------------------
// projected (m, f, 2) gated or (m, f) plain, as `gated` says; filled may be empty.

static ffi::Error GluForward(hipStream_t s, In projected, In weights, In filled, BUX_FFN_PARAMS,
                             Out h) {
  const bux_ffn ffn = BUX_FFN;
  if (f32(projected))  // a layer in float32
    return status(bux_glu_forward_f32(at<const float>(projected), at<const float>(weights),
                                      at<const int32_t>(filled), dim(h, 0), dim(h, 1), &ffn,
                                      at<float>(h), s));
  return status(bux_glu_forward(at<const uint16_t>(projected), at<const uint16_t>(weights),
                                at<const int32_t>(filled), dim(h, 0), dim(h, 1), &ffn,
                                at<uint16_t>(h), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxGluForward, GluForward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  BUX_FFN_ATTRS.Ret<In>());

static ffi::Error GluBackward(hipStream_t s, In projected, In weights, In dh, In filled,
                              BUX_FFN_PARAMS, Out d_projected, Out d_weights) {
  const bux_ffn ffn = BUX_FFN;
  if (f32(projected))  // a layer in float32
    return status(bux_glu_backward_f32(at<const float>(projected), at<const float>(weights),
                                       at<const float>(dh), at<const int32_t>(filled), dim(dh, 0),
                                       dim(dh, 1), &ffn, at<float>(d_projected),
                                       at<float>(d_weights), s));
  return status(bux_glu_backward(at<const uint16_t>(projected), at<const uint16_t>(weights),
                                 at<const uint16_t>(dh), at<const int32_t>(filled), dim(dh, 0),
                                 dim(dh, 1), &ffn, at<uint16_t>(d_projected),
                                 at<uint16_t>(d_weights), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxGluBackward, GluBackward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>() BUX_FFN_ATTRS.Ret<In>().Ret<In>());

// h may be an empty result (not kept); f from the row copy's K is not exact, so it is an
// attribute, as are m and height.
static ffi::Error GluQuantize(hipStream_t s, In projected, In weights, In filled, BUX_FFN_PARAMS,
                              int64_t m, int64_t f, int64_t height, Out h, Out values, Out scales,
                              Out t_values, Out t_scales) {
  const bux_ffn ffn = BUX_FFN;
  if (f32(projected))  // a layer in float32: projected, weights and h float32
    return status(bux_glu_quantize_f32(at<const float>(projected), at<const float>(weights),
                                       at<const int32_t>(filled), m, f, &ffn, height,
                                       at<float>(h), at<uint8_t>(values), at<uint8_t>(scales),
                                       at<uint8_t>(t_values), at<uint8_t>(t_scales), s));
  return status(bux_glu_quantize(at<const uint16_t>(projected), at<const uint16_t>(weights),
                                 at<const int32_t>(filled), m, f, &ffn, height, at<uint16_t>(h),
                                 at<uint8_t>(values), at<uint8_t>(scales), at<uint8_t>(t_values),
                                 at<uint8_t>(t_scales), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxGluQuantize, GluQuantize,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  BUX_FFN_ATTRS.Attr<int64_t>("m").Attr<int64_t>("f")
                                  .Attr<int64_t>("height").Ret<In>().Ret<In>().Ret<In>()
                                  .Ret<In>().Ret<In>());

static ffi::Error GluBackwardQuantize(hipStream_t s, In projected, In weights, In dh, In filled,
                                      BUX_FFN_PARAMS, int64_t height, Out d_projected,
                                      Out values, Out scales, Out t_values, Out t_scales,
                                      Out d_weights, Out ws) {
  const bux_ffn ffn = BUX_FFN;
  if (f32(projected))  // a layer in float32
    return status(bux_glu_backward_quantize_f32(
        at<const float>(projected), at<const float>(weights), at<const float>(dh),
        at<const int32_t>(filled), dim(dh, 0), dim(dh, 1), &ffn, height, at<float>(d_projected),
        at<uint8_t>(values), at<uint8_t>(scales), at<uint8_t>(t_values), at<uint8_t>(t_scales),
        at<float>(d_weights), at<void>(ws), ws->size_bytes(), s));
  return status(bux_glu_backward_quantize(
      at<const uint16_t>(projected), at<const uint16_t>(weights), at<const uint16_t>(dh),
      at<const int32_t>(filled), dim(dh, 0), dim(dh, 1), &ffn, height, at<uint16_t>(d_projected),
      at<uint8_t>(values), at<uint8_t>(scales), at<uint8_t>(t_values), at<uint8_t>(t_scales),
      at<uint16_t>(d_weights), at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxGluBackwardQuantize, GluBackwardQuantize,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>() BUX_FFN_ATTRS.Attr<int64_t>("height")
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>()
                                  .Ret<In>());

static ffi::Error MxGroupedGlu(hipStream_t s, In av, In as, In bv, In bs, In sizes, In weights,
                               BUX_FFN_PARAMS, Out projected, Out values, Out scales,
                               Out t_values, Out t_scales, Out ws) {
  const bux_ffn ffn = BUX_FFN;
  return status(bux_mx_grouped_glu(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<const int32_t>(sizes), static_cast<int32_t>(dim(bv, 0)), dim(av, 1), dim(bv, 2),
      dim(av, 0) * 64, dim(projected, 0), at<const uint16_t>(weights), &ffn,
      at<uint16_t>(projected), at<uint8_t>(values), at<uint8_t>(scales), at<uint8_t>(t_values),
      at<uint8_t>(t_scales), at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxGroupedGlu, MxGroupedGlu,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>() BUX_FFN_ATTRS.Ret<In>()
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// dy values [K/64, height, 64], W_down values [g, K/64, f, 64]; projected [rows, 2f]; the
// results d projected's two copies, then d_weights [rows], then the workspace.
static ffi::Error MxGroupedDglu(hipStream_t s, In av, In as, In bv, In bs, In sizes,
                                In projected, In weights, BUX_FFN_PARAMS, Out values,
                                Out scales, Out t_values, Out t_scales, Out d_weights, Out ws) {
  const bux_ffn ffn = BUX_FFN;
  return status(bux_mx_grouped_dglu(
      at<const uint8_t>(av), at<const uint8_t>(as), at<const uint8_t>(bv), at<const uint8_t>(bs),
      at<const int32_t>(sizes), static_cast<int32_t>(dim(bv, 0)), dim(av, 1), dim(bv, 2),
      dim(av, 0) * 64, dim(projected, 0), at<const uint16_t>(projected),
      at<const uint16_t>(weights), &ffn, nullptr, at<uint8_t>(values), at<uint8_t>(scales),
      at<uint8_t>(t_values), at<uint8_t>(t_scales), at<uint16_t>(d_weights), at<void>(ws),
      ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxGroupedDglu, MxGroupedDglu,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Arg<In>() BUX_FFN_ATTRS
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// The bias and norm entry points by element type: the bfloat16 ones (T uint16_t) or
// their float32 twins (T float); each handler picks by its rows' element type.
namespace {
int bias_add(uint16_t* x, int64_t m, int64_t w, const uint16_t* b, const int32_t* o, int32_t e,
             hipStream_t s) {
  return bux_expert_bias_add(x, m, w, b, o, e, s);
}
int bias_add(float* x, int64_t m, int64_t w, const float* b, const int32_t* o, int32_t e,
             hipStream_t s) {
  return bux_expert_bias_add_f32(x, m, w, b, o, e, s);
}
int expert_sums(const uint16_t* x, const int32_t* i, int32_t div, int64_t src,
                const uint16_t* w, int64_t m, int64_t width, const int32_t* o, int32_t e,
                float* out, hipStream_t s) {
  return bux_expert_sums(x, i, div, src, w, m, width, o, e, out, s);
}
int expert_sums(const float* x, const int32_t* i, int32_t div, int64_t src, const float* w,
                int64_t m, int64_t width, const int32_t* o, int32_t e, float* out,
                hipStream_t s) {
  return bux_expert_sums_f32(x, i, div, src, w, m, width, o, e, out, s);
}
int sums_biased(const uint16_t* y, int64_t rows, const int32_t* inv, int64_t t, int32_t k,
                int64_t width, const uint16_t* b, const int32_t* o, int32_t e,
                const uint16_t* w, uint16_t* out, hipStream_t s) {
  return bux_token_sums_biased(y, rows, inv, t, k, width, b, o, e, w, out, s);
}
int sums_biased(const float* y, int64_t rows, const int32_t* inv, int64_t t, int32_t k,
                int64_t width, const float* b, const int32_t* o, int32_t e, const float* w,
                float* out, hipStream_t s) {
  return bux_token_sums_biased_f32(y, rows, inv, t, k, width, b, o, e, w, out, s);
}
int weight_grad(const uint16_t* dy, const int32_t* i, int32_t div, int64_t src, int64_t m,
                int64_t width, const uint16_t* b, const int32_t* o, int32_t e, uint16_t* dw,
                hipStream_t s) {
  return bux_expert_bias_weight_grad(dy, i, div, src, m, width, b, o, e, dw, s);
}
int weight_grad(const float* dy, const int32_t* i, int32_t div, int64_t src, int64_t m,
                int64_t width, const float* b, const int32_t* o, int32_t e, float* dw,
                hipStream_t s) {
  return bux_expert_bias_weight_grad_f32(dy, i, div, src, m, width, b, o, e, dw, s);
}
int norm_forward(const uint16_t* y, int64_t m, int64_t d, const uint16_t* db, const int32_t* o,
                 int32_t e, const bux_norm* n, const uint16_t* sc, const uint16_t* b,
                 const uint16_t* w, uint16_t* out, hipStream_t s) {
  return bux_expert_norm_forward(y, m, d, db, o, e, n, sc, b, w, out, s);
}
int norm_forward(const float* y, int64_t m, int64_t d, const float* db, const int32_t* o,
                 int32_t e, const bux_norm* n, const float* sc, const float* b, const float* w,
                 float* out, hipStream_t s) {
  return bux_expert_norm_forward_f32(y, m, d, db, o, e, n, sc, b, w, out, s);
}
int norm_backward(const uint16_t* dy, const int32_t* i, int32_t div, int64_t src,
                  const uint16_t* y, int64_t m, int64_t d, const uint16_t* db, const int32_t* o,
                  int32_t e, const bux_norm* n, const uint16_t* sc, const uint16_t* b,
                  const uint16_t* w, uint16_t* dv, uint16_t* dw, float* dsc, float* dbias,
                  void* ws, size_t bytes, hipStream_t s) {
  return bux_expert_norm_backward(dy, i, div, src, y, m, d, db, o, e, n, sc, b, w, dv, dw, dsc,
                                  dbias, ws, bytes, s);
}
int norm_backward(const float* dy, const int32_t* i, int32_t div, int64_t src, const float* y,
                  int64_t m, int64_t d, const float* db, const int32_t* o, int32_t e,
                  const bux_norm* n, const float* sc, const float* b, const float* w, float* dv,
                  float* dw, float* dsc, float* dbias, void* ws, size_t bytes, hipStream_t s) {
  return bux_expert_norm_backward_f32(dy, i, div, src, y, m, d, db, o, e, n, sc, b, w, dv, dw,
                                      dsc, dbias, ws, bytes, s);
}
int32_t experts_in(const In& offsets) { return static_cast<int32_t>(offsets.element_count() - 1); }

template <typename T>
ffi::Error expert_bias_add_as(hipStream_t s, In bias, In offsets, Out& x_out) {
  return status(bias_add(at<T>(x_out), dim(x_out, 0),
                         static_cast<int64_t>(x_out->element_count()) / dim(x_out, 0),
                         at<const T>(bias), at<const int32_t>(offsets), experts_in(offsets), s));
}
template <typename T>
ffi::Error expert_sums_as(hipStream_t s, In x, In index, In weights, In offsets,
                          int64_t index_div, Out& out) {
  const int64_t m = index.size_bytes() ? static_cast<int64_t>(index.element_count()) : dim(x, 0);
  return status(expert_sums(at<const T>(x), at<const int32_t>(index),
                            static_cast<int32_t>(index_div), dim(x, 0), at<const T>(weights), m,
                            dim(out, 1), at<const int32_t>(offsets), experts_in(offsets),
                            at<float>(out), s));
}
template <typename T>
ffi::Error token_sums_biased_as(hipStream_t s, In y, In inverse, In bias, In offsets,
                                In weights, Out& out) {
  return status(sums_biased(at<const T>(y), dim(y, 0), at<const int32_t>(inverse),
                            dim(inverse, 0), static_cast<int32_t>(dim(inverse, 1)), dim(y, 1),
                            at<const T>(bias), at<const int32_t>(offsets), experts_in(offsets),
                            at<const T>(weights), at<T>(out), s));
}
template <typename T>
ffi::Error bias_weight_grad_as(hipStream_t s, In dy, In index, In bias, In offsets,
                               int64_t index_div, Out& d_weights_out) {
  return status(weight_grad(at<const T>(dy), at<const int32_t>(index),
                            static_cast<int32_t>(index_div), dim(dy, 0),
                            static_cast<int64_t>(d_weights_out->element_count()), dim(dy, 1),
                            at<const T>(bias), at<const int32_t>(offsets), experts_in(offsets),
                            at<T>(d_weights_out), s));
}
template <typename T>
ffi::Error norm_forward_as(hipStream_t s, In y, In down_bias, In offsets, In scale, In bias,
                           In weights, const bux_norm& norm, Out& out) {
  return status(norm_forward(at<const T>(y), dim(y, 0), dim(y, 1), at<const T>(down_bias),
                             at<const int32_t>(offsets), experts_in(offsets), &norm,
                             at<const T>(scale), at<const T>(bias), at<const T>(weights),
                             at<T>(out), s));
}
template <typename T>
ffi::Error norm_backward_as(hipStream_t s, In dy, In index, In y, In down_bias, In offsets,
                            In scale, In bias, In weights, int64_t index_div,
                            const bux_norm& norm, Out& dv, Out& d_weights, Out& d_scale,
                            Out& d_bias, Out& ws) {
  return status(norm_backward(
      at<const T>(dy), at<const int32_t>(index), static_cast<int32_t>(index_div), dim(dy, 0),
      at<const T>(y), dim(y, 0), dim(y, 1), at<const T>(down_bias), at<const int32_t>(offsets),
      experts_in(offsets), &norm, at<const T>(scale), at<const T>(bias), at<const T>(weights),
      at<T>(dv), at<T>(d_weights), at<float>(d_scale), at<float>(d_bias), at<void>(ws),
      ws->size_bytes(), s));
}
}  // namespace

// x is aliased to the result (in place): the caller passes input_output_aliases={0: 0}.
static ffi::Error ExpertBiasAdd(hipStream_t s, In x, In bias, In offsets, Out x_out) {
  return f32(x) ? expert_bias_add_as<float>(s, bias, offsets, x_out)
                : expert_bias_add_as<uint16_t>(s, bias, offsets, x_out);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxExpertBiasAdd, ExpertBiasAdd,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Ret<In>());

// index and weights may be empty; m = the index's entries, or x's rows.
static ffi::Error ExpertSums(hipStream_t s, In x, In index, In weights, In offsets,
                             int64_t index_div, Out out) {
  return f32(x) ? expert_sums_as<float>(s, x, index, weights, offsets, index_div, out)
                : expert_sums_as<uint16_t>(s, x, index, weights, offsets, index_div, out);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxExpertSums, ExpertSums,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Attr<int64_t>("index_div").Ret<In>());

// inverse [t, k]; weights are the sorted rows'.
static ffi::Error TokenSumsBiased(hipStream_t s, In y, In inverse, In bias, In offsets,
                                  In weights, Out out) {
  return f32(y) ? token_sums_biased_as<float>(s, y, inverse, bias, offsets, weights, out)
                : token_sums_biased_as<uint16_t>(s, y, inverse, bias, offsets, weights, out);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxTokenSumsBiased, TokenSumsBiased,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Ret<In>());

// d_weights is aliased to the result (added to in place): input_output_aliases={4: 0}.
static ffi::Error ExpertBiasWeightGrad(hipStream_t s, In dy, In index, In bias, In offsets,
                                       In d_weights, int64_t index_div, Out d_weights_out) {
  (void)d_weights;
  return f32(dy) ? bias_weight_grad_as<float>(s, dy, index, bias, offsets, index_div, d_weights_out)
                 : bias_weight_grad_as<uint16_t>(s, dy, index, bias, offsets, index_div,
                                                 d_weights_out);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxExpertBiasWeightGrad, ExpertBiasWeightGrad,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Attr<int64_t>("index_div").Ret<In>());

// down_bias, scale and bias may be empty.
static ffi::Error ExpertNormForward(hipStream_t s, In y, In down_bias, In offsets, In scale,
                                    In bias, In weights, BUX_NORM_PARAMS, Out out) {
  const bux_norm norm = BUX_NORM;
  return f32(y) ? norm_forward_as<float>(s, y, down_bias, offsets, scale, bias, weights, norm, out)
                : norm_forward_as<uint16_t>(s, y, down_bias, offsets, scale, bias, weights, norm,
                                            out);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxExpertNormForward, ExpertNormForward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>() BUX_NORM_ATTRS.Ret<In>());

static ffi::Error ExpertNormBackward(hipStream_t s, In dy, In index, In y, In down_bias,
                                     In offsets, In scale, In bias, In weights, int64_t index_div,
                                     BUX_NORM_PARAMS, Out dv, Out d_weights, Out d_scale,
                                     Out d_bias, Out ws) {
  const bux_norm norm = BUX_NORM;
  if (f32(y))
    return norm_backward_as<float>(s, dy, index, y, down_bias, offsets, scale, bias, weights,
                                   index_div, norm, dv, d_weights, d_scale, d_bias, ws);
  return norm_backward_as<uint16_t>(s, dy, index, y, down_bias, offsets, scale, bias, weights,
                                    index_div, norm, dv, d_weights, d_scale, d_bias, ws);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxExpertNormBackward, ExpertNormBackward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("index_div") BUX_NORM_ATTRS.Ret<In>()
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// --- the tokens' norm -------------------------------------------------------------------
// x [m, d]; residual (with summed), scale, bias, stats and d_summed may be empty.

template <typename T>
static ffi::Error token_norm_as(hipStream_t s, In x, In residual, In scale, In bias,
                                const bux_norm& norm, Out summed, Out out, Out stats) {
  if constexpr (sizeof(T) == 4)
    return status(bux_norm_forward_f32(at<const T>(x), at<const T>(residual), dim(x, 0), dim(x, 1),
                                       &norm, at<const T>(scale), at<const T>(bias), at<T>(summed),
                                       at<T>(out), at<float>(stats), s));
  else
    return status(bux_norm_forward(at<const T>(x), at<const T>(residual), dim(x, 0), dim(x, 1),
                                   &norm, at<const T>(scale), at<const T>(bias), at<T>(summed),
                                   at<T>(out), at<float>(stats), s));
}
template <typename T>
static ffi::Error token_norm_grad_as(hipStream_t s, In dy, In x, In stats, In d_summed, In scale,
                                     const bux_norm& norm, Out dx, Out d_scale, Out d_bias,
                                     Out ws) {
  if constexpr (sizeof(T) == 4)
    return status(bux_norm_backward_f32(
        at<const T>(dy), at<const T>(x), at<const float>(stats), at<const T>(d_summed), dim(x, 0),
        dim(x, 1), &norm, at<const T>(scale), at<T>(dx), at<float>(d_scale), at<float>(d_bias),
        at<void>(ws), ws->size_bytes(), s));
  else
    return status(bux_norm_backward(
        at<const T>(dy), at<const T>(x), at<const float>(stats), at<const T>(d_summed), dim(x, 0),
        dim(x, 1), &norm, at<const T>(scale), at<T>(dx), at<float>(d_scale), at<float>(d_bias),
        at<void>(ws), ws->size_bytes(), s));
}

static ffi::Error NormForward(hipStream_t s, In x, In residual, In scale, In bias,
                              BUX_NORM_PARAMS, Out summed, Out out, Out stats) {
  const bux_norm norm = BUX_NORM;
  if (!ranked(x, 2) || !layer_type(x)) return mismatch("BuxNormForward: x is bfloat16 or float32 [m, d]");
  const int64_t m = dim(x, 0), d = dim(x, 1);
  const ffi::DataType type = x.element_type();
  if (!absent_or(residual, type, m * d) || !absent_or(summed, type, m * d) || !holds(out, type, m * d))
    return mismatch("BuxNormForward: residual, summed and out have x's shape and dtype");
  if (!absent_or(scale, type, d) || !absent_or(bias, type, d))
    return mismatch("BuxNormForward: scale and bias are [d] of x's dtype");
  if (!absent_or(stats, ffi::DataType::F32, 2 * m))
    return mismatch("BuxNormForward: stats are float32 [m, 2]");
  return f32(x) ? token_norm_as<float>(s, x, residual, scale, bias, norm, summed, out, stats)
                : token_norm_as<uint16_t>(s, x, residual, scale, bias, norm, summed, out, stats);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxNormForward, NormForward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>() BUX_NORM_ATTRS.Ret<In>().Ret<In>().Ret<In>());

static ffi::Error NormBackward(hipStream_t s, In dy, In x, In stats, In d_summed, In scale,
                               BUX_NORM_PARAMS, Out dx, Out d_scale, Out d_bias, Out ws) {
  const bux_norm norm = BUX_NORM;
  if (!ranked(x, 2) || !layer_type(x)) return mismatch("BuxNormBackward: x is bfloat16 or float32 [m, d]");
  const int64_t m = dim(x, 0), d = dim(x, 1);
  const ffi::DataType type = x.element_type();
  if (!holds(dy, type, m * d) || !absent_or(d_summed, type, m * d) || !holds(dx, type, m * d))
    return mismatch("BuxNormBackward: dy, d_summed and dx have x's shape and dtype");
  if (!absent_or(scale, type, d)) return mismatch("BuxNormBackward: scale is [d] of x's dtype");
  if (!holds(stats, ffi::DataType::F32, 2 * m))
    return mismatch("BuxNormBackward: stats are float32 [m, 2]");
  if (!absent_or(d_scale, ffi::DataType::F32, d) || !absent_or(d_bias, ffi::DataType::F32, d))
    return mismatch("BuxNormBackward: d_scale and d_bias are float32 [d]");
  return f32(x) ? token_norm_grad_as<float>(s, dy, x, stats, d_summed, scale, norm, dx, d_scale,
                                            d_bias, ws)
                : token_norm_grad_as<uint16_t>(s, dy, x, stats, d_summed, scale, norm, dx, d_scale,
                                               d_bias, ws);
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxNormBackward, NormBackward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>() BUX_NORM_ATTRS.Ret<In>().Ret<In>()
                                  .Ret<In>().Ret<In>());

// --- the experts' products in 8-bit integers -----------------------------------------------
// values [K/64, height, 64] (a stack: [groups, K/64, n, 64]), scales [height] ([groups, n]);
// index, filled and bias may be empty.

static ffi::Error Int8Quantize(hipStream_t s, In x, In index, In filled, int64_t index_div,
                               int64_t rows, Out values, Out scales, Out ws) {
  if (!ranked(x, 2) || !layer_type(x) || !ranked(values, 3))
    return mismatch("BuxInt8Quantize: x is bfloat16 or float32 [sources, cols], values [K/64, height, 64]");
  const int64_t height = dim(values, 1), cols = dim(x, 1), sources = dim(x, 0);
  if (!holds_bytes(values, whole_128(cols) * height) || !holds(scales, ffi::DataType::F32, height))
    return mismatch("BuxInt8Quantize: values [K/64, height, 64] of cols in whole 128s, scales float32 [height]");
  if (!absent_or(index, ffi::DataType::S32, static_cast<int64_t>(index.element_count())) ||
      rows > (index.size_bytes() ? static_cast<int64_t>(index.element_count()) : sources) ||
      index_div < 1 || index_div > INT32_MAX)
    return mismatch("BuxInt8Quantize: at most the rows of x, or of an int32 index with its divisor");
  if (!absent_or(filled, ffi::DataType::S32, 1)) return mismatch("BuxInt8Quantize: filled is an int32");
  const int32_t div = static_cast<int32_t>(index_div);
  if (f32(x))
    return status(bux_int8_quantize_f32(at<const float>(x), at<const int32_t>(index), div, sources,
                                        rows, cols, height, at<const int32_t>(filled),
                                        at<uint8_t>(values), at<float>(scales), at<void>(ws),
                                        ws->size_bytes(), s));
  return status(bux_int8_quantize(at<const uint16_t>(x), at<const int32_t>(index), div, sources,
                                  rows, cols, height, at<const int32_t>(filled),
                                  at<uint8_t>(values), at<float>(scales), at<void>(ws),
                                  ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxInt8Quantize, Int8Quantize,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("index_div").Attr<int64_t>("rows").Ret<In>()
                                  .Ret<In>().Ret<In>());

// projected [m, f, p] (p = 2 gated, 1 plain), weights [m].
static ffi::Error Int8Glu(hipStream_t s, In projected, In weights, In filled, BUX_FFN_PARAMS,
                          Out values, Out scales) {
  const bux_ffn ffn = BUX_FFN;
  if (!ranked(projected, 3) || !layer_type(projected) || dim(projected, 2) != (gated ? 2 : 1) ||
      !ranked(values, 3))
    return mismatch("BuxInt8Glu: projected is bfloat16 or float32 [m, f, 2 (gated) or 1], values "
                    "[K/64, height, 64]");
  const int64_t m = dim(projected, 0), f = dim(projected, 1), height = dim(values, 1);
  if (!holds(weights, projected.element_type(), m) || !absent_or(filled, ffi::DataType::S32, 1))
    return mismatch("BuxInt8Glu: weights are [m] of projected's dtype, filled an int32");
  if (!holds_bytes(values, whole_128(f) * height) || !holds(scales, ffi::DataType::F32, height))
    return mismatch("BuxInt8Glu: values [K/64, height, 64] of f in whole 128s, scales float32 [height]");
  if (f32(projected))
    return status(bux_int8_glu_f32(at<const float>(projected), at<const float>(weights),
                                   at<const int32_t>(filled), m, f, &ffn, height,
                                   at<uint8_t>(values), at<float>(scales), s));
  return status(bux_int8_glu(at<const uint16_t>(projected), at<const uint16_t>(weights),
                             at<const int32_t>(filled), m, f, &ffn, height, at<uint8_t>(values),
                             at<float>(scales), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxInt8Glu, Int8Glu,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  BUX_FFN_ATTRS.Ret<In>().Ret<In>());

// w [groups, k, n].
static ffi::Error Int8QuantizeColumns(hipStream_t s, In w, Out values, Out scales) {
  if (!ranked(w, 3) || !layer_type(w) ||
      !holds_bytes(values, dim(w, 0) * whole_128(dim(w, 1)) * dim(w, 2)) ||
      !holds(scales, ffi::DataType::F32, dim(w, 0) * dim(w, 2)))
    return mismatch("BuxInt8QuantizeColumns: w is bfloat16 or float32 [groups, k, n], values "
                    "[groups, K/64, n, 64], scales float32 [groups, n]");
  if (f32(w))
    return status(bux_int8_quantize_columns_f32(at<const float>(w), dim(w, 0), dim(w, 1), dim(w, 2),
                                                at<uint8_t>(values), at<float>(scales), s));
  return status(bux_int8_quantize_columns(at<const uint16_t>(w), dim(w, 0), dim(w, 1), dim(w, 2),
                                          at<uint8_t>(values), at<float>(scales), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxInt8QuantizeColumns, Int8QuantizeColumns,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Ret<In>().Ret<In>());

static ffi::Error Int8GroupedRowsListed(hipStream_t s, In a_values, In a_scales, In b_values,
                                        In b_scales, In list, In bias, Out y) {
  if (!ranked(a_values, 3) || !ranked(b_values, 4) || !ranked(y, 2) || !layer_type(*y) ||
      dim(a_values, 2) != 64 || dim(b_values, 3) != 64 || dim(b_values, 1) != dim(a_values, 0) ||
      dim(y, 1) != dim(b_values, 2) ||
      !holds_bytes(a_values, dim(a_values, 0) * dim(a_values, 1) * 64) ||
      !holds_bytes(b_values, dim(b_values, 0) * dim(b_values, 1) * dim(b_values, 2) * 64))
    return mismatch("BuxInt8GroupedRowsListed: codes [K/64, m, 64] times [groups, K/64, n, 64], the "
                    "product bfloat16 or float32 [height, n]");
  const int64_t columns = dim(b_values, 0) * dim(b_values, 2);
  if (!holds(a_scales, ffi::DataType::F32, dim(a_values, 1)) ||
      !holds(b_scales, ffi::DataType::F32, columns))
    return mismatch("BuxInt8GroupedRowsListed: scales are float32 [m] and [groups, n]");
  if (!absent_or(bias, y->element_type(), columns))
    return mismatch("BuxInt8GroupedRowsListed: bias is [groups, n] of the product's dtype");
  return status(bux_int8_grouped_rows_listed(
      at<const uint8_t>(a_values), at<const float>(a_scales), at<const uint8_t>(b_values),
      at<const float>(b_scales), at<void>(list), list.size_bytes(),
      static_cast<int32_t>(dim(b_values, 0)), dim(a_values, 1), dim(b_values, 2),
      dim(a_values, 0) * 64, dim(y, 0), dtype_of(y), at<const void>(bias), at<void>(y), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxInt8GroupedRowsListed, Int8GroupedRowsListed,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Ret<In>());

// --- the router ----------------------------------------------------------------------
// x [t, d], kernel [d, n_logits]; bias and choice_bias may be empty, as may the sinks,
// scores and logits results.

static ffi::Error Route(hipStream_t s, In x, In kernel, In bias, In choice_bias,
                        float logit_scale, int64_t router, int64_t scored, int64_t groups,
                        int64_t keep, int64_t k, int64_t normalize, float scaling, Out idx,
                        Out weights, Out sinks, Out scores, Out logits, Out ws) {
  return status(bux_route(
      at<const uint16_t>(x), at<const uint16_t>(kernel), at<const float>(bias), dim(x, 0),
      dim(x, 1), static_cast<int32_t>(dim(kernel, 1)), logit_scale, static_cast<int>(router),
      static_cast<int32_t>(scored), at<const float>(choice_bias), static_cast<int32_t>(groups),
      static_cast<int32_t>(keep), static_cast<int32_t>(k), static_cast<int>(normalize), scaling,
      at<int32_t>(idx), at<uint16_t>(weights), at<uint16_t>(sinks), at<float>(scores),
      at<float>(logits), at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxRoute, Route,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Attr<float>("logit_scale").Attr<int64_t>("router")
                                  .Attr<int64_t>("scored").Attr<int64_t>("groups")
                                  .Attr<int64_t>("keep").Attr<int64_t>("k")
                                  .Attr<int64_t>("normalize").Attr<float>("scaling")
                                  .Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>().Ret<In>());

// x [t, d], kernel [d, n_logits]; d_sinks, d_scores, d_logits and dz may be empty, as may the
// bias's gradient.
static ffi::Error RouteBackward(hipStream_t s, In x, In kernel, In idx, In logits, In d_weights,
                                In d_sinks, In d_scores, In d_logits, In dz, float logit_scale,
                                int64_t router, int64_t scored, int64_t normalize, float scaling,
                                Out dx, Out d_kernel, Out d_bias, Out ws) {
  constexpr ffi::DataType BF16 = ffi::DataType::BF16, F32 = ffi::DataType::F32;
  if (!ranked(x, 2) || !ranked(kernel, 2) || !ranked(idx, 2))
    return mismatch("BuxRouteBackward: x [t, d], kernel [d, n_logits] and idx [t, k]");
  const int64_t t = dim(x, 0), d = dim(x, 1), n = dim(kernel, 1), k = dim(idx, 1);
  if (!holds(x, BF16, t * d) || !holds(kernel, BF16, d * n) || !absent_or(dz, BF16, t * d) ||
      !holds(dx, BF16, t * d) || !holds(d_kernel, BF16, d * n))
    return mismatch("BuxRouteBackward: x, dz and dx are bfloat16 [t, d], kernel and d_kernel [d, n_logits]");
  if (!holds(idx, ffi::DataType::S32, t * k) || !holds(d_weights, BF16, t * k))
    return mismatch("BuxRouteBackward: idx int32 and d_weights bfloat16 [t, k]");
  if (scored < 1 || scored > n || !absent_or(d_sinks, BF16, t * (n - scored)) ||
      !absent_or(d_scores, F32, t * scored))
    return mismatch("BuxRouteBackward: d_scores float32 [t, scored], d_sinks bfloat16 [t, n_logits - scored]");
  if (!holds(logits, F32, t * n) || !absent_or(d_logits, F32, t * n) || !absent_or(d_bias, F32, n))
    return mismatch("BuxRouteBackward: logits and d_logits float32 [t, n_logits], d_bias [n_logits]");
  return status(bux_route_backward(
      at<const uint16_t>(x), at<const uint16_t>(kernel), dim(x, 0), dim(x, 1),
      static_cast<int32_t>(dim(kernel, 1)), logit_scale, static_cast<int>(router),
      static_cast<int32_t>(scored), at<const int32_t>(idx), static_cast<int32_t>(dim(idx, 1)),
      static_cast<int>(normalize), scaling, at<const float>(logits),
      at<const uint16_t>(d_weights), at<const uint16_t>(d_sinks), at<const float>(d_scores),
      at<const float>(d_logits), at<const uint16_t>(dz), at<uint16_t>(dx), at<uint16_t>(d_kernel),
      at<float>(d_bias), at<void>(ws), ws->size_bytes(), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxRouteBackward, RouteBackward,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>().Arg<In>()
                                  .Arg<In>().Arg<In>().Arg<In>().Arg<In>().Arg<In>().Arg<In>()
                                  .Attr<float>("logit_scale").Attr<int64_t>("router")
                                  .Attr<int64_t>("scored").Attr<int64_t>("normalize")
                                  .Attr<float>("scaling").Ret<In>().Ret<In>().Ret<In>()
                                  .Ret<In>());

// --- the MXFP8 wire rows ----------------------------------------------------------------

// packed [m, d + d/32]; index may be empty.
static ffi::Error MxPackRows(hipStream_t s, In x, In index, int64_t index_div, Out packed) {
  const int64_t d = dim(x, 1);
  return status(bux_mx_pack_rows(at<const uint16_t>(x), at<const int32_t>(index),
                                 static_cast<int32_t>(index_div), dim(x, 0), dim(packed, 0), d,
                                 at<uint8_t>(packed), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxPackRows, MxPackRows,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Arg<In>()
                                  .Attr<int64_t>("index_div").Ret<In>());

static ffi::Error MxUnpackRows(hipStream_t s, In packed, Out out) {
  return status(bux_mx_unpack_rows(at<const uint8_t>(packed), dim(out, 0), dim(out, 1),
                                   at<uint16_t>(out), s));
}
XLA_FFI_DEFINE_HANDLER_SYMBOL(BuxMxUnpackRows, MxUnpackRows,
                              ffi::Ffi::Bind().Ctx<Stream>().Arg<In>().Ret<In>());

#endif  // __has_include("xla/ffi/api/ffi.h")
