// Calls the XLA FFI handlers of the norm, the router's backward and the 8-bit products on made-up
// buffers, the library's entry points replaced by ones that say they were reached. Prints a line a
// case: its handler, whether it is meant to be taken, and whether the library was called; after a
// refusal the error's code has to be that of an invalid argument.
#include "../bux_amd/xla/xla_ffi.cc"

#include <cstdio>

static int calls = 0;
extern "C" {
const char* bux_last_error() { return ""; }
int bux_norm_forward(const uint16_t*, const uint16_t*, int64_t, int64_t, const bux_norm*, const uint16_t*,
                     const uint16_t*, uint16_t*, uint16_t*, float*, void*) { return ++calls, 0; }
int bux_norm_forward_f32(const float*, const float*, int64_t, int64_t, const bux_norm*, const float*,
                         const float*, float*, float*, float*, void*) { return ++calls, 0; }
int bux_norm_backward(const uint16_t*, const uint16_t*, const float*, const uint16_t*, int64_t, int64_t,
                      const bux_norm*, const uint16_t*, uint16_t*, float*, float*, void*, size_t,
                      void*) { return ++calls, 0; }
int bux_norm_backward_f32(const float*, const float*, const float*, const float*, int64_t, int64_t,
                          const bux_norm*, const float*, float*, float*, float*, void*, size_t,
                          void*) { return ++calls, 0; }
int bux_int8_quantize(const uint16_t*, const int32_t*, int32_t, int64_t, int64_t, int64_t, int64_t,
                      const int32_t*, uint8_t*, float*, void*, size_t, void*) { return ++calls, 0; }
int bux_int8_quantize_f32(const float*, const int32_t*, int32_t, int64_t, int64_t, int64_t, int64_t,
                          const int32_t*, uint8_t*, float*, void*, size_t, void*) { return ++calls, 0; }
int bux_int8_glu(const uint16_t*, const uint16_t*, const int32_t*, int64_t, int64_t, const bux_ffn*,
                 int64_t, uint8_t*, float*, void*) { return ++calls, 0; }
int bux_int8_glu_f32(const float*, const float*, const int32_t*, int64_t, int64_t, const bux_ffn*, int64_t,
                     uint8_t*, float*, void*) { return ++calls, 0; }
int bux_int8_quantize_columns(const uint16_t*, int64_t, int64_t, int64_t, uint8_t*, float*,
                              void*) { return ++calls, 0; }
int bux_int8_quantize_columns_f32(const float*, int64_t, int64_t, int64_t, uint8_t*, float*,
                                  void*) { return ++calls, 0; }
int bux_int8_grouped_rows_listed(const uint8_t*, const float*, const uint8_t*, const float*, void*, size_t,
                                 int32_t, int64_t, int64_t, int64_t, int64_t, int, const void*, void*,
                                 void*) { return ++calls, 0; }
int bux_route_backward(const uint16_t*, const uint16_t*, int64_t, int64_t, int32_t, float, int, int32_t,
                       const int32_t*, int32_t, int, float, const float*, const uint16_t*,
                       const uint16_t*, const float*, const float*, const uint16_t*, uint16_t*, uint16_t*,
                       float*, void*, size_t, void*) { return ++calls, 0; }
}

using ffi::DataType;
constexpr DataType BF = DataType::BF16, F = DataType::F32, I = DataType::S32, U = DataType::U8;
static char memory[64];
struct B {  // a buffer's dtype and dimensions
  DataType type;
  std::vector<int64_t> dims;
  In in() const { return In(type, dims, memory); }
  Out out() const { return Out(in()); }
};
static const B NONE{BF, {0}};
static const B WS{U, {4096}};

static void line(const char* what, bool taken, const ffi::Error& e) {
  const bool right = calls ? e.success() : e.errc() == ffi::ErrorCode::kInvalidArgument;
  std::printf("%s %d %d %d\n", what, taken ? 1 : 0, calls, right ? 1 : 0);
  calls = 0;
}

// norm: [5, 64] rows
struct Norm {
  B x{BF, {5, 64}}, residual{BF, {5, 64}}, scale{BF, {64}}, bias{BF, {64}}, summed{BF, {5, 64}}, out{BF, {5, 64}},
      stats{F, {5, 2}}, dy{BF, {5, 64}}, d_summed{BF, {5, 64}}, dx{BF, {5, 64}}, d_scale{F, {64}}, d_bias{F, {64}};
  void forward(bool taken) const {
    line("norm", taken, NormForward(nullptr, x.in(), residual.in(), scale.in(), bias.in(), 0, 1, 0, 0, 1, 1e-6f,
                                    summed.out(), out.out(), stats.out()));
  }
  void backward(bool taken) const {
    line("norm backward", taken, NormBackward(nullptr, dy.in(), x.in(), stats.in(), d_summed.in(), scale.in(), 0,
                                              1, 0, 0, 1, 1e-6f, dx.out(), d_scale.out(), d_bias.out(), WS.out()));
  }
};
static Norm in_f32() {
  Norm n;
  for (B* b : {&n.x, &n.residual, &n.scale, &n.bias, &n.summed, &n.out, &n.dy, &n.d_summed, &n.dx}) b->type = F;
  return n;
}
template <typename S>
static S with(B S::*field, B value, S base = S{}) {
  base.*field = value;
  return base;
}

// router: 6 tokens of 32, 10 logits of which 8 are scored, 2 picks
struct Routed {
  B x{BF, {6, 32}}, kernel{BF, {32, 10}}, idx{I, {6, 2}}, logits{F, {6, 10}}, d_weights{BF, {6, 2}},
      d_sinks{BF, {6, 2}}, d_scores{F, {6, 8}}, d_logits{F, {6, 10}}, dz{BF, {6, 32}}, dx{BF, {6, 32}},
      d_kernel{BF, {32, 10}}, d_bias{F, {10}};
  int64_t scored = 8;
  void call(bool taken) const {
    line("route backward", taken,
         RouteBackward(nullptr, x.in(), kernel.in(), idx.in(), logits.in(), d_weights.in(), d_sinks.in(),
                       d_scores.in(), d_logits.in(), dz.in(), 1.0f, 0, scored, 1, 1.0f, dx.out(), d_kernel.out(),
                       d_bias.out(), WS.out()));
  }
};

// quantizer: 8 tokens of 100 columns, 12 picks, a copy of 16 rows
struct Quantize {
  B x{BF, {8, 100}}, index{I, {12}}, filled{I, {1}}, values{U, {2, 16, 64}}, scales{F, {16}};
  int64_t div = 2, rows = 12;
  void call(bool taken) const {
    line("quantize", taken, Int8Quantize(nullptr, x.in(), index.in(), filled.in(), div, rows, values.out(),
                                         scales.out(), WS.out()));
  }
};

// activation: 5 rows of 68 units, a copy of 7 rows
struct Glu {
  B projected{BF, {5, 68, 2}}, weights{BF, {5}}, filled{I, {1}}, values{U, {2, 7, 64}}, scales{F, {7}};
  int64_t gated = 1;
  void call(bool taken) const {
    line("glu", taken, Int8Glu(nullptr, projected.in(), weights.in(), filled.in(), 0, gated, 0, 0.0f, 0, 0.0f,
                               0.0f, values.out(), scales.out()));
  }
};

struct Columns {
  B w{BF, {3, 100, 12}}, values{U, {3, 2, 12, 64}}, scales{F, {3, 12}};
  void call(bool taken) const {
    line("columns", taken, Int8QuantizeColumns(nullptr, w.in(), values.out(), scales.out()));
  }
};

struct Rows {
  B a{U, {4, 20, 64}}, as{F, {20}}, b{U, {3, 4, 12, 64}}, bs{F, {3, 12}}, list{U, {512}}, bias{BF, {3, 12}},
      y{BF, {25, 12}};
  void call(bool taken) const {
    line("rows", taken, Int8GroupedRowsListed(nullptr, a.in(), as.in(), b.in(), bs.in(), list.in(), bias.in(),
                                              y.out()));
  }
};

int main() {
  for (const Norm& n : {Norm{}, in_f32(), with(&Norm::residual, NONE, with(&Norm::summed, NONE)),
                        with(&Norm::scale, NONE), with(&Norm::bias, NONE), with(&Norm::stats, NONE)})
    n.forward(true);
  for (const Norm& n :
       {with(&Norm::scale, B{F, {64}}), with(&Norm::scale, B{BF, {63}}), with(&Norm::bias, B{F, {64}}),
        with(&Norm::bias, B{BF, {32}}), with(&Norm::residual, B{F, {5, 64}}), with(&Norm::residual, B{BF, {4, 64}}),
        with(&Norm::summed, B{BF, {4, 64}}), with(&Norm::out, B{F, {5, 64}}), with(&Norm::out, B{BF, {5, 60}}),
        with(&Norm::stats, B{BF, {5, 2}}), with(&Norm::stats, B{F, {5}}), with(&Norm::x, B{F, {5, 64}}),
        with(&Norm::x, B{I, {5, 64}}), with(&Norm::x, B{BF, {5, 8, 8}}), with(&Norm::scale, B{BF, {64}}, in_f32())})
    n.forward(false);
  for (const Norm& n : {Norm{}, in_f32(), with(&Norm::d_summed, NONE), with(&Norm::scale, NONE),
                        with(&Norm::d_scale, NONE), with(&Norm::d_bias, NONE)})
    n.backward(true);
  for (const Norm& n :
       {with(&Norm::dy, B{F, {5, 64}}), with(&Norm::dy, B{BF, {4, 64}}), with(&Norm::d_summed, B{F, {5, 64}}),
        with(&Norm::d_summed, B{BF, {5, 63}}), with(&Norm::scale, B{F, {64}}), with(&Norm::scale, B{BF, {60}}),
        with(&Norm::stats, B{F, {4, 2}}), with(&Norm::stats, NONE), with(&Norm::dx, B{F, {5, 64}}),
        with(&Norm::d_scale, B{BF, {64}}), with(&Norm::d_bias, B{F, {32}}), with(&Norm::x, B{F, {5, 64}}),
        with(&Norm::dy, B{BF, {5, 64}}, in_f32())})
    n.backward(false);

  for (const Routed& r : {Routed{}, with(&Routed::d_sinks, NONE), with(&Routed::d_scores, NONE),
                         with(&Routed::d_logits, NONE), with(&Routed::dz, NONE), with(&Routed::d_bias, NONE)})
    r.call(true);
  for (const Routed& r :
       {with(&Routed::x, B{F, {6, 32}}), with(&Routed::x, B{BF, {2, 3, 32}}), with(&Routed::kernel, B{F, {32, 10}}),
        with(&Routed::kernel, B{BF, {16, 10}}), with(&Routed::idx, B{F, {6, 2}}), with(&Routed::idx, B{I, {5, 2}}),
        with(&Routed::logits, B{BF, {6, 10}}), with(&Routed::logits, B{F, {6, 8}}),
        with(&Routed::d_weights, B{F, {6, 2}}), with(&Routed::d_weights, B{BF, {6, 1}}),
        with(&Routed::d_sinks, B{F, {6, 2}}), with(&Routed::d_sinks, B{BF, {6, 3}}),
        with(&Routed::d_scores, B{BF, {6, 8}}), with(&Routed::d_scores, B{F, {6, 10}}),
        with(&Routed::d_logits, B{F, {5, 10}}), with(&Routed::dz, B{F, {6, 32}}), with(&Routed::dz, B{BF, {5, 32}}),
        with(&Routed::dx, B{F, {6, 32}}), with(&Routed::d_kernel, B{BF, {32, 8}}), with(&Routed::d_bias, B{F, {8}})})
    r.call(false);
  for (int64_t scored : {int64_t{0}, int64_t{11}, (int64_t{1} << 32) + 8}) {
    Routed r;
    r.scored = scored;
    r.call(false);
  }

  for (const Quantize& q : {Quantize{}, with(&Quantize::filled, NONE), with(&Quantize::x, B{F, {8, 100}})})
    q.call(true);
  {
    Quantize q = with(&Quantize::index, NONE);
    q.rows = 8;
    q.call(true);
    q.rows = 9;  // past x
    q.call(false);
    q = Quantize{};
    q.rows = 13;  // past the index
    q.call(false);
    for (int64_t div : {int64_t{0}, (int64_t{1} << 32) + 2}) {
      q = Quantize{};
      q.div = div;
      q.call(false);
    }
  }
  for (const Quantize& q :
       {with(&Quantize::x, B{I, {8, 100}}), with(&Quantize::x, B{BF, {800}}), with(&Quantize::x, B{BF, {8, 130}}),
        with(&Quantize::index, B{F, {12}}), with(&Quantize::filled, B{F, {1}}),
        with(&Quantize::values, B{U, {1, 16, 64}}), with(&Quantize::scales, B{F, {15}}),
        with(&Quantize::scales, B{BF, {16}})})
    q.call(false);

  for (const Glu& g : {Glu{}, with(&Glu::filled, NONE), with(&Glu::weights, B{F, {5}}, with(&Glu::projected, B{F, {5, 68, 2}}))})
    g.call(true);
  for (const Glu& g :
       {with(&Glu::weights, B{F, {5}}), with(&Glu::weights, B{BF, {4}}), with(&Glu::projected, B{BF, {5, 68, 1}}),
        with(&Glu::projected, B{BF, {5, 136}}), with(&Glu::filled, B{F, {1}}), with(&Glu::values, B{U, {1, 7, 64}}),
        with(&Glu::scales, B{F, {5}})})
    g.call(false);

  for (const Columns& c : {Columns{}, with(&Columns::w, B{F, {3, 100, 12}})}) c.call(true);
  for (const Columns& c : {with(&Columns::w, B{I, {3, 100, 12}}), with(&Columns::w, B{BF, {3, 1200}}),
                           with(&Columns::values, B{U, {3, 1, 12, 64}}), with(&Columns::scales, B{F, {3, 11}}),
                           with(&Columns::scales, B{BF, {3, 12}})})
    c.call(false);

  for (const Rows& r : {Rows{}, with(&Rows::bias, NONE), with(&Rows::bias, B{F, {3, 12}}, with(&Rows::y, B{F, {25, 12}}))})
    r.call(true);
  for (const Rows& r :
       {with(&Rows::as, B{F, {19}}), with(&Rows::as, B{BF, {20}}), with(&Rows::bs, B{F, {2, 12}}),
        with(&Rows::bias, B{F, {3, 12}}), with(&Rows::bias, B{BF, {2, 12}}), with(&Rows::y, B{BF, {25, 16}}),
        with(&Rows::y, B{I, {25, 12}}), with(&Rows::b, B{U, {3, 2, 12, 64}}), with(&Rows::a, B{F, {4, 20, 64}}),
        with(&Rows::a, B{U, {4, 1280}})})
    r.call(false);
  return 0;
}
