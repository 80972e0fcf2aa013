// Calls the XLA FFI handlers of the dense products and of the gradients' clipping on made-up
// buffers, the library's entry points replaced by ones that say they were reached. Prints a line a
// case: its handler, whether it is meant to be taken, whether the library was called, and whether
// a refusal's code is that of an invalid argument.
#include "../bux_amd/xla/xla_ffi.cc"

#include <cstdio>

static int calls = 0;
extern "C" {
const char* bux_last_error() { return ""; }
int bux_dense_rows(const uint16_t*, const uint16_t*, int, int64_t, int64_t, int64_t, const uint16_t*,
                   const bux_ffn*, const uint16_t*, uint16_t*, uint8_t*, uint16_t*, void*, size_t,
                   void*) { return ++calls, 0; }
int bux_dense_rows_f32(const float*, const float*, int, int64_t, int64_t, int64_t, const float*,
                       const bux_ffn*, const float*, float*, float*, void*, size_t,
                       void*) { return ++calls, 0; }
int bux_dense_units_backward(const uint16_t*, const uint16_t*, int64_t, int64_t, int64_t,
                             const uint16_t*, const uint8_t*, const bux_ffn*, uint16_t*, uint8_t*,
                             void*, size_t, void*) { return ++calls, 0; }
int bux_dense_units_backward_f32(const float*, const float*, int64_t, int64_t, int64_t, const float*,
                                 const bux_ffn*, float*, void*, size_t, void*) { return ++calls, 0; }
int bux_dense_contract(const uint16_t*, const uint16_t*, int64_t, int64_t, int64_t, uint16_t*, void*,
                       size_t, void*) { return ++calls, 0; }
int bux_dense_contract_f32(const float*, const float*, int64_t, int64_t, int64_t, float*, void*,
                           size_t, void*) { return ++calls, 0; }
int bux_dense_slope(const uint16_t*, const uint8_t*, const uint16_t*, const bux_ffn*, int64_t, int64_t, uint16_t*,
                    uint16_t*, void*, size_t, void*) { return ++calls, 0; }
int bux_dense_slope_f32(const float*, const float*, const bux_ffn*, int64_t, int64_t, float*, float*,
                        void*, size_t, void*) { return ++calls, 0; }
int bux_clip(const bux_gradient* g, int32_t count, float, float*, void*, size_t, void*) {
  for (int32_t i = 0; i < count; ++i)
    if (g[i].n < 0 || !g[i].g) return 1;
  return ++calls, 0;
}
}

using ffi::DataType;
constexpr DataType BF = DataType::BF16, F = DataType::F32, U = DataType::U8;
static char memory[64];
static In buffer(DataType t, std::vector<int64_t> dims) { return In(t, std::move(dims), memory); }
static Out result(DataType t, std::vector<int64_t> dims) { return Out(buffer(t, std::move(dims))); }

static void line(const char* what, bool taken, const ffi::Error& e) {
  const bool right = calls ? e.success() : e.errc() == ffi::ErrorCode::kInvalidArgument;
  std::printf("%s %d %d %d\n", what, taken ? 1 : 0, calls, right ? 1 : 0);
  calls = 0;
}

struct Rows {
  DataType t = BF;
  std::vector<int64_t> x{6, 32}, w{32, 20}, bias{20}, residual{6, 20}, product{6, 20}, low{0}, out{6, 20};
  DataType wt = BF;
  int64_t transposed = 0, activation = 0, gated = 0;
  void call(bool taken) const {
    line("rows", taken,
         DenseRows(nullptr, buffer(t, x), buffer(wt, w), buffer(t, bias), buffer(t, residual),
                   transposed, activation, gated, 0, 0.0f, 0, 0.0f, 0.0f, result(t, product),
                   result(U, low),
                   result(t, out), result(U, {64})));
  }
};
template <typename S, typename V>
static S with(V S::*field, V value, S s = S{}) {
  s.*field = value;
  return s;
}
using Dims = std::vector<int64_t>;

int main() {
  Rows().call(true);
  Rows f;
  f.t = f.wt = F;
  f.call(true);
  with(&Rows::residual, Dims{0}).call(true);
  with(&Rows::bias, Dims{0}).call(true);
  with(&Rows::low, Dims{6, 20}).call(true);
  with(&Rows::low, Dims{6, 19}).call(false);
  with(&Rows::activation, int64_t{-1}).call(true);
  Rows g;
  g.gated = 1, g.residual = {0}, g.out = {6, 10};
  g.call(true);
  Rows tr;
  tr.transposed = 1, tr.w = {20, 32};
  tr.call(true);
  with(&Rows::w, Dims{20, 32}).call(false);
  with(&Rows::wt, F).call(false);
  with(&Rows::bias, Dims{19}).call(false);
  with(&Rows::residual, Dims{6, 19}).call(false);
  with(&Rows::product, Dims{5, 20}).call(false);
  with(&Rows::out, Dims{6, 21}).call(false);
  with(&Rows::x, Dims{192}).call(false);
  with(&Rows::gated, int64_t{1}).call(false);  // out of half the columns

  auto units = [](bool taken, DataType t, Dims dy, Dims down, Dims product, Dims dp, int64_t gated,
                  Dims low = {0}, Dims dp_low = {0}) {
    line("units backward", taken,
         DenseUnitsBackward(nullptr, buffer(t, dy), buffer(t, down), buffer(t, product), buffer(U, low), 0,
                            gated, 0,
                            0.0f, 0, 0.0f, 0.0f, result(t, dp), result(U, dp_low),
                            result(U, {64})));
  };
  units(true, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1);
  units(true, F, {6, 32}, {10, 32}, {6, 10}, {6, 10}, 0);
  units(true, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1, {6, 10, 2});
  units(false, F, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1, {6, 10, 2});
  units(false, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1, {6, 10});
  units(true, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1, {0}, {6, 10, 2});
  units(false, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10, 2}, 1, {0}, {5, 10, 2});
  units(false, BF, {6, 32}, {10, 31}, {6, 10, 2}, {6, 10, 2}, 1);
  units(false, BF, {6, 32}, {10, 32}, {6, 10}, {6, 10, 2}, 1);
  units(false, BF, {6, 32}, {10, 32}, {6, 10, 2}, {6, 10}, 1);

  auto contract = [](bool taken, DataType t, DataType dyt, Dims x, Dims dy, Dims dw) {
    line("contract", taken, DenseContract(nullptr, buffer(t, x), buffer(dyt, dy), result(t, dw),
                                          result(U, {64})));
  };
  contract(true, BF, BF, {6, 32}, {6, 10}, {32, 10});
  contract(true, F, F, {6, 32}, {6, 10}, {32, 10});
  contract(false, BF, F, {6, 32}, {6, 10}, {32, 10});
  contract(false, BF, BF, {6, 32}, {5, 10}, {32, 10});
  contract(false, BF, BF, {6, 32}, {6, 10}, {32, 11});

  auto slope = [](bool taken, DataType t, Dims product, int64_t activation, Dims dz, Dims sums,
                  Dims low = {0}) {
    line("slope", taken,
         DenseSlope(nullptr, buffer(t, {6, 20}), buffer(U, low), buffer(t, product), activation, 0, 0, 0.0f, 0, 0.0f,
                    0.0f, result(t, dz), result(t, sums), result(U, {64})));
  };
  slope(true, BF, {6, 20}, 0, {6, 20}, {20});
  slope(true, F, {0}, -1, {0}, {20});
  slope(true, BF, {0}, -1, {0}, {20}, {6, 20});
  slope(false, BF, {0}, -1, {0}, {20}, {6, 21});
  slope(false, F, {0}, -1, {0}, {20}, {6, 20});
  slope(false, BF, {6, 19}, 0, {6, 20}, {20});
  slope(false, BF, {6, 20}, 0, {6, 21}, {20});
  slope(false, BF, {6, 20}, 0, {6, 20}, {6});

  auto clip = [](bool taken, std::vector<In> grads, std::vector<In> rets) {
    line("clip", taken, Clip(nullptr, ffi::RemainingArgs(grads), 1.0f, ffi::RemainingRets(rets)));
  };
  const In a = buffer(BF, {4, 5}), b = buffer(F, {7}), norm = buffer(F, {1}), ws = buffer(U, {64});
  clip(true, {a, b}, {a, b, norm, ws});
  clip(true, {a, b}, {norm, ws});
  clip(false, {}, {norm, ws});
  clip(false, {a, b}, {a, norm, ws});
  clip(false, {a, b}, {b, a, norm, ws});
  clip(false, {a, ws}, {a, ws, norm, ws});
  clip(false, {a, b}, {a, b, ws, ws});
  clip(false, {a}, {buffer(BF, {4, 6}), norm, ws});
  return 0;
}
