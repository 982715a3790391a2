// C entries of the dense layer and layer norm (include/mace/operators.h): argument checks on
// the host, then the launches of dense.cu and layer_norm.cu.  Nothing is launched by a call
// that returns -1 for its arguments.
#include "mace/operators.h"
#include "operators.hpp"
#include <cstdint>

namespace lapis {
void set_c_api_error(const std::string &message);
}
namespace {
using namespace mace::op;
using lapis::Error;

// Rows become 32-bit tile coordinates, and a row's byte length a 32-bit offset.
constexpr long long kMostRows = 2147483647, kMostWidth = 1ll << 28, kMostLd = 1ll << 32;

template <class R, class F> R entry(R failed, F &&body) {
  try {
    lapis::set_c_api_error("");
    return body();
  } catch (const std::exception &e) {
    try {
      lapis::set_c_api_error(e.what());
    } catch (...) {
    }
  } catch (...) {
  }
  return failed;
}

void check_common(int type, int activation, long long rows) {
  if (type < F32 || type > F16)
    throw Error("Invalid element type");
  if (activation < None || activation > Relu)
    throw Error("Invalid activation");
  if (rows < 0 || rows > kMostRows)
    throw Error("Invalid row count");
}
void check_width(long long width) {
  if (width < 1 || width > kMostWidth)
    throw Error("Invalid row length");
}

// A [rows][cols] array of the caller.
struct Array {
  const void *p;
  long long rows, cols, ld;
  int size; // bytes of an element
  uintptr_t begin() const { return reinterpret_cast<uintptr_t>(p); }
  uintptr_t end() const { return begin() + uintptr_t((rows - 1) * ld + cols) * uintptr_t(size); }
};
void check_array(const Array &a, const char *name) {
  if (!a.rows)
    return;
  if (!a.p)
    throw Error(std::string("Null array: ") + name);
  if (a.begin() % unsigned(a.size))
    throw Error(std::string("Misaligned array: ") + name);
  if (a.ld < a.cols || a.ld > kMostLd)
    throw Error(std::string("Invalid row distance: ") + name);
  if (a.rows > (1ll << 60) / a.ld)
    throw Error(std::string("Array too large: ") + name);
}
// Whether two arrays share a byte.  Column blocks of one buffer (same row distance) do not.
bool overlap(const Array &a, const Array &b) {
  if (!a.p || !b.p || !a.rows || !b.rows || a.end() <= b.begin() || b.end() <= a.begin())
    return false;
  uintptr_t lda = uintptr_t(a.ld) * a.size, ldb = uintptr_t(b.ld) * b.size;
  if (lda != ldb)
    return true;
  const Array &lo = a.begin() <= b.begin() ? a : b, &hi = a.begin() <= b.begin() ? b : a;
  uintptr_t off = (hi.begin() - lo.begin()) % lda;
  return off < uintptr_t(lo.cols) * lo.size || off + uintptr_t(hi.cols) * hi.size > lda;
}
bool same(const Array &a, const Array &b) { return a.p == b.p && (a.ld == b.ld || a.rows <= 1); }
void check_apart(const Array &out, std::initializer_list<Array> others) {
  for (const Array &o : others)
    if (overlap(out, o))
      throw Error("An output overlaps another array");
}
Array bytes(const void *p, long long n) { return {n > 0 ? p : nullptr, 1, n, n, 1}; }

void check_workspace(const void *p, long long have, long long need) {
  if (have < need || (need && !p))
    throw Error("Workspace too small: " + std::to_string(need) + " bytes are needed");
  if (need && reinterpret_cast<uintptr_t>(p) % 16)
    throw Error("Misaligned workspace");
}
} // namespace

extern "C" {
long long mace_dense_workspace(int type, long long rows, long long inputs, long long outputs, const void *x,
                               long long ldx, const void *weight, long long ldw) {
  return entry(-1ll, [&] {
    check_common(type, None, rows);
    check_width(inputs);
    check_width(outputs);
    int b = bytes_of(type);
    check_array({x, rows, inputs, ldx, b}, "x");
    check_array({weight, rows ? outputs : 0, inputs, ldw, b}, "weight");
    return rows ? dense_workspace({type, rows, inputs, outputs, x, ldx, weight, ldw}) : 0ll;
  });
}

int mace_dense(int type, long long rows, long long inputs, long long outputs, const void *x, long long ldx,
               const void *weight, long long ldw, const void *bias, int activation, const void *residual,
               long long ldr, void *y, long long ldy, void *z, long long ldz, void *workspace,
               long long workspace_bytes, void *stream) {
  return entry(-1, [&] {
    check_common(type, activation, rows);
    check_width(inputs);
    check_width(outputs);
    if (!rows)
      return 0;
    int b = bytes_of(type);
    Array ax{x, rows, inputs, ldx, b}, aw{weight, outputs, inputs, ldw, b},
        ab{bias, bias ? 1 : 0, outputs, outputs, b}, ar{residual, residual ? rows : 0, outputs, ldr, b},
        ay{y, rows, outputs, ldy, b}, az{z, z ? rows : 0, outputs, ldz, b};
    check_array(ax, "x");
    check_array(aw, "weight");
    check_array(ab, "bias");
    check_array(ar, "residual");
    check_array(ay, "y");
    check_array(az, "z");
    Dense d{type, rows, inputs, outputs, x, ldx, weight, ldw, bias, activation, residual, ldr, y, ldy, z, ldz};
    long long need = dense_workspace(d);
    check_workspace(workspace, workspace_bytes, need);
    Array ws = bytes(workspace, need);
    check_apart(ay, {ax, aw, ab, az, ws});
    if (!same(ay, ar))
      check_apart(ay, {ar});
    check_apart(az, {ax, aw, ab, ar, ws});
    check_apart(ws, {ax, aw, ab, ar});
    dense(d, workspace, static_cast<cudaStream_t>(stream));
    return 0;
  });
}

long long mace_dense_backward_workspace(int type, long long rows, long long inputs, long long outputs,
                                        const void *dy, long long lddy, const void *x, long long ldx,
                                        const void *weight, long long ldw, int activation) {
  return entry(-1ll, [&] {
    check_common(type, activation, rows);
    check_width(inputs);
    check_width(outputs);
    if (!rows)
      return 0ll;
    DenseBackward d{type, rows, inputs, outputs, dy, lddy, x, ldx, weight, ldw, activation};
    return dense_backward_workspace(d);
  });
}

int mace_dense_backward(int type, long long rows, long long inputs, long long outputs, const void *dy,
                        long long lddy, const void *x, long long ldx, const void *weight, long long ldw,
                        int activation, const void *z, long long ldz, void *dx, long long lddx, void *dweight,
                        long long lddw, void *dbias, void *workspace, long long workspace_bytes, void *stream) {
  return entry(-1, [&] {
    check_common(type, activation, rows);
    check_width(inputs);
    check_width(outputs);
    int b = bytes_of(type);
    Array ady{dy, rows, outputs, lddy, b}, ax{x, dweight ? rows : 0, inputs, ldx, b},
        aw{weight, dx && rows ? outputs : 0, inputs, ldw, b},
        az{z, activation != None ? rows : 0, outputs, ldz, b}, adx{dx, dx ? rows : 0, inputs, lddx, b},
        adw{dweight, dweight ? outputs : 0, inputs, lddw, b}, adb{dbias, dbias ? 1 : 0, outputs, outputs, b};
    check_array(ady, "dy");
    check_array(ax, "x");
    check_array(aw, "weight");
    check_array(az, "z");
    check_array(adx, "dx");
    check_array(adw, "dweight");
    check_array(adb, "dbias");
    DenseBackward d{type, rows,    inputs, outputs, dy,   lddy,    x,    ldx,  weight,
                    ldw,  activation, z,   ldz,     dx, lddx, dweight, lddw, dbias};
    long long need = rows ? dense_backward_workspace(d) : 0;
    check_workspace(workspace, workspace_bytes, need);
    Array ws = bytes(workspace, need);
    check_apart(adx, {ady, ax, aw, az, adw, adb, ws});
    check_apart(adw, {ady, ax, aw, az, adb, ws});
    check_apart(adb, {ady, ax, aw, az, ws});
    check_apart(ws, {ady, ax, aw, az});
    dense_backward(d, workspace, static_cast<cudaStream_t>(stream));
    return 0;
  });
}

int mace_layer_norm(int type, long long rows, long long width, const void *x, long long ldx, const void *gamma,
                    const void *beta, float eps, int activation, void *y, long long ldy, float *mean, float *rstd,
                    void *stream) {
  return entry(-1, [&] {
    check_common(type, activation, rows);
    check_width(width);
    if (!(eps >= 0.f))
      throw Error("Invalid eps");
    if (!mean != !rstd)
      throw Error("mean and rstd go together");
    if (!rows)
      return 0;
    int b = bytes_of(type);
    Array ax{x, rows, width, ldx, b}, ag{gamma, gamma ? 1 : 0, width, width, b},
        ab{beta, beta ? 1 : 0, width, width, b}, ay{y, rows, width, ldy, b}, am{mean, mean ? 1 : 0, rows, rows, 4},
        as{rstd, rstd ? 1 : 0, rows, rows, 4};
    check_array(ax, "x");
    check_array(ag, "gamma");
    check_array(ab, "beta");
    check_array(ay, "y");
    check_array(am, "mean");
    check_array(as, "rstd");
    if (!same(ay, ax))
      check_apart(ay, {ax});
    check_apart(ay, {ag, ab, am, as});
    check_apart(am, {ax, ag, ab, as});
    check_apart(as, {ax, ag, ab});
    layer_norm({type, rows, width, x, ldx, gamma, beta, eps, activation, y, ldy, mean, rstd},
               static_cast<cudaStream_t>(stream));
    return 0;
  });
}

long long mace_layer_norm_backward_workspace(int type, long long rows, long long width) {
  return entry(-1ll, [&] {
    check_common(type, None, rows);
    check_width(width);
    return rows ? layer_norm_backward_workspace(type, rows, width) : 0ll;
  });
}

int mace_layer_norm_backward(int type, long long rows, long long width, const void *dy, long long lddy,
                             const void *x, long long ldx, const float *mean, const float *rstd, const void *gamma,
                             const void *beta, int activation, void *dx, long long lddx, void *dgamma, void *dbeta,
                             void *workspace, long long workspace_bytes, void *stream) {
  return entry(-1, [&] {
    check_common(type, activation, rows);
    check_width(width);
    int b = bytes_of(type), stats = rows ? 1 : 0;
    Array ady{dy, rows, width, lddy, b}, ax{x, rows, width, ldx, b}, am{mean, stats, rows, rows, 4},
        as{rstd, stats, rows, rows, 4}, ag{gamma, gamma ? 1 : 0, width, width, b},
        ab{beta, beta ? 1 : 0, width, width, b}, adx{dx, dx ? rows : 0, width, lddx, b},
        adg{dgamma, dgamma ? 1 : 0, width, width, b}, adb{dbeta, dbeta ? 1 : 0, width, width, b};
    check_array(ady, "dy");
    check_array(ax, "x");
    check_array(am, "mean");
    check_array(as, "rstd");
    check_array(ag, "gamma");
    check_array(ab, "beta");
    check_array(adx, "dx");
    check_array(adg, "dgamma");
    check_array(adb, "dbeta");
    long long need = rows ? layer_norm_backward_workspace(type, rows, width) : 0;
    if (!dgamma && !dbeta)
      need = 0;
    check_workspace(workspace, workspace_bytes, need);
    Array ws = bytes(workspace, need);
    if (!same(adx, ady))
      check_apart(adx, {ady});
    check_apart(adx, {ax, am, as, ag, ab, adg, adb, ws});
    check_apart(adg, {ady, ax, am, as, ag, ab, adb, ws});
    check_apart(adb, {ady, ax, am, as, ag, ab, ws});
    check_apart(ws, {ady, ax, am, as, ag, ab});
    layer_norm_backward({type, rows, width, dy, lddy, x, ldx, mean, rstd, gamma, beta, activation, dx, lddx, dgamma,
                         dbeta},
                        workspace, static_cast<cudaStream_t>(stream));
    return 0;
  });
}
}
