// C ABI of the linear-layer operators (include/qrb200_linear.h): argument
// validation, the workspace of each call and the kernel sequence it enqueues.
#include "qrb_linear.cuh"

namespace qrb {
namespace lin {
namespace {

constexpr int64_t kMaxDim = 1LL << 30;  // tensor-map coordinates are 32-bit

bool dtype_ok(int d) { return d == QRBL_F32 || d == QRBL_F16 || d == QRBL_BF16; }
bool act_ok(int a) { return a >= QRBL_ACT_NONE && a <= QRBL_ACT_SILU; }
// A matrix argument with `cols` columns: row stride, and the element alignment
// that every access relies on.
bool mat_ok(const void* p, int64_t ld, int64_t rows, int64_t cols, int elem) {
  return p != nullptr && (ld >= cols || rows <= 1) && ld >= 0 && ld <= (1LL << 40) &&
         reinterpret_cast<uintptr_t>(p) % elem == 0;
}
bool vec_ok(const void* p, int elem) {
  return p == nullptr || reinterpret_cast<uintptr_t>(p) % elem == 0;
}
size_t up256(size_t b) { return (b + 255) / 256 * 256; }
int64_t up8(int64_t v) { return (v + 7) / 8 * 8; }

// Workspace, handed out front to back (base null: only counted).
struct Carve {
  uint8_t* base;
  size_t used = 0;
  void* take(size_t bytes) {
    void* p = base == nullptr ? nullptr : base + used;
    used += up256(bytes);
    return p;
  }
};

// How one operand reaches the product: read in place, or staged into the
// workspace (FP32 planes; rows or base not 16-byte aligned; packed).
struct Source {
  const void* p = nullptr;
  int64_t ld = 0;
  const int8_t* codes = nullptr;
  const int8_t* exps = nullptr;
  int64_t rows = 0, cols = 0;
};
bool in_place(int dtype, const Source& s) {
  return dtype != QRBL_F32 && s.codes == nullptr && aligned16(s.p) &&
         (s.rows <= 1 || s.ld % 8 == 0) && s.ld < (1LL << 38);
}
Operand staged_operand(int dtype, int64_t rows, int64_t cols, Carve* c) {
  Operand o;
  o.rows = rows;
  o.cols = cols;
  o.ld = up8(cols);
  o.plane = o.ld * rows;
  o.p = c->take((size_t)o.plane * 2 * (dtype == QRBL_F32 ? 3 : 1));
  return o;
}
// (the operand; *stage is set where launch_stage has to fill it first)
Operand operand_of(int dtype, const Source& s, Carve* c, bool* stage) {
  *stage = !in_place(dtype, s);
  if (*stage) return staged_operand(dtype, s.rows, s.cols, c);
  Operand o;
  o.p = s.p;
  o.rows = s.rows;
  o.cols = s.cols;
  o.ld = s.rows <= 1 ? up8(s.cols) : s.ld;  // one row: any legal stride
  return o;
}
void add_stage(Prepare* p, const Source& s, const Operand& o) {
  StageArgs& a = p->stage[p->stages++];
  a.src = s.p;
  a.lds = s.ld;
  a.codes = s.codes;
  a.exps = s.exps;
  a.rows = s.rows;
  a.cols = s.cols;
  a.dst = const_cast<void*>(o.p);
  a.ldd = o.ld;
  a.plane = o.plane;
}

// ---------------------------------------------------------------------------
// forward
// ---------------------------------------------------------------------------
int check(const qrbl_linear_args& a) {
  if (!dtype_ok(a.dtype) || !act_ok(a.activation) || a.m < 0 || a.n < 0 || a.k < 0)
    return QRB_ERR_INVALID_ARG;
  if ((a.z_codes == nullptr) != (a.z_exponents == nullptr)) return QRB_ERR_INVALID_ARG;
  if (a.m == 0 || a.n == 0) return QRB_OK;
  const int es = elem_size(a.dtype);
  if (a.k > 0 && (!mat_ok(a.x, a.ldx, a.m, a.k, es) || !mat_ok(a.w, a.ldw, a.n, a.k, es)))
    return QRB_ERR_INVALID_ARG;
  if (!mat_ok(a.y, a.ldy, a.m, a.n, es)) return QRB_ERR_INVALID_ARG;
  if (a.residual != nullptr && !mat_ok(a.residual, a.ldr, a.m, a.n, es))
    return QRB_ERR_INVALID_ARG;
  if (a.z != nullptr && !mat_ok(a.z, a.ldz, a.m, a.n, es)) return QRB_ERR_INVALID_ARG;
  if (!vec_ok(a.bias, es)) return QRB_ERR_INVALID_ARG;
  if (a.m > kMaxDim || a.n > kMaxDim || a.k > kMaxDim) return QRB_ERR_UNSUPPORTED;
  return QRB_OK;
}

struct Forward {
  bool rows = false;  // few rows: their own kernel
  Source xs, ws;
  Operand x, w;
  bool stage_x = false, stage_w = false;
  ProductSize size;
  ProductPlan plan;
  float* part = nullptr;
  float* chains = nullptr;
};
Forward plan_forward(const qrbl_linear_args& a, Carve* c) {
  Forward f;
  f.rows = takes_rows(a.dtype, a.m, a.n, a.k, a.z_codes != nullptr);
  if (f.rows) {
    f.x.p = a.x; f.x.ld = a.ldx;
    f.w.p = a.w; f.w.ld = a.ldw;
    return f;
  }
  f.xs.p = a.x; f.xs.ld = a.ldx; f.xs.rows = a.m; f.xs.cols = a.k;
  f.ws.p = a.w; f.ws.ld = a.ldw; f.ws.rows = a.n; f.ws.cols = a.k;
  f.x = operand_of(a.dtype, f.xs, c, &f.stage_x);
  f.w = operand_of(a.dtype, f.ws, c, &f.stage_w);
  f.size.m = a.m; f.size.n = a.n; f.size.k = a.k;
  f.size.epilogue = (a.activation > QRBL_ACT_RELU ? 1 : 0) |
                    (a.z != nullptr || a.z_codes != nullptr ? 2 : 0) |
                    (a.residual != nullptr ? 4 : 0) | (a.z_codes != nullptr ? 8 : 0);
  f.plan = plan_products(a.dtype, &f.size, 1);
  f.part = reinterpret_cast<float*>(c->take(f.plan.part_bytes[0]));
  if (f.plan.chain_bytes > 0) f.chains = reinterpret_cast<float*>(c->take(f.plan.chain_bytes));
  return f;
}

int forward(const qrbl_linear_args& a, void* workspace, size_t bytes, cudaStream_t s) {
  int rc = check(a);
  if (rc != QRB_OK || a.m == 0 || a.n == 0) return rc;
  if (take_injected_failure_any()) return QRB_ERR_INJECTED;
  Epilogue e;
  const int es = elem_size(a.dtype);
  e.out = a.y; e.ldo = a.ldy;
  e.bias = a.bias;
  e.residual = a.residual; e.ldr = a.ldr;
  e.z = a.z; e.ldz = a.ldz;
  e.z_codes = a.z_codes; e.z_exps = a.z_exponents;
  e.act = a.activation;
  auto rows16 = [&](const void* p, int64_t ld) {
    return p == nullptr || (aligned16(p) && (a.m <= 1 || (ld * es) % 16 == 0));
  };
  e.vec = rows16(a.y, a.ldy) && rows16(a.residual, a.ldr) && rows16(a.z, a.ldz);
  if (a.k == 0) return launch_join(a.dtype, nullptr, 0, 0, 0, a.m, a.n, e, false, s);
  Carve c{reinterpret_cast<uint8_t*>(workspace)};
  const Forward f = plan_forward(a, &c);
  if (!f.rows && !f.plan.ok) return QRB_ERR_UNSUPPORTED;
  if (c.used > 0 && (workspace == nullptr || bytes < c.used)) return QRB_ERR_WORKSPACE;
  if (c.used > 0 && !aligned16(workspace)) return QRB_ERR_INVALID_ARG;
  if (f.rows) return launch_rows(a.dtype, f.x, f.w, a.m, a.n, a.k, e, s);
  Prepare before;
  if (f.stage_x) add_stage(&before, f.xs, f.x);
  if (f.stage_w) add_stage(&before, f.ws, f.w);
  if (before.stages > 0 && (rc = launch_prepare(a.dtype, before, s)) != QRB_OK) return rc;
  Product p;
  p.kind = kForward;
  p.size = f.size;
  p.a = f.x; p.b = f.w;
  p.part = f.part;
  p.e = e;
  return launch_products(a.dtype, &p, 1, f.plan, f.chains, nullptr, before.stages > 0, s);
}

// ---------------------------------------------------------------------------
// backward
// ---------------------------------------------------------------------------
int check(const qrbl_linear_backward_args& a) {
  if (!dtype_ok(a.dtype) || !act_ok(a.activation) || a.m < 0 || a.n < 0 || a.k < 0)
    return QRB_ERR_INVALID_ARG;
  if ((a.x_codes == nullptr) != (a.x_exponents == nullptr) ||
      (a.z_codes == nullptr) != (a.z_exponents == nullptr) ||
      (a.x != nullptr && a.x_codes != nullptr) || (a.z != nullptr && a.z_codes != nullptr))
    return QRB_ERR_INVALID_ARG;
  const bool dx = a.dx != nullptr && a.m > 0 && a.k > 0;
  const bool dw = a.dw != nullptr && a.n > 0 && a.k > 0;
  const bool db = a.dbias != nullptr && a.n > 0;
  if (!dx && !dw && !db) return QRB_OK;
  const int es = elem_size(a.dtype);
  if (dx && !mat_ok(a.dx, a.lddx, a.m, a.k, es)) return QRB_ERR_INVALID_ARG;
  if (dw && !mat_ok(a.dw, a.lddw, a.n, a.k, es)) return QRB_ERR_INVALID_ARG;
  if (!vec_ok(a.dbias, es)) return QRB_ERR_INVALID_ARG;
  if (a.m > 0 && a.n > 0) {
    if (!mat_ok(a.dy, a.lddy, a.m, a.n, es)) return QRB_ERR_INVALID_ARG;
    if (dx && !mat_ok(a.w, a.ldw, a.n, a.k, es)) return QRB_ERR_INVALID_ARG;
    if (dw && a.x_codes == nullptr && !mat_ok(a.x, a.ldx, a.m, a.k, es))
      return QRB_ERR_INVALID_ARG;
    if (a.activation != QRBL_ACT_NONE && a.z_codes == nullptr &&
        !mat_ok(a.z, a.ldz, a.m, a.n, es))
      return QRB_ERR_INVALID_ARG;
    if (a.activation == QRBL_ACT_RELU && a.z_codes != nullptr) return QRB_ERR_INVALID_ARG;
  }
  if (a.m > kMaxDim || a.n > kMaxDim || a.k > kMaxDim) return QRB_ERR_UNSUPPORTED;
  return QRB_OK;
}

struct Backward {
  bool dx = false, dw = false, db = false;
  bool dz_kernel = false;  // dz (or its sums) are computed first
  bool dz_stored = false;
  bool stage_x = false, stage_w = false;
  Source xs, ws;
  Operand dz, x, w;
  ProductSize size[2];  // of the products there are, dW before dx
  int products = 0;
  ProductPlan plan;
  float* part[2] = {nullptr, nullptr};
  float* chains = nullptr;
  float* colsum = nullptr;
  int64_t colsum_blocks = 0;
};
Backward plan_backward(const qrbl_linear_backward_args& a, Carve* c) {
  Backward b;
  b.dx = a.dx != nullptr && a.m > 0 && a.k > 0;
  b.dw = a.dw != nullptr && a.n > 0 && a.k > 0;
  b.db = a.dbias != nullptr && a.n > 0;
  if (a.m == 0 || a.n == 0) return b;
  const bool products = b.dx || b.dw;
  Source dys;
  dys.p = a.dy; dys.ld = a.lddy; dys.rows = a.m; dys.cols = a.n;
  b.dz_stored = products && (a.activation != QRBL_ACT_NONE || !in_place(a.dtype, dys));
  b.dz_kernel = b.dz_stored || b.db;
  if (b.dz_stored)
    b.dz = staged_operand(a.dtype, a.m, a.n, c);
  else if (products)
    b.dz = operand_of(a.dtype, dys, c, &b.dz_stored);  // in place
  if (b.dw) {
    b.xs.p = a.x; b.xs.ld = a.ldx; b.xs.rows = a.m; b.xs.cols = a.k;
    b.xs.codes = a.x_codes; b.xs.exps = a.x_exponents;
    b.x = operand_of(a.dtype, b.xs, c, &b.stage_x);
    ProductSize& z = b.size[b.products++];
    z.m = a.n; z.n = a.k; z.k = a.m;
  }
  if (b.dx) {
    b.ws.p = a.w; b.ws.ld = a.ldw; b.ws.rows = a.n; b.ws.cols = a.k;
    b.w = operand_of(a.dtype, b.ws, c, &b.stage_w);
    ProductSize& z = b.size[b.products++];
    z.m = a.m; z.n = a.k; z.k = a.n;
  }
  if (b.db) {
    const int rows = colsum_rows(a.m, a.n);
    b.colsum_blocks = (a.m + rows - 1) / rows;
    b.colsum = reinterpret_cast<float*>(c->take((size_t)b.colsum_blocks * a.n * sizeof(float)));
  }
  if (b.products > 0) {
    b.plan = plan_products(a.dtype, b.size, b.products);
    for (int i = 0; i < b.products; ++i)
      b.part[i] = reinterpret_cast<float*>(c->take(b.plan.part_bytes[i]));
    if (b.plan.chain_bytes > 0) b.chains = reinterpret_cast<float*>(c->take(b.plan.chain_bytes));
  }
  return b;
}

// (in one piece where it is one: a pitch ends at 2^31 bytes)
int zero_rows(void* p, int64_t ld, int64_t rows, int64_t cols, int es, cudaStream_t s) {
  const size_t row = (size_t)cols * es;
  const cudaError_t e = rows <= 1 || ld == cols
                            ? cudaMemsetAsync(p, 0, row * (size_t)rows, s)
                            : cudaMemset2DAsync(p, (size_t)ld * es, 0, row, (size_t)rows, s);
  return e == cudaSuccess ? QRB_OK : QRB_ERR_LAUNCH;
}

int backward(const qrbl_linear_backward_args& a, void* workspace, size_t bytes, cudaStream_t s) {
  int rc = check(a);
  if (rc != QRB_OK) return rc;
  if (take_injected_failure_any()) return QRB_ERR_INJECTED;
  const int es = elem_size(a.dtype);
  Carve c{reinterpret_cast<uint8_t*>(workspace)};
  const Backward b = plan_backward(a, &c);
  if (b.products > 0 && !b.plan.ok) return QRB_ERR_UNSUPPORTED;
  if (c.used > 0 && (workspace == nullptr || bytes < c.used)) return QRB_ERR_WORKSPACE;
  if (c.used > 0 && !aligned16(workspace)) return QRB_ERR_INVALID_ARG;
  if (a.m == 0 || a.n == 0) {  // sums over nothing
    if (b.dx && (rc = zero_rows(a.dx, a.lddx, a.m, a.k, es, s)) != QRB_OK) return rc;
    if (b.dw && (rc = zero_rows(a.dw, a.lddw, a.n, a.k, es, s)) != QRB_OK) return rc;
    if (b.db && (rc = zero_rows(a.dbias, a.n, 1, a.n, es, s)) != QRB_OK) return rc;
    return QRB_OK;
  }
  Prepare before;
  if (b.dz_kernel) {
    DzArgs& d = before.dz;
    before.has_dz = true;
    d.dy = a.dy; d.lddy = a.lddy;
    d.z = a.z; d.ldz = a.ldz;
    d.z_codes = a.z_codes; d.z_exps = a.z_exponents;
    d.act = a.activation;
    d.m = a.m; d.n = a.n;
    if (b.dz_stored) {
      d.dst = const_cast<void*>(b.dz.p);
      d.ldd = b.dz.ld;
      d.plane = b.dz.plane;
    }
    d.part = b.colsum;
  }
  if (b.stage_x) add_stage(&before, b.xs, b.x);
  if (b.stage_w) add_stage(&before, b.ws, b.w);
  const bool prepared = before.has_dz || before.stages > 0;
  if (prepared &&
      (rc = launch_prepare(a.dtype, before, s)) != QRB_OK)
    return rc;
  ColSum sum;
  sum.part = b.colsum;
  sum.blocks = b.colsum_blocks;
  sum.n = a.n;
  sum.out = a.dbias;
  sum.slices = colsum_slices(b.colsum_blocks, a.n);
  auto rows16 = [&](const void* p, int64_t ld, int64_t rows) {
    return aligned16(p) && (rows <= 1 || (ld * es) % 16 == 0);
  };
  Product p[2];
  int i = 0;
  if (b.dw) {
    p[i].kind = kGradW;
    p[i].a = b.dz; p[i].b = b.x;
    p[i].e.out = a.dw; p[i].e.ldo = a.lddw;
    p[i].e.vec = rows16(a.dw, a.lddw, a.n);
    ++i;
  }
  if (b.dx) {
    p[i].kind = kGradIn;
    p[i].a = b.dz; p[i].b = b.w;
    p[i].e.out = a.dx; p[i].e.ldo = a.lddx;
    p[i].e.vec = rows16(a.dx, a.lddx, a.m);
    ++i;
  }
  for (int j = 0; j < i; ++j) {
    p[j].size = b.size[j];
    p[j].part = b.part[j];
  }
  if (i > 0)
    return launch_products(a.dtype, p, i, b.plan, b.chains, b.db ? &sum : nullptr, prepared, s);
  return b.db ? launch_colsum(a.dtype, sum, s) : QRB_OK;
}

int check_packed(int dtype, const void* x, int64_t ld, int64_t rows, int64_t cols,
                 const int8_t* codes, const int8_t* exps) {
  if (!dtype_ok(dtype) || rows < 0 || cols < 0) return QRB_ERR_INVALID_ARG;
  if (rows == 0 || cols == 0) return QRB_OK;
  if (!mat_ok(x, ld, rows, cols, elem_size(dtype)) || codes == nullptr || exps == nullptr)
    return QRB_ERR_INVALID_ARG;
  if (rows > (1LL << 40) || cols > kMaxDim) return QRB_ERR_UNSUPPORTED;
  return QRB_OK;
}

}  // namespace
}  // namespace lin
}  // namespace qrb

extern "C" {

QRB_API size_t qrbl_linear_workspace_bytes(const qrbl_linear_args* a) {
  if (a == nullptr || qrb::lin::check(*a) != QRB_OK || a->m == 0 || a->n == 0 || a->k == 0)
    return 0;
  qrb::lin::Carve c{nullptr};
  (void)qrb::lin::plan_forward(*a, &c);
  return c.used;
}

QRB_API int qrbl_linear(const qrbl_linear_args* a, void* workspace, size_t workspace_bytes,
                        void* stream) {
  if (a == nullptr) return QRB_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return qrb::finish_call(qrb::lin::forward(*a, workspace, workspace_bytes, s), s);
}

QRB_API size_t qrbl_linear_backward_workspace_bytes(const qrbl_linear_backward_args* a) {
  if (a == nullptr || qrb::lin::check(*a) != QRB_OK) return 0;
  qrb::lin::Carve c{nullptr};
  (void)qrb::lin::plan_backward(*a, &c);
  return c.used;
}

QRB_API int qrbl_linear_backward(const qrbl_linear_backward_args* a, void* workspace,
                                 size_t workspace_bytes, void* stream) {
  if (a == nullptr) return QRB_ERR_INVALID_ARG;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return qrb::finish_call(qrb::lin::backward(*a, workspace, workspace_bytes, s), s);
}

QRB_API int qrbl_pack(int32_t dtype, const void* x, int64_t ld, int64_t rows, int64_t cols,
                      int8_t* codes, int8_t* exponents, void* stream) {
  int rc = qrb::lin::check_packed(dtype, x, ld, rows, cols, codes, exponents);
  if (rc != QRB_OK || rows == 0 || cols == 0) return rc;
  if (qrb::take_injected_failure_any()) return QRB_ERR_INJECTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return qrb::finish_call(qrb::lin::launch_pack(dtype, x, ld, rows, cols, codes, exponents, s), s);
}

QRB_API int qrbl_unpack(int32_t dtype, const int8_t* codes, const int8_t* exponents, int64_t rows,
                        int64_t cols, void* x, int64_t ld, void* stream) {
  int rc = qrb::lin::check_packed(dtype, x, ld, rows, cols, codes, exponents);
  if (rc != QRB_OK || rows == 0 || cols == 0) return rc;
  if (qrb::take_injected_failure_any()) return QRB_ERR_INJECTED;
  cudaStream_t s = static_cast<cudaStream_t>(stream);
  return qrb::finish_call(qrb::lin::launch_unpack(dtype, codes, exponents, rows, cols, x, ld, s),
                          s);
}

}  // extern "C"
