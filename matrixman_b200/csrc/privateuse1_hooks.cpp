// C++ PrivateUse1 plumbing for the `matrixman` device, built as a small torch
// extension (torch.utils.cpp_extension) in-tree.
//
// Replaces drivers/matrixman/native/autograd_privateuse1.cpp of the reference
// (lines 7-66), whose hooks and DeviceGuard hard-wired one device and a no-op
// default stream.  Here the guard reports the real CUDA device count, switches
// the current CUDA device, and maps the c10 default stream of each device onto
// the runtime stream of libmatrixman_b200 (queried / synchronised through the
// C ABI).  The library is resolved at run time with dlsym, so this extension
// links against neither CUDA nor libmatrixman_b200 directly.
#include <ATen/detail/PrivateUse1HooksInterface.h>
#include <c10/core/impl/DeviceGuardImplInterface.h>
#include <dlfcn.h>
#include <torch/extension.h>

#include <atomic>
#include <cstring>
#include <vector>

namespace {

using count_fn = int (*)(int*);
using dev_fn = int (*)(int);
using stream_fn = int (*)(int, void**);
using sync_fn = int (*)(void*, int64_t);
using query_fn = int (*)(void*, int*);
using fault_fn = int (*)(int, int**);
using kernel_error_fn = int (*)(int, int*, int);

template <class F>
F resolve(const char* name) {
  void* p = dlsym(RTLD_DEFAULT, name);
  TORCH_CHECK(p != nullptr, "matrixman hooks: libmatrixman_b200 symbol ", name,
              " not loaded (import matrixman_b200 first)");
  return reinterpret_cast<F>(p);
}

// The symbol, looked up once per use in the source: a lookup walks every loaded
// library (several microseconds), and autograd switches devices and asks for
// streams several times per operator.
#define MM_SYMBOL(F, name)                \
  ([]() -> F {                            \
    static const F f = resolve<F>(name);  \
    return f;                             \
  }())

thread_local int t_current_device = 0;

// Upper bound of every stream wait the guard makes (matrixman.config
// waitTimeoutMs, passed in at backend init; the config is locked from then on).
std::atomic<int64_t> g_wait_timeout_ms{600000};

int device_count() {
  int n = 0;
  if (MM_SYMBOL(count_fn, "mm_device_count")(&n) != 0) return 0;
  return n;
}

void* runtime_stream(int device) {
  void* s = nullptr;
  MM_SYMBOL(dev_fn, "mm_init")(device);
  MM_SYMBOL(stream_fn, "mm_runtime_stream")(device, &s);
  return s;
}

constexpr int MM_STATUS_TIMEOUT = 5;  // MM_ERR_TIMEOUT of the C ABI

// Bounded synchronisation of a device's runtime stream: raises with the C
// ABI's message when the wait gives up (MM_ERR_TIMEOUT) or fails.
void sync_runtime_stream(int device, const char* what) {
  const int rc = MM_SYMBOL(sync_fn, "mm_stream_sync")(runtime_stream(device), g_wait_timeout_ms.load());
  if (rc == 0) {
    int* fault = nullptr;
    if (MM_SYMBOL(fault_fn, "mm_fault_word")(device, &fault) != 0 || *(volatile int*)fault == 0) return;
    int code = 0;
    MM_SYMBOL(kernel_error_fn, "mm_kernel_error")(device, &code, 1);
    TORCH_CHECK(code == 0, "matrixman guard: ", what, " of device ", device,
                ": a tensor-core kernel stopped after a bounded wait (code ", code, ")");
    return;
  }
  char msg[512] = {0};
  using err_fn = int (*)(char*, size_t);
  if (void* p = dlsym(RTLD_DEFAULT, "mm_last_error")) reinterpret_cast<err_fn>(p)(msg, sizeof(msg));
  TORCH_CHECK(rc != MM_STATUS_TIMEOUT, "matrixman guard: ", what, " of device ", device,
              " did not finish within ", g_wait_timeout_ms.load(), " ms (waitTimeoutMs): ", msg);
  TORCH_CHECK(false, "matrixman guard: ", what, " of device ", device, " failed: ", msg);
}

using pin_alloc_fn = int (*)(size_t, void**);
using pin_free_fn = int (*)(void*);
using is_pinned_fn = int (*)(const void*, int*);

void free_pinned(void* p) {
  if (p) MM_SYMBOL(pin_free_fn, "mm_host_free_pinned")(p);
}

// Page-locked host memory for Tensor.pin_memory() on this backend, so that
// uploads from pinned buffers run as asynchronous copy-engine transfers.
class PinnedAllocator final : public c10::Allocator {
 public:
  c10::DataPtr allocate(size_t n) override {
    void* p = nullptr;
    if (n > 0) {
      TORCH_CHECK(MM_SYMBOL(pin_alloc_fn, "mm_host_alloc_pinned")(n, &p) == 0,
                  "matrixman: pinned host allocation of ", n, " bytes failed");
    }
    return {p, p, &free_pinned, c10::Device(c10::DeviceType::CPU)};
  }
  c10::DeleterFnPtr raw_deleter() const override { return &free_pinned; }
  void copy_data(void* dst, const void* src, std::size_t count) const override {
    std::memcpy(dst, src, count);
  }
};

PinnedAllocator g_pinned;

class MatrixManHooks final : public at::PrivateUse1HooksInterface {
 public:
  bool isBuilt() const override { return true; }
  bool isAvailable() const override { return device_count() > 0; }
  bool hasPrimaryContext(c10::DeviceIndex) const override { return true; }
  c10::Device getDeviceFromPtr(void*) const override {
    return c10::Device(c10::DeviceType::PrivateUse1, (c10::DeviceIndex)t_current_device);
  }
  bool isPinnedPtr(const void* data) const override {
    int pinned = 0;
    MM_SYMBOL(is_pinned_fn, "mm_host_is_pinned")(data, &pinned);
    return pinned != 0;
  }
  c10::Allocator* getPinnedMemoryAllocator() const override { return &g_pinned; }
};

class MatrixManGuardImpl final : public c10::impl::DeviceGuardImplInterface {
 public:
  c10::DeviceType type() const override { return c10::DeviceType::PrivateUse1; }

  c10::Device exchangeDevice(c10::Device d) const override {
    c10::Device old = getDevice();
    if (d.index() != old.index()) setDevice(d);
    return old;
  }

  c10::Device getDevice() const override {
    return c10::Device(c10::DeviceType::PrivateUse1, (c10::DeviceIndex)t_current_device);
  }

  void setDevice(c10::Device d) const override {
    TORCH_CHECK(d.type() == c10::DeviceType::PrivateUse1, "matrixman guard: wrong device type");
    int idx = d.index() < 0 ? 0 : d.index();
    TORCH_CHECK(MM_SYMBOL(dev_fn, "mm_set_device")(idx) == 0, "matrixman guard: cannot select device ", idx);
    t_current_device = idx;
  }

  void uncheckedSetDevice(c10::Device d) const noexcept override {
    int idx = d.index() < 0 ? 0 : d.index();
    static void* const p = dlsym(RTLD_DEFAULT, "mm_set_device");
    if (p) reinterpret_cast<dev_fn>(p)(idx);
    t_current_device = idx;
  }

  // One runtime stream per device (id 0 == the libmatrixman_b200 runtime stream).
  c10::Stream getStream(c10::Device d) const override {
    return c10::Stream(c10::Stream::DEFAULT, d);
  }
  c10::Stream getNewStream(c10::Device d, int) const override {
    return c10::Stream(c10::Stream::DEFAULT, d);
  }
  c10::Stream exchangeStream(c10::Stream s) const noexcept override { return s; }

  c10::DeviceIndex deviceCount() const noexcept override {
    static void* const p = dlsym(RTLD_DEFAULT, "mm_device_count");
    if (!p) return 0;
    int n = 0;
    if (reinterpret_cast<count_fn>(p)(&n) != 0) return 0;
    return (c10::DeviceIndex)n;
  }

  bool queryStream(const c10::Stream& s) const override {
    int done = 1;
    MM_SYMBOL(query_fn, "mm_stream_query")(runtime_stream(s.device_index()), &done);
    return done != 0;
  }

  void synchronizeStream(const c10::Stream& s) const override {
    sync_runtime_stream(s.device_index(), "stream synchronize");
  }

  void synchronizeDevice(const c10::DeviceIndex idx) const override {
    sync_runtime_stream(idx, "device synchronize");
  }
};

C10_REGISTER_GUARD_IMPL(PrivateUse1, MatrixManGuardImpl);

MatrixManHooks g_hooks;
std::atomic<bool> g_registered{false};

void register_hooks() {
  bool expected = false;
  if (g_registered.compare_exchange_strong(expected, true)) {
    at::RegisterPrivateUse1HooksInterface(&g_hooks);
  }
}

int guard_device_count() { return (int)MatrixManGuardImpl().deviceCount(); }

void set_wait_timeout_ms(int64_t ms) {
  TORCH_CHECK(ms > 0, "matrixman hooks: wait timeout must be positive");
  g_wait_timeout_ms.store(ms);
}

int64_t wait_timeout_ms() { return g_wait_timeout_ms.load(); }

// ---------------------------------------------------------------------------
// Calls of the layer-norm and linear entry points in one step: checks, output
// tensors and the native call, without the interpreter in between.  They take
// the ordinary case (float32 matrixman tensors of the current device, dense
// rows) and return None in any other, which the Python code then handles and
// words the errors of.  A training step of a small block spends most of its
// time on the host: layer norm forward + backward of 64 x 128 147 us before,
// 114 after.
// ---------------------------------------------------------------------------

using alloc_fn = int (*)(int, size_t, int, void*, void**);
using norm_fn = int (*)(const void*, int64_t, int64_t, int64_t, const void*, const void*, double, void*, void*, void*,
                        void*);
using norm_back_fn = int (*)(const void*, int64_t, const void*, int64_t, int64_t, int64_t, const void*, const void*,
                             const void*, void*, void*, void*, void*, size_t, void*);
using linear_fn = int (*)(const void*, int64_t, int64_t, const void*, int64_t, int64_t, const void*, const void*,
                          int64_t, int64_t, int64_t, int64_t, int, int, void*, void*, void*, size_t, void*);
using linear_back_fn = int (*)(const void*, int64_t, const void*, int64_t, int64_t, const void*, int64_t, int64_t,
                               const void*, int64_t, int64_t, int64_t, int, void*, void*, void*, void*, void*, size_t,
                               void*);

// A call into the native library without the interpreter's lock (as ctypes makes
// it): a full launch queue or an allocation may block, and the program's other
// threads go on meanwhile.  Every tensor whose address it takes is held by the
// caller.
template <class F, class... Args>
int unlocked(F f, Args... args) {
  py::gil_scoped_release released;
  return f(args...);
}

// A matrixman tensor's metadata and address.
struct Operand {
  bool given = false;
  const at::Tensor* t = nullptr;
  PyObject* owner = nullptr;  // borrowed: the tensor holds it
  char* ptr = nullptr;
  int64_t size(int i) const { return t->size(i); }
  int64_t dim() const { return t->dim(); }
};

// Interned, so that look-ups compare addresses.
py::object name(const char* s) { return py::reinterpret_steal<py::object>(PyUnicode_InternFromString(s)); }

struct Names {
  py::object owner = name("_owner"), pointer = name("pointer"), runtime = name("runtime"),
             index = name("index"), stream = name("stream"), offset = name("_storage_offset"),
             strides = name("_logical_strides");
  py::object make, storage, tensor, f32, strided, device_for, keywords;
  bool ready = false;
};

Names& names() {
  static Names* n = new Names();  // outlives the interpreter's own teardown
  return *n;
}

// The classes that results are made of (called once by the Python side).
void bind_tensors(py::object tensor_cls, py::object storage_cls, py::object device_for) {
  Names& n = names();
  py::module_ torch = py::module_::import("torch");
  n.make = torch.attr("Tensor").attr("_make_wrapper_subclass");
  n.tensor = tensor_cls;
  n.storage = storage_cls;
  n.device_for = device_for;
  n.f32 = torch.attr("float32");
  n.strided = torch.attr("strided");
  n.keywords = py::make_tuple("strides", "storage_offset", "dtype", "layout", "device", "requires_grad");
  n.ready = true;
}

py::object attribute(PyObject* o, const py::object& name) {
  PyObject* v = PyObject_GetAttr(o, name.ptr());
  if (v == nullptr) throw py::error_already_set();
  return py::reinterpret_steal<py::object>(v);
}

// False where o is not a float32 matrixman tensor (None: `given` stays false).
bool operand(const py::handle& o, Operand* out) {
  if (o.is_none()) return true;
  const Names& n = names();
  if (!PyObject_TypeCheck(o.ptr(), (PyTypeObject*)n.tensor.ptr())) return false;  // (a class below torch.Tensor)
  out->t = &THPVariable_Unpack(o.ptr());
  if (out->t->scalar_type() != at::kFloat) return false;
  py::object owner = attribute(o.ptr(), n.owner);
  out->owner = owner.ptr();
  out->ptr = (char*)PyLong_AsVoidPtr(attribute(out->owner, n.pointer).ptr()) + 4 * out->t->storage_offset();
  out->given = true;
  return true;
}

// The runtime that results belong to.
struct Target {
  py::object runtime, device;
  at::Device place = at::Device(at::kCPU);
  int index = 0;
  void* stream = nullptr;
  // False unless its device is the current one.
  bool of(const Operand& x) {
    const Names& n = names();
    runtime = attribute(x.owner, n.runtime);
    index = (int)PyLong_AsLong(attribute(runtime.ptr(), n.index).ptr());
    stream = PyLong_AsVoidPtr(attribute(runtime.ptr(), n.stream).ptr());
    int current = -1;
    if (MM_SYMBOL(count_fn, "mm_get_device")(&current) != 0 || current != index) return false;
    device = n.device_for(index);
    place = x.t->device();
    return true;
  }
  // (one runtime per device)
  bool owns(const Operand& o) const { return !o.given || o.t->device() == place; }
};

py::tuple int_tuple(at::IntArrayRef v) {
  py::tuple t(v.size());
  for (size_t i = 0; i < v.size(); ++i) PyTuple_SET_ITEM(t.ptr(), (Py_ssize_t)i, PyLong_FromLongLong(v[i]));
  return t;
}

// A block of `numel` floats of the activation pool as a DeviceStorage; null
// (the arena's message stands) where it cannot be had.
py::object new_storage(const Target& t, int64_t numel, char** ptr) {
  const size_t bytes = (size_t)(numel > 0 ? numel : 1) * 4;
  void* p = nullptr;
  if (unlocked(MM_SYMBOL(alloc_fn, "mm_alloc"), t.index, bytes, 0, t.stream, &p) != 0) return py::object();
  *ptr = (char*)p;
  return names().storage(t.runtime, (int64_t)(intptr_t)p, bytes, names().f32, 0);
}

py::object new_tensor(const Target& t, const py::object& owner, const py::tuple& shape, const py::tuple& strides,
                      int64_t offset) {
  const Names& n = names();
  py::object off = py::int_(offset);
  PyObject* args[] = {n.tensor.ptr(), shape.ptr(), strides.ptr(),    off.ptr(),
                      n.f32.ptr(),    n.strided.ptr(), t.device.ptr(), Py_False};
  PyObject* r = PyObject_Vectorcall(n.make.ptr(), args, 2, n.keywords.ptr());
  if (r == nullptr) throw py::error_already_set();
  py::object out = py::reinterpret_steal<py::object>(r);
  if (PyObject_SetAttr(r, n.owner.ptr(), owner.ptr()) != 0 || PyObject_SetAttr(r, n.offset.ptr(), off.ptr()) != 0 ||
      PyObject_SetAttr(r, n.strides.ptr(), strides.ptr()) != 0)
    throw py::error_already_set();
  return out;
}

py::tuple dense_strides(at::IntArrayRef shape) {
  std::vector<int64_t> s(shape.size());
  int64_t n = 1;
  for (size_t i = shape.size(); i-- > 0;) {
    s[i] = n;
    n *= shape[i] > 1 ? shape[i] : 1;
  }
  return int_tuple(s);
}

// A new dense tensor of this shape in a block of its own; *ptr is its address.
py::object new_dense(const Target& t, at::IntArrayRef shape, char** ptr) {
  int64_t n = 1;
  for (int64_t v : shape) n *= v;
  py::object owner = new_storage(t, n, ptr);
  return owner ? new_tensor(t, owner, int_tuple(shape), dense_strides(shape), 0) : py::object();
}

// Rows of dense values: their distance; -1 where the strides are others.
int64_t row_stride(const Operand& x, int64_t width) {
  if (x.dim() == 2) return x.t->stride(1) == 1 || width == 1 ? x.t->stride(0) : -1;
  return x.t->is_contiguous() ? width : -1;
}

bool is_vector(const Operand& o, int64_t n) {
  return !o.given || (o.dim() == 1 && o.size(0) == n && (n <= 1 || o.t->stride(0) == 1));
}

// Any of these functions returns None (not the ordinary case), an int (the
// status of a native call that failed), or its results.
py::object layer_norm(py::handle x_, int64_t width, py::handle w_, py::handle b_, double eps) {
  Operand x, w, b;
  Target t;
  if (!names().ready || !operand(x_, &x) || !operand(w_, &w) || !operand(b_, &b) || !x.given) return py::none();
  const int64_t d = x.dim();
  if (d < 1 || width < 1 || x.size(d - 1) != width || !is_vector(w, width) || !is_vector(b, width)) return py::none();
  const int64_t stride = row_stride(x, width);
  if (stride < 0 || !t.of(x) || !t.owns(w) || !t.owns(b)) return py::none();
  const int64_t rows = x.t->numel() / width;
  // mean and rstd share a block, apart from y's: they are kept for the backward pass, y may go.
  char *py_ = nullptr, *ps = nullptr;
  py::object y = new_dense(t, x.t->sizes(), &py_);
  if (!y) return py::none();
  py::object owner = new_storage(t, 2 * rows, &ps);
  if (!owner) return py::none();
  const int status = unlocked(MM_SYMBOL(norm_fn, "mm_layer_norm"), x.ptr, stride, rows, width, w.ptr, b.ptr, eps, py_,
                              ps, ps + 4 * rows, t.stream);
  if (status != 0) return py::int_(status);
  std::vector<int64_t> shape = x.t->sizes().vec();
  shape.back() = 1;
  py::tuple stat = int_tuple(shape), strides = dense_strides(shape);
  return py::make_tuple(y, new_tensor(t, owner, stat, strides, 0), new_tensor(t, owner, stat, strides, rows));
}

py::object layer_norm_backward(py::handle dy_, py::handle x_, int64_t width, py::handle mean_, py::handle rstd_,
                               py::handle w_, py::handle b_, bool need_x, bool need_w, bool need_b) {
  Operand dy, x, mean, rstd, w, b;
  Target t;
  if (!names().ready || !operand(dy_, &dy) || !operand(x_, &x) || !operand(mean_, &mean) || !operand(rstd_, &rstd) ||
      !operand(w_, &w) || !operand(b_, &b) || !dy.given || !x.given || !mean.given || !rstd.given)
    return py::none();
  const int64_t d = x.dim();
  if (d < 1 || width < 1 || x.size(d - 1) != width || dy.t->sizes() != x.t->sizes() || !is_vector(w, width) ||
      (need_w && !w.given) || (need_b && !b.given) || !mean.t->is_contiguous() || !rstd.t->is_contiguous())
    return py::none();
  const int64_t rows = x.t->numel() / width, xs = row_stride(x, width), gs = row_stride(dy, width);
  if (xs < 0 || gs < 0 || mean.t->numel() != rows || rstd.t->numel() != rows || !t.of(x) || !t.owns(dy) ||
      !t.owns(mean) || !t.owns(rstd) || !t.owns(w) || !t.owns(b))
    return py::none();
  char *px = nullptr, *pw = nullptr;
  py::object dx = py::none(), dw = py::none(), db = py::none();
  if (need_x && !(dx = new_dense(t, x.t->sizes(), &px))) return py::none();
  const int64_t each = (width + 63) / 64 * 64;  // dw and db share a block, each at a 256-byte boundary
  if (need_w || need_b) {
    py::object owner = new_storage(t, 2 * each, &pw);
    if (!owner) return py::none();
    py::tuple shape = py::make_tuple(width), one = py::make_tuple(1);
    if (need_w) dw = new_tensor(t, owner, shape, one, 0);
    if (need_b) db = new_tensor(t, owner, shape, one, each);
  }
  const int status = unlocked(MM_SYMBOL(norm_back_fn, "mm_layer_norm_backward"), dy.ptr, gs, x.ptr, xs, rows, width,
                              mean.ptr, rstd.ptr, w.ptr, px, need_w ? pw : nullptr, need_b ? pw + 4 * each : nullptr,
                              nullptr, 0, t.stream);
  if (status != 0) return py::int_(status);
  return py::make_tuple(dx, dw, db);
}

// [..., k] as rows: their number and the two strides; false where that takes a copy.
bool matrix(const Operand& x, int64_t* rows, int64_t* s0, int64_t* s1) {
  const int64_t d = x.dim();
  if (d == 2) {
    *rows = x.size(0);
    *s0 = x.t->stride(0);
    *s1 = x.t->stride(1);
    return true;
  }
  if (d < 2 || !x.t->is_contiguous()) return false;
  *s0 = x.size(d - 1);
  *s1 = 1;
  *rows = 1;
  for (int64_t i = 0; i + 1 < d; ++i) *rows *= x.size(i);
  return true;
}

// The operands of a linear call in the ordinary case.
struct LinearCall {
  Operand x, w, b, r;
  Target t;
  int64_t m = 0, n = 0, k = 0, xs0 = 0, xs1 = 0, rs = 0;
  std::vector<int64_t> shape;
  bool setup(const py::handle& x_, const py::handle& w_, const py::handle& b_, const py::handle& r_) {
    if (!names().ready || !operand(x_, &x) || !operand(w_, &w) || !operand(b_, &b) || !operand(r_, &r) || !x.given ||
        !w.given || w.dim() != 2)
      return false;
    n = w.size(0);
    k = w.size(1);
    if (!matrix(x, &m, &xs0, &xs1) || x.size(x.dim() - 1) != k || !is_vector(b, n)) return false;
    shape = x.t->sizes().vec();
    shape.back() = n;
    if (r.given && (r.t->sizes() != at::IntArrayRef(shape) || (rs = row_stride(r, n)) < 0)) return false;
    return t.of(x) && t.owns(w) && t.owns(b) && t.owns(r);
  }
};

bool linear_ready(py::handle x, py::handle w, py::handle b, py::handle r) {
  LinearCall c;
  return c.setup(x, w, b, r);
}

py::object linear(py::handle x_, py::handle w_, py::handle b_, py::handle r_, int act, bool first, bool keep) {
  LinearCall c;
  if (!c.setup(x_, w_, b_, r_)) return py::none();
  char *py_ = nullptr, *pz = nullptr;
  py::object y = new_dense(c.t, c.shape, &py_), z = py::none();
  if (!y || (keep && !(z = new_dense(c.t, c.shape, &pz)))) return py::none();
  const int status = unlocked(MM_SYMBOL(linear_fn, "mm_linear"), c.x.ptr, c.xs0, c.xs1, c.w.ptr, c.w.t->stride(0),
                              c.w.t->stride(1), c.b.ptr, c.r.ptr, c.rs, c.m, c.n, c.k, act, first, py_, pz, nullptr, 0,
                              c.t.stream);
  if (status != 0) return py::int_(status);
  return py::make_tuple(y, z);
}

py::object linear_backward(py::handle dy_, py::handle x_, py::handle w_, py::handle z_, int act, bool need_x,
                           bool need_w, bool need_b, bool need_z) {
  Operand dy, x, w, z;
  Target t;
  if (!names().ready || !operand(dy_, &dy) || !operand(x_, &x) || !operand(w_, &w) || !operand(z_, &z) || !dy.given ||
      !x.given || !w.given || w.dim() != 2 || dy.dim() < 2)
    return py::none();
  const int64_t n = w.size(0), k = w.size(1), gs = row_stride(dy, n);
  int64_t m, xs0, xs1;
  if (gs < 0 || dy.size(dy.dim() - 1) != n || !matrix(x, &m, &xs0, &xs1) || dy.t->numel() != m * n ||
      (z.given && !z.t->is_contiguous()))
    return py::none();
  if (!t.of(x) || !t.owns(dy) || !t.owns(w) || !t.owns(z)) return py::none();
  char *px = nullptr, *pw = nullptr, *pb = nullptr, *pz = nullptr;
  py::object dx = py::none(), dw = py::none(), db = py::none(), dz = py::none();
  const int64_t wn[] = {n, k};
  if (need_x && !(dx = new_dense(t, x.t->sizes(), &px))) return py::none();
  if (need_w && !(dw = new_dense(t, wn, &pw))) return py::none();
  if (need_b && !(db = new_dense(t, at::IntArrayRef(wn, 1), &pb))) return py::none();
  if (need_z && !(dz = new_dense(t, dy.t->sizes(), &pz))) return py::none();
  const int status = unlocked(MM_SYMBOL(linear_back_fn, "mm_linear_backward"), dy.ptr, gs, x.ptr, xs0, xs1, w.ptr,
                              w.t->stride(0), w.t->stride(1), z.ptr, m, n, k, act, px, pw, pb, pz, nullptr, 0,
                              t.stream);
  if (status != 0) return py::int_(status);
  return py::make_tuple(dx, dw, db, dz);
}

using adamw_fn = int (*)(const void*, int, int, double, double, double, double, double, int, int, int, void*, size_t,
                         void*);
using decode_fn = int (*)(const void*, const void*, const void*, const void*, int64_t, void*, void*, void*);

// Whether 8-bit codes (four to a float) and their scales are those of p's elements.
bool holds_codes(const Operand& codes, const Operand& scales, const Operand& p) {
  const int64_t blocks = (p.t->numel() + 255) / 256;
  return codes.t->numel() == 64 * blocks && scales.t->numel() == blocks && codes.t->is_contiguous() &&
         scales.t->is_contiguous();
}

// An optimiser step over parameters with gradients and the states of
// optim.AdamW (dicts): the table of addresses and the native call.  True, an
// int (its status), or None where a tensor is not as usual.
py::object adamw_step(const py::list& params, const py::list& states, int bits, double lr, double beta1, double beta2,
                      double eps, double decay, bool maximize) {
  static const py::object& grad_name = *new py::object(name("grad"));
  static const py::object& step_name = *new py::object(name("step"));
  static const py::object* const wide = new py::object[2]{name("exp_avg"), name("exp_avg_sq")};
  static const py::object* const narrow = new py::object[4]{name("exp_avg_code"), name("exp_avg_sq_code"),
                                                            name("exp_avg_scale"), name("exp_avg_sq_scale")};
  const size_t count = params.size();
  if (!names().ready || count == 0 || states.size() != count) return py::none();
  std::vector<int64_t> table(8 * count);
  std::vector<py::object> held;  // the lists and dicts are the program's: it may change them during the call
  held.reserve(8 * count);
  Target t;
  auto state_of = [&](const py::handle& state, const py::object& name, Operand* out) {
    PyObject* v = PyDict_GetItemWithError(state.ptr(), name.ptr());
    if (v == nullptr) return false;
    held.push_back(py::reinterpret_borrow<py::object>(v));
    return operand(v, out) && out->given && t.owns(*out);
  };
  for (size_t i = 0; i < count; ++i) {
    Operand p, g, m, v, ms, vs, step;
    if (!operand(params[i], &p) || !p.given || !p.t->is_non_overlapping_and_dense()) return py::none();
    if (i == 0 ? !t.of(p) : !t.owns(p)) return py::none();
    held.push_back(params[i]);
    held.push_back(attribute(params[i].ptr(), grad_name));
    if (!operand(held.back(), &g) || !g.given || !t.owns(g) || g.t->sizes() != p.t->sizes() ||
        g.t->strides() != p.t->strides())
      return py::none();
    const py::handle state = states[i];
    if (!PyDict_Check(state.ptr()) || !state_of(state, step_name, &step) || step.t->numel() != 1) return py::none();
    if (bits == 8) {
      if (!state_of(state, narrow[0], &m) || !state_of(state, narrow[1], &v) || !state_of(state, narrow[2], &ms) ||
          !state_of(state, narrow[3], &vs) || !holds_codes(m, ms, p) || !holds_codes(v, vs, p))
        return py::none();
    } else if (!state_of(state, wide[0], &m) || !state_of(state, wide[1], &v) || m.t->sizes() != p.t->sizes() ||
               v.t->sizes() != p.t->sizes() || m.t->strides() != p.t->strides() || v.t->strides() != p.t->strides()) {
      return py::none();
    }
    const Operand* order[] = {&p, &g, &m, &v, &ms, &vs, &step};
    for (int j = 0; j < 7; ++j) table[8 * i + j] = (int64_t)(intptr_t)order[j]->ptr;
    table[8 * i + 7] = p.t->numel();
  }
  const int status = unlocked(MM_SYMBOL(adamw_fn, "mm_adamw"), table.data(), (int)count, bits, lr, beta1, beta2, eps,
                              decay, 1, maximize, 1, nullptr, 0, t.stream);
  return status == 0 ? py::object(py::bool_(true)) : py::object(py::int_(status));
}

// The float32 values of 8-bit states, of a parameter's shape and strides (the step
// is only looked at: the whole state has to fit).
py::object adamw_values(py::handle p_, py::handle mc_, py::handle ms_, py::handle vc_, py::handle vs_,
                        py::handle step_) {
  Operand p, mc, ms, vc, vs, step;
  Target t;
  if (!names().ready || !operand(p_, &p) || !operand(mc_, &mc) || !operand(ms_, &ms) || !operand(vc_, &vc) ||
      !operand(vs_, &vs) || !operand(step_, &step) || !p.given || !mc.given || !ms.given || !vc.given || !vs.given ||
      !step.given || step.t->numel() != 1 ||
      !p.t->is_non_overlapping_and_dense() || !holds_codes(mc, ms, p) || !holds_codes(vc, vs, p) || !t.of(p) ||
      !t.owns(mc) || !t.owns(ms) || !t.owns(vc) || !t.owns(vs) || !t.owns(step))
    return py::none();
  const int64_t n = p.t->numel(), at = (n + 63) / 64 * 64;  // both in one block
  char* ptr = nullptr;
  py::object owner = new_storage(t, at + n, &ptr);
  if (!owner) return py::none();
  const int status = unlocked(MM_SYMBOL(decode_fn, "mm_adamw_decode"), mc.ptr, ms.ptr, vc.ptr, vs.ptr, n, ptr,
                              ptr + 4 * at, t.stream);
  if (status != 0) return py::int_(status);
  const py::tuple shape = int_tuple(p.t->sizes()), strides = int_tuple(p.t->strides());
  return py::make_tuple(new_tensor(t, owner, shape, strides, 0), new_tensor(t, owner, shape, strides, at));
}

}  // namespace

PYBIND11_MODULE(TORCH_EXTENSION_NAME, m) {
  m.def("register_hooks", &register_hooks, "Register the matrixman PrivateUse1 hooks");
  m.def("device_count", &guard_device_count, "Device count seen by the DeviceGuard");
  m.def("set_wait_timeout_ms", &set_wait_timeout_ms, "Bound of the guard's stream waits (ms)");
  m.def("wait_timeout_ms", &wait_timeout_ms, "Bound of the guard's stream waits (ms)");
  m.def("bind_tensors", &bind_tensors, "Classes that the operators below make their results of");
  m.def("layer_norm", &layer_norm, "mm_layer_norm with its outputs, or None");
  m.def("layer_norm_backward", &layer_norm_backward, "mm_layer_norm_backward with its outputs, or None");
  m.def("linear", &linear, "mm_linear with its outputs, or None");
  m.def("linear_ready", &linear_ready, "Whether linear would take these operands");
  m.def("adamw_step", &adamw_step, "mm_adamw over parameters and their states, or None");
  m.def("adamw_values", &adamw_values, "mm_adamw_decode with its outputs, or None");
  m.def("linear_backward", &linear_backward, "mm_linear_backward with its outputs, or None");
}
