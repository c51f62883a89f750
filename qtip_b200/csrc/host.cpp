// Host path of one QTIP linear: BitshiftLinear.forward (lib/codebook/bitshift.py:428-472 upstream) as one native call.
//
// A layer call is two transforms around a decode + product, 8..60 us of GPU work.  Issued from Python - three wrappers,
// each with its own device switch, stream query, argument checks, tensor construction and ctypes conversion - it cost
// 80-93 us of host time per call (measured at every layer shape that runs for less), so the GPU waited for the
// interpreter.  Here the whole call is made from C++: one scratch allocation for the two intermediates, one for the
// result, and the library's launches back to back on the current stream.
//
// Module functions (CPython API, no binding layer):
//   linear_forward(input, trellis, tlut|None, SU, SV, bits_left|None, k_left, bits_right|None, k_right, code, K,
//                  kernel_layout, rcp, tp, workspace|None) -> (output, launches)
//   matvec_workspace(device_index, m, n, bs) -> uint8 tensor    the fused matvec's scratch of (device, current stream)
//   gemm_status(device_index) -> int32 tensor                   the decompress-GEMM's status word of a device
//   kv_plan, rope_kv_append_paged, attn_decode_paged, beam_select, beam_reorder: the checks and launches of the functions of the same
//   names in ops.py (calls of 3 to 8 us of GPU work, for which the checks in Python took 13 to 25 us) -> launches
#include <torch/csrc/autograd/python_variable.h>

#include <ATen/ATen.h>
#include <ATen/cuda/CUDAContext.h>
#include <c10/core/GradMode.h>
#include <c10/cuda/CUDACachingAllocator.h>
#include <c10/cuda/CUDAGuard.h>

#include <cmath>
#include <algorithm>
#include <map>
#include <memory>
#include <mutex>
#include <string>
#include <utility>
#include <vector>

#include "../../include/qtip_b200.h"

namespace {

constexpr int64_t kMaxMatvecBatch = 8, kMaxGemmBatch = 128;
constexpr double kInternalScale = 32.0;    // bitshift.py:373 upstream: keeps the fp16 activation in range

struct Failure {
    std::string what;
};

void check(int status, const char *what) {
    if (status == QTIP_OK) return;
    std::string msg = std::string(what) + ": " + qtip_status_string(status);
    if (status == QTIP_ERR_CUDA) msg += " (cudaError " + std::to_string(qtip_last_cuda_error()) + ")";
    throw Failure{msg};
}

int dtype_id(const at::Tensor &t) {
    if (t.scalar_type() == at::kHalf) return QTIP_F16;
    if (t.scalar_type() == at::kFloat) return QTIP_F32;
    throw Failure{std::string("unsupported dtype ") + c10::toString(t.scalar_type()) + " (fp16 / fp32 only)"};
}

// Per-device / per-stream scratch that outlives a call.  One matvec workspace per (device, stream): calls on one stream
// are ordered, so they can share it; torch hands out a bounded set of streams.  It is zeroed once and the kernels leave
// it zeroed.  Never destroyed at exit (the CUDA context may be gone by then).
// A CUDA graph keeps the addresses it was captured with: a workspace that has to grow is replaced by one of at least twice its
// size and kept (all replaced ones of a stream are smaller together than the one in use), and a capture that finds none gets one
// of its own from the graph's memory, zeroed by the graph (a zeroing recorded into a graph is no zeroing of what others use).
//
// g_mutex is taken with and without the GIL, so nothing that may call into Python (and wait for the GIL) happens under it:
// no allocation or release of a tensor (memory history, allocator hooks) and no copy of a tensor handle (its Python object).
// The maps hold shared pointers; those are what is read and exchanged under the lock.
using TensorPtr = std::shared_ptr<const at::Tensor>;
std::mutex g_mutex;
std::map<std::pair<int, void *>, TensorPtr> &workspaces() {
    static auto *m = new std::map<std::pair<int, void *>, TensorPtr>();
    return *m;
}
std::vector<TensorPtr> &replaced() {
    static auto *v = new std::vector<TensorPtr>();
    return *v;
}
std::map<int, TensorPtr> &status_words() {
    static auto *m = new std::map<int, TensorPtr>();
    return *m;
}

// The entry of `key`, made by `make` when it is missing or `ok` refuses it.  Of two threads that make one at the same time
// the first to store it wins; what the other made is released outside the lock.
template <class Map, class Key, class Ok, class Make>
TensorPtr find_or_make(Map &map, const Key &key, Ok ok, Make make) {
    size_t had = 0;      // bytes of the entry that is too small
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        const auto it = map.find(key);
        if (it != map.end()) {
            if (ok(*it->second)) return it->second;
            had = it->second->nbytes();
        }
    }
    bool keep = true;
    TensorPtr made = std::make_shared<const at::Tensor>(make(had, keep)), got;
    if (!keep) return made;
    {
        std::lock_guard<std::mutex> lock(g_mutex);
        TensorPtr &slot = map[key];
        if (!slot || !ok(*slot)) {
            if (slot) replaced().push_back(std::move(slot));
            slot = std::move(made);
        }
        got = slot;
    }
    return got;
}

at::Tensor matvec_workspace(int dev, int64_t m, int64_t n, int64_t bs, void *stream) {
    const size_t need = qtip_matvec_workspace_bytes((int)m, (int)n, (int)bs);
    return *find_or_make(workspaces(), std::make_pair(dev, stream), [&](const at::Tensor &t) { return (size_t)t.numel() >= need; },
                         [&](size_t had, bool &keep) {
        cudaStreamCaptureStatus capture = cudaStreamCaptureStatusNone;
        if (cudaStreamIsCapturing(static_cast<cudaStream_t>(stream), &capture) != cudaSuccess) throw Failure{"cudaStreamIsCapturing failed"};
        keep = capture == cudaStreamCaptureStatusNone;
        const size_t bytes = keep ? std::max<size_t>({need, 2 * had, (size_t)1 << 20}) : need;
        return at::zeros({(int64_t)bytes}, at::TensorOptions().dtype(at::kByte).device(at::kCUDA, dev));
    });
}

at::Tensor gemm_status(int dev) {
    return *find_or_make(status_words(), dev, [](const at::Tensor &) { return true; },
                         [&](size_t, bool &) { return at::zeros({1}, at::TensorOptions().dtype(at::kInt).device(at::kCUDA, dev)); });
}

struct Layer {
    const at::Tensor &trellis, &SU, &SV;
    at::Tensor tlut, bits_left, bits_right, workspace;   // undefined = absent
    int k_left, k_right, code, K, rcp, tp;
    bool kernel_layout;
};

bool aligned16(const at::Tensor &t) { return reinterpret_cast<uintptr_t>(t.data_ptr()) % 16 == 0; }

at::Tensor linear_forward(const at::Tensor &input, Layer &L, int &launches) {
    const int64_t n = L.SU.numel(), m = L.SV.numel();
    for (const at::Tensor *t : {&input, &L.trellis, &L.SU, &L.SV, (const at::Tensor *)&L.tlut, (const at::Tensor *)&L.bits_left,
                                (const at::Tensor *)&L.bits_right})
        if (t->defined() && !t->is_cuda()) throw Failure{"qtip_b200 runs on CUDA tensors only (no CPU fallback)"};
    const int dev = input.get_device();
    c10::cuda::OptionalCUDAGuard guard;
    if (dev != c10::cuda::current_device()) guard.set_index((c10::DeviceIndex)dev);
    void *stream = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();

    at::Tensor x = input.is_contiguous() ? input : input.contiguous();
    if (n == 0 || x.numel() % n) throw Failure{"the input's last dimension does not match SU"};
    const int64_t bs = x.numel() / n;
    const auto in_type = input.scalar_type();
    if (in_type != at::kHalf && in_type != at::kFloat) x = x.to(at::kFloat);
    const auto out_type = in_type == at::kHalf ? at::kHalf : at::kFloat;
    const at::Tensor SU = L.SU.is_contiguous() ? L.SU : L.SU.contiguous();
    const at::Tensor SV = L.SV.scalar_type() == at::kFloat && L.SV.is_contiguous() ? L.SV : L.SV.to(at::kFloat).contiguous();
    const at::Tensor trellis = L.trellis.is_contiguous() ? L.trellis : L.trellis.contiguous();
    if (trellis.nbytes() != (size_t)(m * n * L.K / 8))
        throw Failure{"codes hold " + std::to_string(trellis.nbytes()) + " bytes, expected " + std::to_string(m * n * L.K / 8)};
    at::Tensor tlut = L.tlut;
    if (tlut.defined() && (tlut.scalar_type() != at::kHalf || !tlut.is_contiguous())) tlut = tlut.to(at::kHalf).contiguous();
    const uint32_t *bl = L.bits_left.defined() ? static_cast<const uint32_t *>(L.bits_left.data_ptr()) : nullptr;
    const uint32_t *br = L.bits_right.defined() ? static_cast<const uint32_t *>(L.bits_right.data_ptr()) : nullptr;

    const auto opts = at::TensorOptions().device(at::kCUDA, dev);
    std::vector<int64_t> shape(input.sizes().begin(), input.sizes().end());
    shape.back() = m;
    at::Tensor out = at::empty(shape, opts.dtype(out_type));
    if (bs == 0) return in_type == out_type ? out : out.to(in_type);

    const bool v1 = L.code != QTIP_CODE_HYB;
    const bool whole_tiles = m % 128 == 0 && n % 64 == 0;      // what the tensor-core kernel needs
    // compute codes: the tensor-core kernel decodes eight states per 44-bit window and is the faster one at every batch
    // size it takes; HYB: above 8 rows the matvec's single B fragment is full
    const bool gemm = whole_tiles && bs <= kMaxGemmBatch && (v1 || (L.kernel_layout && bs > kMaxMatvecBatch));
    // long prompts: the tensor-core kernel again where it is the faster way, else decoded once and a dense product
    const bool wide = whole_tiles && bs > kMaxGemmBatch && (v1 || L.kernel_layout) && aligned16(trellis) &&
                      qtip_decompress_gemm_f16_faster(L.code, (int)m, (int)n, (int)bs);
    const bool dense = !gemm && !wide && bs > kMaxMatvecBatch;

    // one allocation for both intermediates: the transformed activation (fp16) and, unless the dense product makes its
    // own, the raw result (fp32; fp16 of a long prompt, as from the dense product)
    const int64_t xh_bytes = (bs * n * 2 + 255) / 256 * 256;
    // (straight from the caching allocator, on the current stream: a tensor around it costs half a microsecond)
    const c10::DataPtr scratch = c10::cuda::CUDACachingAllocator::get()->allocate(xh_bytes + (dense ? 0 : bs * m * (wide ? 2 : 4)));
    char *base = static_cast<char *>(scratch.get());
    void *xh = base;
    float *y = reinterpret_cast<float *>(base + xh_bytes);

    // input side: x * SU -> Hadamard^T (per chunk when row-parallel) -> / 32 -> fp16
    const int64_t seg_n = L.rcp == 1 ? n / L.tp : n;
    // rows that the matvec takes in fragment order are written so by the transform
    const bool fragments = !gemm && !wide && !dense && L.kernel_layout && seg_n == n && aligned16(x) && aligned16(SU) &&
                           qtip_matvec_x_fragments(L.K, (int)m, (int)n, (int)bs);
    check(qtip_rht(xh, fragments ? QTIP_F16_FRAGMENTS : QTIP_F16, x.data_ptr(), dtype_id(x), bs * (n / seg_n), (int)seg_n, SU.data_ptr(), dtype_id(SU), nullptr,
                   n, bl, L.k_left, 1, (float)(1.0 / (std::sqrt((double)seg_n) * kInternalScale)), stream),
          "qtip_rht");
    launches = 3;
    at::Tensor dense_y;
    const void *y_in = y;
    int y_type = QTIP_F32;
    if (gemm || wide) {
        // (qtip_rht starts it when the weights, whatever wrote them, are complete)
        y_type = wide ? QTIP_F16 : QTIP_F32;
        check(qtip_decompress_gemm_settled(y, y_type, trellis.data_ptr(), xh, v1 ? nullptr : tlut.data_ptr(), L.code, L.K, (int)m, (int)n, (int)bs,
                                           static_cast<unsigned *>(gemm_status(dev).data_ptr()), stream),
              "qtip_decompress_gemm_settled");
    } else if (!dense) {
        at::Tensor ws = L.workspace.defined() ? L.workspace : matvec_workspace(dev, m, n, bs, stream);
        if (fragments)
            check(qtip_decompress_matvec_fragments(y, trellis.data_ptr(), xh, tlut.data_ptr(), L.K, (int)m, (int)n, (int)bs, ws.data_ptr(),
                                                   (size_t)ws.nbytes(), stream),
                  "qtip_decompress_matvec_fragments");
        else if (L.kernel_layout)
            check(qtip_decompress_matvec(y, trellis.data_ptr(), xh, tlut.data_ptr(), L.K, (int)m, (int)n, (int)bs, ws.data_ptr(),
                                         (size_t)ws.nbytes(), stream),
                  "qtip_decompress_matvec");
        else
            check(qtip_decompress_matvec_plain(y, trellis.data_ptr(), xh, L.code, L.K, (int)m, (int)n, (int)bs, ws.data_ptr(),
                                               (size_t)ws.nbytes(), stream),
                  "qtip_decompress_matvec_plain");
    } else {
        // anything else: decode once, dense fp16 GEMM (BitshiftLinearKernelAG upstream, bitshift.py:476-489); the fp16
        // product goes to the output transform as it is
        at::Tensor W = at::empty({m, n}, opts.dtype(at::kHalf));
        if (L.kernel_layout)
            check(qtip_decode_hyb_settled(W.data_ptr(), trellis.data_ptr(), tlut.data_ptr(), L.K, (int)m, (int)n, stream),
                  "qtip_decode_hyb_settled");
        else
            check(qtip_decode_plain(W.data_ptr(), trellis.data_ptr(), L.code, tlut.defined() ? tlut.data_ptr() : nullptr, L.K, (int)m,
                                    (int)n, stream),
                  "qtip_decode_plain");
        at::Tensor xt = at::from_blob(xh, {bs, n}, opts.dtype(at::kHalf));
        dense_y = at::mm(xt, W.t());
        y_in = dense_y.data_ptr();
        y_type = QTIP_F16;
    }

    // output side: Hadamard (per chunk when column-parallel) -> * SV * 32
    const int64_t seg_m = L.rcp == 2 ? m / L.tp : m;
    check(qtip_rht(out.data_ptr(), dtype_id(out), y_in, y_type, bs * (m / seg_m), (int)seg_m, nullptr, QTIP_F16,
                   static_cast<const float *>(SV.data_ptr()), m, br, L.k_right, 0, (float)(kInternalScale / std::sqrt((double)seg_m)),
                   stream),
          "qtip_rht");
    return in_type == out_type ? out : out.to(in_type);
}

// ---- CPython module ------------------------------------------------------------------------------------------
at::Tensor tensor_arg(PyObject *o, const char *name) {
    if (o == Py_None) return at::Tensor();
    if (!THPVariable_Check(o)) throw Failure{std::string(name) + " must be a tensor"};
    return THPVariable_Unpack(o);
}
long int_arg(PyObject *o) {
    const long v = PyLong_AsLong(o);
    if (v == -1 && PyErr_Occurred()) throw Failure{""};
    return v;
}

struct WithoutGil {
    PyThreadState *s = PyEval_SaveThread();
    ~WithoutGil() { PyEval_RestoreThread(s); }
};

// Runs `body`, turning failures (the library's and torch's) into RuntimeError as the Python wrappers raise.
template <class F>
PyObject *guarded(F body) {
    try {
        return body();
    } catch (const Failure &f) {
        if (!PyErr_Occurred()) PyErr_SetString(PyExc_RuntimeError, f.what.c_str());
    } catch (const c10::Error &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what_without_backtrace());
    } catch (const std::exception &e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject *py_linear_forward(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 15) throw Failure{"linear_forward takes 15 arguments"};
        const at::Tensor input = tensor_arg(a[0], "input"), trellis = tensor_arg(a[1], "trellis"), SU = tensor_arg(a[3], "SU"),
                         SV = tensor_arg(a[4], "SV");
        if (!input.defined() || !trellis.defined() || !SU.defined() || !SV.defined()) throw Failure{"linear_forward: missing tensor"};
        Layer L{trellis, SU, SV, tensor_arg(a[2], "tlut"), tensor_arg(a[5], "bits_left"), tensor_arg(a[7], "bits_right"),
                tensor_arg(a[14], "workspace"), (int)int_arg(a[6]), (int)int_arg(a[8]), (int)int_arg(a[9]), (int)int_arg(a[10]),
                (int)int_arg(a[12]), (int)int_arg(a[13]), int_arg(a[11]) != 0};
        if (L.code == QTIP_CODE_HYB && !L.tlut.defined()) throw Failure{"the HYB code needs its table"};
        int launches = 0;
        at::Tensor out;
        {
            c10::NoGradGuard no_grad;       // raw launches: nothing here can be differentiated through
            WithoutGil nogil;
            out = linear_forward(input, L, launches);
        }
        return Py_BuildValue("(Ni)", THPVariable_Wrap(std::move(out)), launches);
    });
}

PyObject *py_matvec_workspace(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 4) throw Failure{"matvec_workspace takes 4 arguments"};
        const int dev = (int)int_arg(a[0]);
        const long m = int_arg(a[1]), n = int_arg(a[2]), bs = int_arg(a[3]);
        void *stream = at::cuda::getCurrentCUDAStream((c10::DeviceIndex)dev).stream();
        return THPVariable_Wrap(matvec_workspace(dev, m, n, bs, stream));
    });
}

PyObject *py_gemm_status(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return guarded([&]() -> PyObject * {
        if (nargs != 1) throw Failure{"gemm_status takes 1 argument"};
        return THPVariable_Wrap(gemm_status((int)int_arg(a[0])));
    });
}

// ---- batched decoding over the 8-bit cache, and beam search: checks and launches -----------------------------------------------------------
const at::Tensor *maybe(PyObject *o, const char *name) {
    if (o == Py_None) return nullptr;
    if (!THPVariable_Check(o)) throw Failure{std::string(name) + " must be a tensor"};
    return &THPVariable_Unpack(o);
}
const at::Tensor &given(PyObject *o, const char *name) {
    const at::Tensor *t = maybe(o, name);
    if (!t) throw Failure{std::string(name) + " must be a tensor"};
    return *t;
}
// The call goes to the current device and stream (so that a step can be captured): tensors that live elsewhere are refused.
void here(std::initializer_list<const at::Tensor *> tensors) {
    for (const at::Tensor *t : tensors)
        if (t && !t->is_cuda()) throw Failure{"qtip_b200 runs on CUDA tensors only (no CPU fallback)"};
    const int cur = c10::cuda::current_device();
    for (const at::Tensor *t : tensors)
        if (t && t->get_device() != cur)
            throw Failure{"tensor on cuda:" + std::to_string(t->get_device()) + " but the current device is cuda:" + std::to_string(cur) +
                          ": call torch.cuda.set_device() / use torch.cuda.device() around qtip_b200 launches"};
}
std::string text(at::IntArrayRef shape) {
    std::string s = "(";
    for (size_t i = 0; i < shape.size(); i++) s += (i ? ", " : "") + std::to_string(shape[i]);
    return s + ")";
}
void expect(const char *name, const at::Tensor &t, at::ScalarType type, at::IntArrayRef shape, bool contiguous = true) {
    if (t.scalar_type() != type) throw Failure{std::string(name) + ": " + c10::toString(type) + " expected, not " + c10::toString(t.scalar_type())};
    if (t.sizes() != shape) throw Failure{std::string(name) + ": shape " + text(shape) + " expected, not " + text(t.sizes())};
    if (contiguous && !t.is_contiguous()) throw Failure{std::string(name) + " has to be contiguous"};
}
// Row stride of a (rows, width) fp16 matrix whose rows are contiguous.
long rows_of(const char *name, const at::Tensor &t, int64_t rows, int64_t width) {
    if (t.dim() != 2 || t.scalar_type() != at::kHalf || t.size(0) != rows || t.size(1) != width)
        throw Failure{std::string(name) + ": " + text({rows, width}) + " fp16 expected, not " + text(t.sizes()) + " " + c10::toString(t.scalar_type())};
    if (width > 1 && t.stride(1) != 1) throw Failure{std::string(name) + ": the values of a row have to be contiguous"};
    return rows > 1 ? t.stride(0) : width;
}
// The library counts in 32 bits: a size or number beyond them must not come out as another one.
int narrow(const char *name, int64_t v) {
    if (v < INT32_MIN || v > INT32_MAX) throw Failure{std::string(name) + " is out of range: " + std::to_string(v)};
    return (int)v;
}
void *current_stream() { return at::cuda::getCurrentCUDAStream(c10::cuda::current_device()).stream(); }
unsigned *status_of(const at::Tensor *t) {
    if (!t) return nullptr;
    if (t->nbytes() < 4 || t->element_size() != 4) throw Failure{"status: a 32-bit word expected"};
    return static_cast<unsigned *>(t->data_ptr());
}

struct KvCache {
    const at::Tensor &data, &scales, &tail_k, &tail_v;
    int64_t blocks, kv, block, hd, seqs;
    KvCache(PyObject *d, PyObject *s, PyObject *k, PyObject *v)
        : data(given(d, "data")), scales(given(s, "scales")), tail_k(given(k, "tail_k")), tail_v(given(v, "tail_v")) {
        if (data.dim() != 5 || data.size(3) != 2 || data.size(4) % 16 || tail_k.dim() != 4)
            throw Failure{"data: (n_blocks, n_kv, block/16, 2, 16*head_dim) uint8 and tail_k: (n_seqs, n_kv, block, head_dim) fp16 expected"};
        blocks = data.size(0); kv = data.size(1); block = data.size(2) * 16; hd = data.size(4) / 16; seqs = tail_k.size(0);
        expect("data", data, at::kByte, data.sizes());
        expect("scales", scales, at::kFloat, {blocks, kv, 4});
        expect("tail_k", tail_k, at::kHalf, {seqs, kv, block, hd}, false);
        expect("tail_v", tail_v, at::kHalf, {seqs, kv, block / 2, hd, 2}, false);
        if (hd == 0 || blocks == 0 || seqs == 0 || kv == 0) throw Failure{"an empty cache"};
        // one sequence's part is contiguous
        if (tail_k.stride(3) != 1 || tail_k.stride(2) != hd || (kv > 1 && tail_k.stride(1) != block * hd) || tail_v.stride(4) != 1 || tail_v.stride(3) != 2 ||
            (block > 2 && tail_v.stride(2) != 2 * hd) || (kv > 1 && tail_v.stride(1) != block * hd))
            throw Failure{"the tails of one sequence have to be contiguous"};
        if (seqs > 1 && (tail_k.stride(0) < kv * block * hd || tail_v.stride(0) < kv * block * hd)) throw Failure{"the tails of two sequences overlap"};
    }
    int n_seqs() const { return narrow("n_seqs", seqs); }
    int n_blocks() const { return narrow("n_blocks", blocks); }
    int n_kv() const { return narrow("n_kv", kv); }
    int head_dim() const { return narrow("head_dim", hd); }
    int block_size() const { return narrow("block", block); }
    long stride_k() const { return seqs > 1 ? tail_k.stride(0) : 0; }
    long stride_v() const { return seqs > 1 ? tail_v.stride(0) : 0; }
    const at::Tensor *list[4] = {&data, &scales, &tail_k, &tail_v};
};

template <class F>
PyObject *launching(Py_ssize_t nargs, Py_ssize_t want, const char *name, F body) {
    return guarded([&]() -> PyObject * {
        if (nargs != want) throw Failure{std::string(name) + " takes " + std::to_string(want) + " arguments"};
        return PyLong_FromLong(body());
    });
}

PyObject *py_kv_plan(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return launching(nargs, 10, "kv_plan", [&] {
        const at::Tensor &tables = given(a[0], "tables"), &lengths = given(a[1], "lengths"), &fresh = given(a[2], "new"),
                         &lengths_out = given(a[3], "lengths_out"), &runs = given(a[4], "runs"), &n_runs = given(a[5], "n_runs"),
                         *status = maybe(a[9], "status");
        const long n_blocks = int_arg(a[6]), block = int_arg(a[7]), n_tokens = int_arg(a[8]);
        here({&tables, &lengths, &fresh, &lengths_out, &runs, &n_runs, status});
        if (tables.dim() != 2 || runs.dim() != 2) throw Failure{"tables: (n_seqs, max_blocks), runs: (max_runs, 8) expected"};
        const int64_t S = tables.size(0);
        expect("tables", tables, at::kInt, {S, tables.size(1)});
        expect("lengths", lengths, at::kInt, {S});
        expect("new", fresh, at::kInt, {S});
        expect("lengths_out", lengths_out, at::kInt, {S});
        expect("runs", runs, at::kInt, {runs.size(0), 8});
        expect("n_runs", n_runs, at::kInt, {1});
        check(qtip_kv_plan(static_cast<int *>(tables.data_ptr()), static_cast<const int *>(lengths.data_ptr()), static_cast<const int *>(fresh.data_ptr()),
                           static_cast<int *>(lengths_out.data_ptr()), static_cast<int *>(runs.data_ptr()), static_cast<int *>(n_runs.data_ptr()), narrow("n_seqs", S),
                           narrow("max_blocks", tables.size(1)), narrow("n_blocks", n_blocks), narrow("block", block), narrow("n_tokens", n_tokens),
                           (int)std::min<int64_t>(runs.size(0), INT32_MAX), status_of(status),
                           current_stream()),
              "qtip_kv_plan");
        return 1L;
    });
}

PyObject *py_rope_kv_append_paged(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return launching(nargs, 13, "rope_kv_append_paged", [&] {
        const at::Tensor &q_out = given(a[0], "q_out"), &q = given(a[1], "q"), &k = given(a[2], "k"), &v = given(a[3], "v");
        const KvCache c(a[4], a[5], a[6], a[7]);
        const at::Tensor &runs = given(a[8], "runs"), &n_runs = given(a[9], "n_runs"), &inv_freq = given(a[10], "inv_freq"), *status = maybe(a[12], "status");
        here({&q_out, &q, &k, &v, c.list[0], c.list[1], c.list[2], c.list[3], &runs, &n_runs, &inv_freq, status});
        if (q.dim() != 2 || runs.dim() != 2) throw Failure{"q: (n_tokens, n_heads*head_dim), runs: (max_runs, 8) expected"};
        const int64_t T = q.size(0), width = q.size(1);
        expect("runs", runs, at::kInt, {runs.size(0), 8});
        expect("n_runs", n_runs, at::kInt, {1});
        expect("inv_freq", inv_freq, at::kDouble, {c.hd / 2});
        if (width % c.hd) throw Failure{"q: a multiple of head_dim values in a row expected"};
        const long sqo = rows_of("q_out", q_out, T, width), sq = rows_of("q", q, T, width), sk = rows_of("k", k, T, c.kv * c.hd), sv = rows_of("v", v, T, c.kv * c.hd);
        check(qtip_rope_kv_append_paged(q_out.data_ptr(), sqo, q.data_ptr(), sq, k.data_ptr(), sk, v.data_ptr(), sv, c.data.data_ptr(),
                                        static_cast<float *>(c.scales.data_ptr()), c.tail_k.data_ptr(), c.stride_k(), c.tail_v.data_ptr(), c.stride_v(),
                                        static_cast<const int *>(runs.data_ptr()), static_cast<const int *>(n_runs.data_ptr()),
                                        (int)std::min<int64_t>(runs.size(0), INT32_MAX), static_cast<const double *>(inv_freq.data_ptr()), narrow("n_tokens", T),
                                        c.n_seqs(), narrow("n_heads", width / c.hd), c.n_kv(), c.head_dim(), c.n_blocks(), c.block_size(), narrow("kind", int_arg(a[11])),
                                        status_of(status), current_stream()),
              "qtip_rope_kv_append_paged");
        return 1L;
    });
}

PyObject *py_attn_decode_paged(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return launching(nargs, 11, "attn_decode_paged", [&] {
        const at::Tensor &out = given(a[0], "out"), &q = given(a[1], "q");
        const KvCache c(a[2], a[3], a[4], a[5]);
        const at::Tensor &tables = given(a[6], "tables"), &lengths = given(a[7], "lengths"), *workspace = maybe(a[9], "workspace"),
                         *status = maybe(a[10], "status");
        here({&out, &q, c.list[0], c.list[1], c.list[2], c.list[3], &tables, &lengths, workspace, status});
        if (q.dim() != 2 || tables.dim() != 2 || q.size(1) % c.hd) throw Failure{"q: (n_seqs, n_heads*head_dim), tables: (n_seqs, max_blocks) expected"};
        const int64_t width = q.size(1), n_heads = width / c.hd;
        expect("tables", tables, at::kInt, {c.seqs, tables.size(1)});
        expect("lengths", lengths, at::kInt, {c.seqs});
        const long so = rows_of("out", out, c.seqs, width), sq = rows_of("q", q, c.seqs, width);
        const int heads = narrow("n_heads", n_heads);
        at::Tensor own;                  // from torch's allocator: of the stream, or of the graph that is being captured
        if (!workspace) {
            const size_t need = qtip_attn_paged_workspace_bytes(c.n_seqs(), heads, c.n_kv(), c.head_dim());
            own = at::empty({(int64_t)std::max<size_t>(need, 1)}, q.options().dtype(at::kByte));
            workspace = &own;
        }
        check(qtip_attn_decode_paged(out.data_ptr(), so, q.data_ptr(), sq, c.data.data_ptr(), static_cast<const float *>(c.scales.data_ptr()),
                                     c.tail_k.data_ptr(), c.stride_k(), c.tail_v.data_ptr(), c.stride_v(), static_cast<const int *>(tables.data_ptr()),
                                     static_cast<const int *>(lengths.data_ptr()), c.n_seqs(), heads, c.n_kv(), c.head_dim(), narrow("max_blocks", tables.size(1)),
                                     c.n_blocks(), c.block_size(), narrow("kind", int_arg(a[8])), workspace->data_ptr(), workspace->nbytes(), status_of(status),
                                     current_stream()),
              "qtip_attn_decode_paged");
        return 1L;
    });
}

PyObject *py_beam_select(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return launching(nargs, 8, "beam_select", [&] {
        const at::Tensor &tokens = given(a[0], "tokens"), &parents = given(a[1], "parents"), &scores = given(a[2], "scores"), &logits = given(a[3], "logits"),
                         &prev_scores = given(a[4], "prev_scores"), *prev_tokens = maybe(a[5], "prev_tokens"), *status = maybe(a[7], "status");
        here({&tokens, &parents, &scores, &logits, &prev_scores, prev_tokens, status});
        if (tokens.dim() != 2 || logits.dim() != 2) throw Failure{"tokens: (groups, width), logits: (groups * width, vocab) expected"};
        const int64_t G = tokens.size(0), W = tokens.size(1), vocab = logits.size(1);
        expect("tokens", tokens, at::kLong, {G, W});
        expect("parents", parents, at::kInt, {G, W});
        expect("scores", scores, at::kFloat, {G, W});
        expect("prev_scores", prev_scores, at::kFloat, {G, W});
        if (prev_tokens) expect("prev_tokens", *prev_tokens, at::kLong, {G, W});
        if (logits.size(0) != G * W || (vocab > 1 && logits.stride(1) != 1)) throw Failure{"logits: (groups * width, vocab) with contiguous rows expected, not " + text(logits.sizes())};
        const long long eos = PyLong_AsLongLong(a[6]);
        if (eos == -1 && PyErr_Occurred()) throw Failure{""};
        check(qtip_beam_select(reinterpret_cast<long long *>(tokens.data_ptr()), static_cast<int *>(parents.data_ptr()), static_cast<float *>(scores.data_ptr()),
                               logits.data_ptr(), dtype_id(logits), G * W > 1 ? logits.stride(0) : vocab, static_cast<const float *>(prev_scores.data_ptr()),
                               prev_tokens ? reinterpret_cast<const long long *>(prev_tokens->data_ptr()) : nullptr, narrow("groups", G), narrow("width", W), narrow("vocab", vocab), eos,
                               status_of(status), current_stream()),
              "qtip_beam_select");
        return 1L;
    });
}

PyObject *py_beam_reorder(PyObject *, PyObject *const *a, Py_ssize_t nargs) {
    return launching(nargs, 4, "beam_reorder", [&] {
        const at::Tensor &parents = given(a[1], "parents"), *lengths = maybe(a[2], "lengths"), *status = maybe(a[3], "status");
        here({&parents, lengths, status});
        if (parents.dim() != 2) throw Failure{"parents: (groups, width) expected"};
        const int64_t G = parents.size(0), W = parents.size(1);
        expect("parents", parents, at::kInt, {G, W});
        if (lengths) expect("lengths", *lengths, at::kInt, {G * W});
        if (!PyList_Check(a[0]) && !PyTuple_Check(a[0])) throw Failure{"states: a list of (tensor, tokens per row, modulus) expected"};
        const Py_ssize_t n = PySequence_Fast_GET_SIZE(a[0]);
        if (n < 1 || n > 8) throw Failure{"1 to 8 states expected, not " + std::to_string(n)};
        qtip_beam_state list[8];
        for (Py_ssize_t i = 0; i < n; i++) {
            PyObject *s = PySequence_Fast_GET_ITEM(a[0], i);
            if (!PyTuple_Check(s) || PyTuple_GET_SIZE(s) != 3) throw Failure{"a state is (tensor, tokens per row, modulus)"};
            const at::Tensor &t = given(PyTuple_GET_ITEM(s, 0), "a state's tensor");
            here({&t});
            const long per_row = int_arg(PyTuple_GET_ITEM(s, 1)), mod = int_arg(PyTuple_GET_ITEM(s, 2));
            if (t.dim() != 4 || t.size(0) != G * W || t.numel() == 0) throw Failure{"a state is (" + std::to_string(G * W) + ", outer, rows, values), not " + text(t.sizes())};
            if ((t.size(3) > 1 && t.stride(3) != 1) || (t.size(2) > 1 && t.stride(2) != t.size(3))) throw Failure{"the rows of a state have to be contiguous"};
            const long size = (long)t.element_size(), piece = t.size(2) * t.size(3) * size;
            if (per_row < 1 || per_row > INT32_MAX || mod < 0 || mod > INT32_MAX || t.size(1) > INT32_MAX || t.size(2) > INT32_MAX || t.size(3) * size > INT32_MAX)
                throw Failure{"a state's tokens per row, modulus or sizes are out of range"};
            list[i].base = t.data_ptr();
            list[i].outer_stride = t.size(1) > 1 ? t.stride(1) * size : piece;
            list[i].seq_stride = G * W > 1 ? t.stride(0) * size : list[i].outer_stride * t.size(1);
            list[i].outer = (int)t.size(1);
            list[i].rows = (int)t.size(2);
            list[i].row_bytes = (int)(t.size(3) * size);
            list[i].per_row = (int)per_row;
            list[i].mod = (int)mod;
        }
        check(qtip_beam_reorder(list, (int)n, static_cast<const int *>(parents.data_ptr()), lengths ? static_cast<const int *>(lengths->data_ptr()) : nullptr,
                                narrow("groups", G), narrow("width", W), status_of(status), current_stream()),
              "qtip_beam_reorder");
        return 1L;
    });
}

PyMethodDef kMethods[] = {
    {"linear_forward", (PyCFunction)(void *)py_linear_forward, METH_FASTCALL, "one QTIP linear on the current stream"},
    {"matvec_workspace", (PyCFunction)(void *)py_matvec_workspace, METH_FASTCALL, "scratch of the fused matvec"},
    {"gemm_status", (PyCFunction)(void *)py_gemm_status, METH_FASTCALL, "status word of the decompress-GEMM"},
    {"kv_plan", (PyCFunction)(void *)py_kv_plan, METH_FASTCALL, "where new tokens of a batch go"},
    {"rope_kv_append_paged", (PyCFunction)(void *)py_rope_kv_append_paged, METH_FASTCALL, "rotary embedding and append to the 8-bit cache"},
    {"attn_decode_paged", (PyCFunction)(void *)py_attn_decode_paged, METH_FASTCALL, "attention over the 8-bit cache"},
    {"beam_select", (PyCFunction)(void *)py_beam_select, METH_FASTCALL, "the best continuations of groups of beams"},
    {"beam_reorder", (PyCFunction)(void *)py_beam_reorder, METH_FASTCALL, "states follow their beams"},
    {nullptr, nullptr, 0, nullptr}};
PyModuleDef kModule = {PyModuleDef_HEAD_INIT, "_host", "native host path of qtip_b200", -1, kMethods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__host() { return PyModule_Create(&kModule); }
