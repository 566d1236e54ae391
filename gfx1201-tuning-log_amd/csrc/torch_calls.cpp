// The torch side of the append and visible-key attention calls: checks of the tensors and the call, in one Python call.
//
// These calls take a dozen tensors, of which five properties each have to be read.  Read one by one from Python that is
// 4 to 6 us a call, as long as the smallest kernels run; here it is a fraction of one.  No device code: the module
// packs a call's arguments into 64-bit words for fp8kv_call (fp8kv_amd.h), whose address it is given.
// Everything here runs under the GIL; a refused tensor raises ValueError, a refused call returns its status.
#include <torch/csrc/autograd/python_variable.h>

#include <cstdint>
#include <cstring>
#include <string>

namespace {

int (*g_call)(int, const int64_t*, int) = nullptr;
int (*g_splits)(int, int, int, int, int, int) = nullptr;
size_t (*g_scratch_bytes)(int, int, int, int, int) = nullptr;
unsigned long long (*g_capture)(void*) = nullptr;

struct Refused {
    std::string what;
};
struct PythonError {};                 // an exception is set already

[[noreturn]] void refuse(const std::string& what) { throw Refused{what}; }

const at::Tensor& tensor(PyObject* o, const char* name)
{
    if (!THPVariable_Check(o)) refuse(std::string(name) + " must be a tensor");
    return THPVariable_Unpack(o);
}

int64_t integer(PyObject* o)
{
    PyObject* i = PyNumber_Index(o);
    if (!i) throw PythonError{};
    const int64_t v = PyLong_AsLongLong(i);
    Py_DECREF(i);
    if (v == -1 && PyErr_Occurred()) throw PythonError{};
    return v;
}

bool is_e4m3(at::ScalarType t) { return t == at::kFloat8_e4m3fn || t == at::kByte; }
int64_t address(const at::Tensor& t) { return reinterpret_cast<int64_t>(t.data_ptr()); }

struct Words {
    int64_t w[48];
    int n = 0;
    void put(int64_t x) { w[n++] = x; }
    void put(const at::Tensor& t) { put(address(t)); }
    void put_float(double x)
    {
        const float f = (float)x;
        uint32_t b;
        std::memcpy(&b, &f, sizeof b);
        put((int64_t)b);
    }
};

// A bf16 [T, H, D] tensor whose heads are contiguous.
struct Rows {
    int64_t T, H, D, stride;
    int dev;
};

Rows rows(const at::Tensor& t, const char* name, const Rows* like = nullptr)
{
    if (!(t.dim() == 3 && t.scalar_type() == at::kBFloat16 && t.get_device() >= 0 && t.stride(2) == 1 &&
          (t.stride(1) == t.size(2) || t.size(1) == 1)))
        refuse(std::string(name) + " must be a bf16 device tensor [T, heads, D] with contiguous heads");
    Rows r{t.size(0), t.size(1), t.size(2), 0, (int)t.get_device()};
    r.stride = r.T > 1 ? t.stride(0) : r.H * r.D;             // a single row's stride says nothing
    if (like && !(r.T == like->T && r.H == like->H && r.D == like->D && r.dev == like->dev))
        refuse(std::string(name) + " must have the shape and device that go with the other rows");
    return r;
}

struct Caches {
    bool bf16;
    int64_t NB, PBLK, HKV;
};

Caches caches(Words& w, const at::Tensor& k, const at::Tensor& v, int dev, int64_t D, bool allow_bf16)
{
    const bool bf16 = k.scalar_type() == at::kBFloat16 && v.scalar_type() == at::kBFloat16;
    if (!(bf16 && allow_bf16) && !(is_e4m3(k.scalar_type()) && is_e4m3(v.scalar_type())))
        refuse(std::string("caches must both be e4m3 (float8_e4m3fn or raw uint8)") + (allow_bf16 ? " or both bf16" : ""));
    if (!(k.dim() == 4 && k.sizes() == v.sizes() && k.size(3) == D && k.stride(3) == 1 && v.stride(3) == 1))
        refuse("caches must be [NB, PBLK, HKV, D] of one shape, contiguous along the head size that q and key have");
    if (!(k.get_device() == dev && v.get_device() == dev)) refuse("tensors on different devices");
    w.put(k);
    w.put(v);
    for (int i = 0; i < 3; ++i) w.put(k.stride(i));
    for (int i = 0; i < 3; ++i) w.put(v.stride(i));
    return {bf16, k.size(0), k.size(1), k.size(2)};
}

void vector(Words& w, PyObject* o, const char* name, at::ScalarType type, int64_t n, int dev)
{
    const at::Tensor& t = tensor(o, name);
    if (!(t.scalar_type() == type && t.dim() == 1 && t.size(0) == n && t.is_contiguous() && t.get_device() == dev))
        refuse(std::string(name) + " must be a contiguous " + c10::toString(type) + " tensor [" + std::to_string(n) + "] on device " +
               std::to_string(dev));
    w.put(t);
}

// The number of sequences.
int64_t sequences(Words& w, PyObject* starts, PyObject* lens, const at::Tensor& table, int dev)
{
    if (!(table.dim() == 2 && table.scalar_type() == at::kInt && (table.size(1) <= 1 || table.stride(1) == 1) &&
          table.get_device() == dev))
        refuse("block_table must be an int32 tensor [NS, max_blocks] on device " + std::to_string(dev) + ", rows contiguous");
    const int64_t NS = table.size(0);
    vector(w, starts, "query_start_loc", at::kInt, NS + 1, dev);
    vector(w, lens, "seq_lens", at::kInt, NS, dev);
    w.put(table);
    w.put(table.stride(0));
    return NS;
}

void kv_scales(Words& w, PyObject* o, const Caches& c, int dev)
{
    const at::Tensor& t = tensor(o, "kv_scales");
    if (!((t.scalar_type() == at::kByte || t.scalar_type() == at::kFloat8_e8m0fnu) && t.dim() == 4 && t.size(0) == c.NB &&
          t.size(1) == c.PBLK / 16 && t.size(2) == c.HKV && t.size(3) == 2 && t.is_contiguous() && t.get_device() == dev))
        refuse("kv_scales must be contiguous uint8 (e8m0) [" + std::to_string(c.NB) + ", " + std::to_string(c.PBLK / 16) + ", " +
               std::to_string(c.HKV) + ", 2] on device " + std::to_string(dev));
    w.put(t);
}

void scale(Words& w, PyObject* o, const char* name, int dev)
{
    if (o == Py_None) refuse(std::string("e4m3 caches need ") + name);
    const at::Tensor& t = tensor(o, name);
    if (!(t.scalar_type() == at::kFloat && t.numel() >= 1 && t.get_device() == dev)) refuse("k/v scales must be fp32 device tensors");
    w.put(t);
}

int call(int64_t entry, Words& w, PyObject* stream)
{
    w.put(integer(stream));
    return g_call((int)entry, w.w, w.n);
}

// Queries, keys, values, caches and rotation of the append calls.
struct Append {
    Rows key;
    int64_t HQ;
    Caches c;
};

Append append_lead(Words& w, PyObject* const* a, bool allow_bf16)
{
    // q, key, value, k_cache, v_cache, positions, cos_sin, q_out, interleaved
    const at::Tensor &key = tensor(a[1], "key"), &value = tensor(a[2], "value");
    Append r{rows(key, "key"), 0, {}};
    const Rows& k = r.key;
    const Rows v = rows(value, "value", &k);
    if (a[0] != Py_None) {
        const at::Tensor &q = tensor(a[0], "q"), &out = tensor(a[7], "q_out");
        const Rows qr = rows(q, "q");
        if (!(qr.T == k.T && qr.D == k.D && qr.dev == k.dev)) refuse("q must be [T, HQ, D] of key's T, D and device");
        const Rows o = rows(out, "q_out", &qr);
        r.HQ = qr.H;
        w.put(q);
        w.put(qr.stride);
        w.put(out);
        w.put(o.stride);
    } else {
        if (a[7] != Py_None) refuse("q_out without q");
        for (int i = 0; i < 4; ++i) w.put(0);
    }
    w.put(key);
    w.put(k.stride);
    w.put(value);
    w.put(v.stride);
    r.c = caches(w, tensor(a[3], "k_cache"), tensor(a[4], "v_cache"), k.dev, k.D, allow_bf16);
    if (r.c.HKV != k.H) refuse("caches must be [NB, PBLK, HKV, D] matching key");
    if (a[6] != Py_None) {
        const at::Tensor& t = tensor(a[6], "cos_sin");
        const bool b16 = t.scalar_type() == at::kBFloat16;
        if (!(t.dim() == 2 && (b16 || t.scalar_type() == at::kFloat) && t.stride(1) == 1 && t.get_device() == k.dev))
            refuse("cos_sin must be fp32 or bf16 [positions, rotary_dim] on key's device");
        if (a[5] == Py_None) refuse("cos_sin without positions");
        const int interleaved = PyObject_IsTrue(a[8]);
        if (interleaved < 0) throw PythonError{};
        vector(w, a[5], "positions", at::kLong, k.T, k.dev);
        w.put(t);
        w.put(t.size(0) > 1 ? t.stride(0) : t.size(1));
        w.put(b16 ? 1 : 0);
        w.put(t.size(0));
        w.put(t.size(1));
        w.put(interleaved);
    } else {
        for (int i = 0; i < 7; ++i) w.put(0);
    }
    return r;
}

void append_tail(Words& w, const Append& r)
{
    w.put(r.key.T);
    w.put(r.HQ);
    w.put(r.key.H);
    w.put(r.key.D);
    w.put(r.c.PBLK);
    w.put(r.c.NB);
}

// entry of e4m3, entry of bf16, stream, [append_lead], slot_mapping, k_scale, v_scale
int rope_append(PyObject* const* a)
{
    Words w;
    const Append r = append_lead(w, a + 3, true);
    vector(w, a[12], "slot_mapping", at::kLong, r.key.T, r.key.dev);
    if (!r.c.bf16) {
        scale(w, a[13], "k_scale", r.key.dev);
        scale(w, a[14], "v_scale", r.key.dev);
    }
    if (r.key.T == 0) return 0;
    append_tail(w, r);
    return call(integer(a[r.c.bf16 ? 1 : 0]), w, a[2]);
}

// entry, stream, [append_lead], kv_scales, query_start_loc, seq_lens, block_table
int rope_append_blk(PyObject* const* a)
{
    Words w;
    const Append r = append_lead(w, a + 2, false);
    kv_scales(w, a[11], r.c, r.key.dev);
    const at::Tensor& table = tensor(a[14], "block_table");
    const int64_t NS = sequences(w, a[12], a[13], table, r.key.dev);
    if (r.key.T == 0 || NS == 0) return 0;
    w.put(table.size(1));
    w.put(NS);
    append_tail(w, r);
    return call(integer(a[0]), w, a[1]);
}

struct Attention {
    Rows q;
    Caches c;
    int64_t NS;
};

// entries of e4m3 and bf16 caches (or of block-scaled ones and None), stream,
// q, k_cache, v_cache, out, starts, seq_lens, block_table, k_scale, v_scale (kv_scales, None), sm_scale, window, sinks
Attention attention_lead(Words& w, PyObject* const* a, bool blk)
{
    const at::Tensor &q = tensor(a[3], "q"), &out = tensor(a[6], "out");
    // the calls write the rows of q in out; looked at first, which needs no device
    if (q.dim() > 0 && out.dim() > 0 && out.size(0) < q.size(0))
        refuse("out has " + std::to_string(out.size(0)) + " rows, fewer than q's " + std::to_string(q.size(0)));
    Attention r{rows(q, "q"), {}, 0};
    const Rows o = rows(out, "out");
    if (!(o.H == r.q.H && o.D == r.q.D && o.dev == r.q.dev)) refuse("out must be [T, HQ, D] of q's heads and device");
    w.put(q);
    w.put(r.q.stride);
    r.c = caches(w, tensor(a[4], "k_cache"), tensor(a[5], "v_cache"), r.q.dev, r.q.D, !blk);
    w.put(out);
    w.put(o.stride);
    r.NS = sequences(w, a[7], a[8], tensor(a[9], "block_table"), r.q.dev);
    if (integer(a[13]) < 0 || integer(a[14]) < 0) refuse("window and sinks must not be negative");
    if (blk) {
        kv_scales(w, a[10], r.c, r.q.dev);
    } else if (!r.c.bf16) {
        scale(w, a[10], "k_scale", r.q.dev);
        scale(w, a[11], "v_scale", r.q.dev);
    }
    const double sm = PyFloat_AsDouble(a[12]);
    if (sm == -1.0 && PyErr_Occurred()) throw PythonError{};
    w.put_float(sm);
    w.put(r.NS);
    w.put(r.q.H);
    w.put(r.c.HKV);
    w.put(r.q.D);
    w.put(r.c.PBLK);
    return r;
}

// [attention_lead], num_splits or None, max_seq_len (0: not known), scratch or None, whether it is for this call.
// A positive result is a status; a negative one the bytes of scratch that the call needs, and has not been given: under
// capture, the buffer that the stream's eager calls use (the last argument false) is not taken.
int64_t decode(PyObject* const* a, bool blk)
{
    Words w;
    const Attention r = attention_lead(w, a, blk);
    if (r.NS == 0) return 0;
    auto size = [](int64_t x) { return (int)(x < 1 << 30 ? x : 1 << 30); };
    const int64_t longest = integer(a[16]), window = integer(a[13]), sinks = integer(a[14]);
    const int64_t splits = a[15] != Py_None ? integer(a[15])
                                            : g_splits(size(r.NS), size(r.c.HKV), size(longest), size(window), size(sinks), r.c.bf16);
    // more splits than 256 are for the call to refuse
    const int64_t need = splits > 1 && splits <= 256 ? (int64_t)g_scratch_bytes(size(r.NS), size(r.q.H), size(r.c.HKV), (int)r.q.D, size(splits)) : 0;
    int64_t where = 0, bytes = 0;
    const bool given = PyObject_IsTrue(a[18]) == 1;
    if (need > 0 && !given && g_capture(reinterpret_cast<void*>(integer(a[2])))) return -need;
    if (a[17] != Py_None) {
        const at::Tensor& t = tensor(a[17], "scratch");
        if (t.get_device() == r.q.dev && t.is_contiguous()) {
            where = address(t);
            bytes = (int64_t)t.nbytes();
        }
        if (given && (where == 0 || bytes < need))
            refuse("scratch needs " + std::to_string(need) + " contiguous bytes on device " + std::to_string(r.q.dev));
    }
    if (bytes < need) return -need;
    w.put(splits);
    w.put(where);
    w.put(bytes);
    w.put(window);
    w.put(sinks);
    w.put(longest);
    return call(integer(a[r.c.bf16 ? 1 : 0]), w, a[2]);
}

// [attention_lead], max_query_len
int prefill(PyObject* const* a, bool blk)
{
    Words w;
    const Attention r = attention_lead(w, a, blk);
    if (r.NS == 0 || r.q.T == 0) return 0;
    w.put(integer(a[13]));
    w.put(integer(a[14]));
    w.put(integer(a[15]));
    w.put(r.q.T);
    return call(integer(a[r.c.bf16 ? 1 : 0]), w, a[2]);
}

template <typename F>
PyObject* guarded(Py_ssize_t given, Py_ssize_t want, F f)
{
    if (given != want) {
        PyErr_Format(PyExc_TypeError, "%zd arguments, not %zd", given, want);
        return nullptr;
    }
    try {
        return PyLong_FromLongLong((long long)f());
    } catch (const Refused& e) {
        PyErr_SetString(PyExc_ValueError, e.what.c_str());
    } catch (const PythonError&) {
    } catch (const std::exception& e) {
        PyErr_SetString(PyExc_RuntimeError, e.what());
    }
    return nullptr;
}

PyObject* py_rope_append(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 15, [&] { return rope_append(a); }); }
PyObject* py_rope_append_blk(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 15, [&] { return rope_append_blk(a); }); }
PyObject* py_decode(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 19, [&] { return decode(a, false); }); }
PyObject* py_decode_blk(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 19, [&] { return decode(a, true); }); }
PyObject* py_prefill(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 16, [&] { return prefill(a, false); }); }
PyObject* py_prefill_blk(PyObject*, PyObject* const* a, Py_ssize_t n) { return guarded(n, 16, [&] { return prefill(a, true); }); }

// Addresses of fp8kv_call, fp8kv_decode_visible_splits, fp8kv_decode_scratch_bytes and fp8kv_stream_capture.
PyObject* py_bind(PyObject*, PyObject* const* a, Py_ssize_t n)
{
    return guarded(n, 4, [&] {
        g_call = reinterpret_cast<decltype(g_call)>(integer(a[0]));
        g_splits = reinterpret_cast<decltype(g_splits)>(integer(a[1]));
        g_scratch_bytes = reinterpret_cast<decltype(g_scratch_bytes)>(integer(a[2]));
        g_capture = reinterpret_cast<decltype(g_capture)>(integer(a[3]));
        return 0;
    });
}

#define FP8KV_METHOD(name, f) {name, reinterpret_cast<PyCFunction>(reinterpret_cast<void (*)()>(f)), METH_FASTCALL, nullptr}
PyMethodDef g_methods[] = {FP8KV_METHOD("bind", py_bind),
                           FP8KV_METHOD("rope_append", py_rope_append),
                           FP8KV_METHOD("rope_append_blk", py_rope_append_blk),
                           FP8KV_METHOD("decode", py_decode),
                           FP8KV_METHOD("decode_blk", py_decode_blk),
                           FP8KV_METHOD("prefill", py_prefill),
                           FP8KV_METHOD("prefill_blk", py_prefill_blk),
                           {nullptr, nullptr, 0, nullptr}};
PyModuleDef g_module = {PyModuleDef_HEAD_INIT, "fp8kv_torch_calls", nullptr, -1, g_methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit_fp8kv_torch_calls() { return PyModule_Create(&g_module); }
