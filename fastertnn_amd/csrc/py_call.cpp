// The device entry points that a program calls once per layer or product, without ctypes: a CPython module over include/ftnn.h.
//
// Such a call is two launches at most, 2.2 us of host time each, and on the device it takes 3 to 7 us; ctypes (0.9 us for the
// arguments of a layer) and the checks on its tensors in Python (1.1 us for five) come on top of that, call after call.  Here
// both take 0.2 us.  A call queued behind others, before and now: TBN layer 8 x 128 x 28 x 28 9.8 -> 8.0 us, TNN 256 x 56 x 56
// 9.9 -> 7.9, fully connected layers of 0.5 M weights 9.2 -> 5.9, TNN product 256 x 256 x 4096 5.7 -> 3.7.
//
// Every function takes the arguments of its wrapper in fastertnn_amd/lib.py and returns the library's status, or None where
// an argument is not of the plain kind that it reads itself (an int, a float, a contiguous torch.Tensor on the GPU that is no
// subclass): the wrapper then goes on through ctypes, which converts or refuses it as it always has.
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <ATen/ops/empty.h>
#include <c10/hip/HIPStream.h>
#include <torch/csrc/Dtype.h>
#include <torch/csrc/autograd/python_variable.h>

#include <climits>

#include "../../include/ftnn.h"

namespace {

struct Args {
    PyObject* const* v;
    bool good = true;   // every argument so far was a plain one

    int i(int k) {
        if (!PyLong_CheckExact(v[k])) return bad();
        int over = 0;
        const long x = PyLong_AsLongAndOverflow(v[k], &over);
        return over || x < INT_MIN || x > INT_MAX ? bad() : (int)x;
    }
    float f(int k) {
        if (PyFloat_CheckExact(v[k])) return (float)PyFloat_AS_DOUBLE(v[k]);
        return (float)i(k);
    }
    // data of a contiguous device tensor
    char* any(int k, int64_t* bytes = nullptr) {
        if (!THPVariable_CheckExact(v[k])) return bad(), nullptr;
        const at::Tensor& t = THPVariable_Unpack(v[k]);
        if (!t.is_cuda() || !t.is_contiguous()) return bad(), nullptr;
        if (bytes) *bytes = t.numel() * (int64_t)t.element_size();
        return static_cast<char*>(t.data_ptr());
    }
    float* f32(int k) {
        if (!THPVariable_CheckExact(v[k]) || THPVariable_Unpack(v[k]).scalar_type() != at::kFloat) return bad(), nullptr;
        return reinterpret_cast<float*>(any(k));
    }
    const int64_t* words(int k) { return reinterpret_cast<const int64_t*>(any(k)); }
    // N, C, H, W of a layer's input
    bool nchw(int k, int d[4]) {
        if (!THPVariable_CheckExact(v[k])) return bad(), false;
        const at::Tensor& t = THPVariable_Unpack(v[k]);
        if (t.dim() != 4) return bad(), false;
        for (int j = 0; j < 4; j++) {
            if (t.size(j) > INT_MAX) return bad(), false;
            d[j] = (int)t.size(j);
        }
        return true;
    }
    int bad() {
        good = false;
        return 0;
    }
};

// fn(arguments, stream) with N arguments, the lock of the interpreter released around the library
template <Py_ssize_t N, typename F>
PyObject* call(PyObject* const* v, Py_ssize_t n, F&& read) {
    if (n != N) Py_RETURN_NONE;
    int rc = 0;
    try {
        Args a{v};
        auto fn = read(a);
        if (!a.good) Py_RETURN_NONE;
        void* stream = c10::hip::getCurrentHIPStream().stream();
        Py_BEGIN_ALLOW_THREADS
        rc = fn(stream);
        Py_END_ALLOW_THREADS
    } catch (...) {   // a tensor without storage, say: the wrapper meets it again
        Py_RETURN_NONE;
    }
    return PyLong_FromLong(rc);
}

// typ, a, b, n, oh, ow, kn, k, alpha, k_unpack, out
PyObject* mm(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<11>(v, n, [](Args& r) {
        return [typ = r.i(0), a = r.words(1), b = r.words(2), n = r.i(3), oh = r.i(4), ow = r.i(5), kn = r.i(6), k = r.i(7),
                alpha = r.f(8), ku = r.i(9), out = r.f32(10)](void* st) { return ftnn_mm(typ, a, b, n, oh, ow, kn, k, ku, alpha, out, st); };
    });
}

// engine, typ, a, b, n, oh, ow, kn, k, alpha, k_unpack, out, scratch
PyObject* mm_engine(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<13>(v, n, [](Args& r) {
        int64_t bytes = 0;
        void* scratch = r.any(12, &bytes);
        return [=, e = r.i(0), typ = r.i(1), a = r.words(2), b = r.words(3), n = r.i(4), oh = r.i(5), ow = r.i(6), kn = r.i(7), k = r.i(8),
                alpha = r.f(9), ku = r.i(10), out = r.f32(11)](void* st) {
            return ftnn_mm_engine(e, typ, a, b, n, oh, ow, kn, k, ku, alpha, out, scratch, bytes, st);
        };
    });
}

// engine, typ, a_exp, b_exp, n, oh, ow, kn, k, alpha, k_unpack, out
PyObject* mm_expanded(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<12>(v, n, [](Args& r) {
        return [e = r.i(0), typ = r.i(1), a = r.any(2), b = r.any(3), n = r.i(4), oh = r.i(5), ow = r.i(6), kn = r.i(7), k = r.i(8),
                alpha = r.f(9), ku = r.i(10), out = r.f32(11)](void* st) { return ftnn_mm_expanded(e, typ, a, b, n, oh, ow, kn, k, ku, alpha, out, st); };
    });
}

struct Layer {
    int typ, d[4], kn, kh, kw, pad, stride;
    const float *x, *thr;
    float alpha, *y;
};
// typ, x, thr, weights, kn, kh, kw, pad, stride, alpha, ..., out
Layer layer(Args& r, int out) {
    Layer l;
    r.nchw(1, l.d);
    l.typ = r.i(0), l.x = r.f32(1), l.thr = r.f32(2);
    l.kn = r.i(4), l.kh = r.i(5), l.kw = r.i(6), l.pad = r.i(7), l.stride = r.i(8), l.alpha = r.f(9), l.y = r.f32(out);
    return l;
}

// ..., scratch, out
PyObject* conv(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<12>(v, n, [](Args& r) {
        return [l = layer(r, 11), w = r.words(3), scratch = r.any(10)](void* st) {
            return ftnn_conv(l.typ, l.x, l.thr, w, l.d[0], l.d[1], l.d[2], l.d[3], l.kn, l.kh, l.kw, l.pad, l.pad, l.stride, l.stride, l.alpha,
                             scratch, l.y, st);
        };
    });
}
PyObject* conv_prepared(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<12>(v, n, [](Args& r) {
        return [l = layer(r, 11), w = r.any(3), scratch = r.any(10)](void* st) {
            return ftnn_conv_prepared(l.typ, l.x, l.thr, w, l.d[0], l.d[1], l.d[2], l.d[3], l.kn, l.kh, l.kw, l.pad, l.pad, l.stride, l.stride,
                                      l.alpha, scratch, l.y, st);
        };
    });
}
// ..., out
PyObject* conv_static(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<11>(v, n, [](Args& r) {
        return [l = layer(r, 10), w = r.words(3)](void* st) {
            return ftnn_conv_static(l.typ, l.x, l.thr, w, l.d[0], l.d[1], l.d[2], l.d[3], l.kn, l.kh, l.kw, l.pad, l.pad, l.stride, l.stride,
                                    l.alpha, l.y, st);
        };
    });
}

// net handle, x, out, use_graph
PyObject* net_run(PyObject*, PyObject* const* v, Py_ssize_t n) {
    return call<4>(v, n, [](Args& r) {
        void* net = PyLong_CheckExact(r.v[0]) ? PyLong_AsVoidPtr(r.v[0]) : nullptr;
        if (!net) PyErr_Clear(), r.bad();
        return [net, x = r.f32(1), out = r.f32(2), graph = r.i(3)](void* st) { return ftnn_net_run(static_cast<ftnn_net_t*>(net), x, out, graph, st); };
    });
}

// ---- operators of token models.  These make the results that they are not given, and return them: a product of one token
// takes 15.8 us through ctypes, 5.6 here, of which the launch is 4.  What does not have the plain form that a wrapper asks for is left to the wrapper, which says why.

struct Tensors {
    bool good = true;
    int device = c10::hip::current_device();

    bool need(bool ok) { return good &= ok; }
    // of `dims` dimensions (any if negative) and type on the current device, its last dimension contiguous; none at all: an empty tensor
    const at::Tensor& get(PyObject* o, int dims, int dtype = -1) {
        static const at::Tensor none;
        if (!THPVariable_CheckExact(o)) return good = false, none;
        const at::Tensor& t = THPVariable_Unpack(o);
        if (!need(t.is_cuda() && t.device().index() == device && (dims < 0 || t.dim() == dims) && (dtype < 0 || (int)t.scalar_type() == dtype))) return none;
        if (t.dim() && !need(t.size(-1) <= 1 || t.stride(-1) == 1)) return none;
        return t;
    }
    // contiguous, of one dimension and n elements
    void* flat(PyObject* o, at::ScalarType dtype, int64_t n) {
        const at::Tensor& t = get(o, 1, (int)dtype);
        return good && need(t.size(0) == n && t.is_contiguous()) ? t.data_ptr() : nullptr;
    }
    int64_t integer(PyObject* o) {
        if (!need(PyLong_CheckExact(o))) return 0;
        int over = 0;
        const long x = PyLong_AsLongAndOverflow(o, &over);
        return need(!over && x >= INT_MIN && x <= INT_MAX) ? x : 0;
    }
    int truth(PyObject* o) { return need(PyBool_Check(o)) && o == Py_True; }
    int type(at::ScalarType s) {
        need(s == at::kFloat || s == at::kHalf || s == at::kBFloat16);
        return s == at::kFloat ? FTNN_F32 : s == at::kHalf ? FTNN_F16 : FTNN_BF16;
    }
};
// values between rows of `least` or more; whatever torch says of a single row, and however wide that is
int64_t row_stride(const at::Tensor& t, int64_t least) { return t.size(0) > 1 ? t.stride(0) : least; }

// what fn() answers: the library's status where it refused, nothing where a tensor was not plain after all
template <typename F>
PyObject* answer(F&& fn) {
    try {
        return fn();
    } catch (...) {
        PyErr_Clear();
        Py_RETURN_NONE;
    }
}
// fn(stream) with the lock of the interpreter released.  What fn takes is plain values: a tensor's data are asked for before, since that may throw (a tensor
// without storage has the sizes of any other)
template <typename F>
int unlocked(F&& fn) {
    void* const stream = c10::hip::getCurrentHIPStream().stream();
    struct Released {
        PyThreadState* const state = PyEval_SaveThread();
        ~Released() { PyEval_RestoreThread(state); }
    } released;
    return fn(stream);
}

// x, q, scale
PyObject* quantize_rows_i8(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 3 || v[1] != Py_None || v[2] != Py_None) Py_RETURN_NONE;
    return answer([&]() -> PyObject* {
        Tensors r;
        const at::Tensor& x = r.get(v[0], 2);
        if (!r.good || !r.need(x.size(1) > 0 && x.size(1) <= INT_MAX)) Py_RETURN_NONE;
        const int dtype = r.type(x.scalar_type());
        if (!r.good) Py_RETURN_NONE;
        const int64_t rows = x.size(0), k = x.size(1), nb = ftnn_i8_row_bytes((int)k);
        const at::Tensor q = at::empty({rows, nb}, x.options().dtype(at::kChar)), s = at::empty({rows}, x.options().dtype(at::kFloat));
        const int rc = unlocked([dtype, xp = x.data_ptr(), x_stride = row_stride(x, k), rows, k, qp = static_cast<int8_t*>(q.data_ptr()), nb,
                                 sp = static_cast<float*>(s.data_ptr())](void* st) { return ftnn_quantize_rows_i8(dtype, xp, x_stride, rows, (int)k, qp, nb, sp, st); });
        if (rc) return PyLong_FromLong(rc);
        return Py_BuildValue("NN", THPVariable_Wrap(q), THPVariable_Wrap(s));
    });
}

// a, a_scale, b, b_scale, k, bias, dtype, out, and for packed rows n, ternary, scratch
PyObject* product(PyObject* const* v, bool packed) {
    return answer([&]() -> PyObject* {
        Tensors r;
        const at::Tensor &a = r.get(v[0], 2, (int)at::kChar), &b = packed ? r.get(v[2], -1, (int)at::kLong) : r.get(v[2], 2, (int)at::kChar);
        const int64_t k = r.integer(v[4]);
        if (!r.good || !r.need(k > 0)) Py_RETURN_NONE;
        const int64_t nb = ftnn_i8_row_bytes((int)k), m = a.size(0), n = packed ? r.integer(v[8]) : b.size(0);
        const int ternary = packed ? r.truth(v[9]) : 0;
        if (!r.good || !r.need(n > 0 && a.size(1) >= nb)) Py_RETURN_NONE;
        if (packed ? !r.need(b.is_contiguous() && k <= INT_MAX - 255 && b.numel() >= n * ftnn_row_words((int)k, 1, 1, ternary)) : !r.need(b.size(1) >= nb)) Py_RETURN_NONE;
        const float *sa = static_cast<float*>(r.flat(v[1], at::kFloat, m)), *sb = static_cast<float*>(r.flat(v[3], at::kFloat, n));
        const float* bias = v[5] == Py_None ? nullptr : static_cast<float*>(r.flat(v[5], at::kFloat, n));
        at::ScalarType type = at::kFloat;
        if (v[6] != Py_None) {
            if (!THPDtype_Check(v[6])) Py_RETURN_NONE;
            type = reinterpret_cast<THPDtype*>(v[6])->scalar_type;
        }
        at::Tensor out;
        if (v[7] != Py_None) {
            out = r.get(v[7], 2, v[6] == Py_None ? -1 : (int)type);
            if (!r.good || !r.need(out.size(0) == m && out.size(1) == n)) Py_RETURN_NONE;
            type = out.scalar_type();
        }
        const int dtype = r.type(type);
        if (!r.good) Py_RETURN_NONE;
        const int64_t need = packed ? ftnn_mm_i8_rows_scratch_bytes(ternary, m, n, (int)k) : 0;
        at::Tensor scratch;
        int64_t have = 0;
        if (packed && v[10] != Py_None) {
            scratch = r.get(v[10], -1);
            if (!r.good || !r.need(scratch.is_contiguous())) Py_RETURN_NONE;
            have = scratch.numel() * (int64_t)scratch.element_size();
        } else if (need > 0) {
            scratch = at::empty({have = need}, a.options().dtype(at::kByte));
        }
        if (!out.defined()) out = at::empty({m, n}, a.options().dtype(type));
        const int8_t* const codes = static_cast<const int8_t*>(a.data_ptr());
        const void* const weights = b.data_ptr();
        void *const y = out.data_ptr(), *const work = scratch.defined() ? scratch.data_ptr() : nullptr;
        const int64_t a_stride = row_stride(a, nb), b_stride = packed ? 0 : row_stride(b, nb), out_stride = row_stride(out, n);
        const int rc = unlocked([=](void* st) {
            if (packed) return ftnn_mm_i8_rows(ternary, dtype, codes, a_stride, sa, static_cast<const int64_t*>(weights), sb, bias, m, n, (int)k, y, out_stride, work, have, st);
            return ftnn_mm_i8(dtype, codes, a_stride, sa, static_cast<const int8_t*>(weights), b_stride, sb, bias, m, n, (int)k, y, out_stride, st);
        });
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}
PyObject* mm_i8(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 8) Py_RETURN_NONE;
    return product(v, false);
}
PyObject* mm_i8_rows(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 11) Py_RETURN_NONE;
    return product(v, true);
}

// cache, table, lens, starts
bool cache_of(Tensors& r, PyObject* const* v, int64_t tokens, int64_t heads, int64_t dim, int64_t page, ftnn_kv4_t* kv) {
    const at::Tensor &cache = r.get(v[0], 2, (int)at::kByte), &table = r.get(v[1], 2, (int)at::kInt);
    if (!r.good || !r.need(heads > 0 && heads <= INT_MAX && dim <= INT_MAX && tokens <= INT_MAX && table.size(0) <= INT_MAX && table.size(1) <= INT_MAX)) return false;
    if (!r.need(cache.is_contiguous() && cache.size(1) == ftnn_kv4_page_bytes((int)heads, (int)dim, (int)page))) return false;
    kv->d_cache = cache.data_ptr(), kv->pages = cache.size(0), kv->heads = (int)heads, kv->dim = (int)dim, kv->page = (int)page;
    kv->sequences = (int)table.size(0), kv->tokens = (int)tokens, kv->width = (int)table.size(1), kv->table_stride = row_stride(table, table.size(1));
    kv->d_table = static_cast<const int32_t*>(table.data_ptr());
    kv->d_lens = static_cast<const int32_t*>(r.flat(v[2], at::kInt, table.size(0)));
    kv->d_starts = static_cast<const int32_t*>(r.flat(v[3], at::kInt, table.size(0) + 1));
    return r.good;
}

// cache, table, lens, starts, k, v, page, q, cos, sin, neighbours, q_out
PyObject* kv4_append(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 12 || v[11] != Py_None || (v[8] == Py_None) != (v[9] == Py_None)) Py_RETURN_NONE;
    return answer([&]() -> PyObject* {
        Tensors r;
        const at::Tensor& k = r.get(v[4], 3);
        if (!r.good) Py_RETURN_NONE;
        const int type = (int)k.scalar_type(), dtype = r.type(k.scalar_type());
        const at::Tensor& val = r.get(v[5], 3, type);
        ftnn_kv4_t kv;
        if (!r.good || !r.need(val.sizes() == k.sizes()) || !cache_of(r, v, k.size(0), k.size(1), k.size(2), r.integer(v[6]), &kv)) Py_RETURN_NONE;
        const float *cos = nullptr, *sin = nullptr;
        int positions = 0, rot = 0;
        if (v[8] != Py_None) {
            const at::Tensor &c = r.get(v[8], 2, (int)at::kFloat), &s = r.get(v[9], 2, (int)at::kFloat);
            if (!r.good || !r.need(c.is_contiguous() && s.is_contiguous() && c.sizes() == s.sizes() && c.size(1) > 0 && c.size(1) <= 32768 && c.size(0) <= INT_MAX)) Py_RETURN_NONE;
            cos = static_cast<const float*>(c.data_ptr()), sin = static_cast<const float*>(s.data_ptr()), positions = (int)c.size(0), rot = 2 * (int)c.size(1);
        }
        at::Tensor q, q_out;
        if (v[7] != Py_None) {
            q = r.get(v[7], 3, type);
            if (!r.good || !r.need(q.size(0) == k.size(0) && q.size(2) == k.size(2) && q.size(1) <= INT_MAX)) Py_RETURN_NONE;
        }
        const int neighbours = r.truth(v[10]);
        if (!r.good) Py_RETURN_NONE;
        if (q.defined()) q_out = at::empty(q.sizes(), q.options());
        struct Rows {
            void* p = nullptr;
            int64_t token = 0, head = 0;
            int heads = 0;
        };
        auto rows = [](const at::Tensor& t) { return t.defined() ? Rows{t.data_ptr(), t.stride(0), t.stride(1), (int)t.size(1)} : Rows{}; };
        const int rc = unlocked([=, &kv, kr = rows(k), vr = rows(val), qr = rows(q), to = rows(q_out).p](void* st) {
            return ftnn_kv4_append(&kv, dtype, kr.p, kr.token, kr.head, vr.p, vr.token, vr.head, cos, sin, positions, rot, neighbours, qr.heads, qr.p, qr.token, qr.head, to, st);
        });
        if (rc) return PyLong_FromLong(rc);
        return Py_BuildValue("(N)", q.defined() ? THPVariable_Wrap(q_out) : Py_NewRef(Py_None));
    });
}

// cache, table, lens, starts, tokens, heads, dim, page, dtype
PyObject* kv4_read(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 9 || !THPDtype_Check(v[8])) Py_RETURN_NONE;
    return answer([&]() -> PyObject* {
        Tensors r;
        const int64_t tokens = r.integer(v[4]), heads = r.integer(v[5]), dim = r.integer(v[6]);
        const at::ScalarType type = reinterpret_cast<THPDtype*>(v[8])->scalar_type;
        const int dtype = r.type(type);
        ftnn_kv4_t kv;
        if (!r.need(tokens >= 0) || !cache_of(r, v, tokens, heads, dim, r.integer(v[7]), &kv)) Py_RETURN_NONE;
        const auto options = THPVariable_Unpack(v[0]).options().dtype(type);
        const at::Tensor k = at::empty({tokens, heads, dim}, options), val = at::empty({tokens, heads, dim}, options);
        const int rc = unlocked([&kv, dtype, kp = k.data_ptr(), vp = val.data_ptr()](void* st) { return ftnn_kv4_read(&kv, dtype, kp, vp, st); });
        if (rc) return PyLong_FromLong(rc);
        return Py_BuildValue("NN", THPVariable_Wrap(k), THPVariable_Wrap(val));
    });
}

// cache, table, lens, starts, q, heads, page, scale, max_len, out, scratch
PyObject* kv4_attention(PyObject*, PyObject* const* v, Py_ssize_t n) {
    if (n != 11 || !PyFloat_CheckExact(v[7])) Py_RETURN_NONE;
    return answer([&]() -> PyObject* {
        Tensors r;
        const at::Tensor& q = r.get(v[4], 3);
        if (!r.good) Py_RETURN_NONE;
        const int dtype = r.type(q.scalar_type());
        const int64_t max_len = r.integer(v[8]);
        ftnn_kv4_t kv;
        if (!r.good || !r.need(q.size(1) <= INT_MAX) || !cache_of(r, v, q.size(0), r.integer(v[5]), q.size(2), r.integer(v[6]), &kv)) Py_RETURN_NONE;
        const int heads_q = (int)q.size(1);
        at::Tensor out, scratch;
        if (v[9] != Py_None) {
            out = r.get(v[9], 3, (int)q.scalar_type());
            if (!r.good || !r.need(out.is_contiguous() && out.sizes() == q.sizes())) Py_RETURN_NONE;
        } else {
            out = at::empty(q.sizes(), q.options());
        }
        int64_t have = 0;
        if (v[10] != Py_None) {
            scratch = r.get(v[10], -1);
            if (!r.good || !r.need(scratch.is_contiguous())) Py_RETURN_NONE;
            have = scratch.numel() * (int64_t)scratch.element_size();
        } else if ((have = ftnn_kv4_attention_scratch_bytes(&kv, heads_q, (int)max_len)) > 0) {
            scratch = at::empty({have}, q.options().dtype(at::kByte));
        }
        const float scale = (float)PyFloat_AS_DOUBLE(v[7]);
        const int rc = unlocked([=, &kv, qp = q.data_ptr(), token = q.stride(0), head = q.stride(1), y = out.data_ptr(), work = scratch.defined() ? scratch.data_ptr() : nullptr](void* st) {
            return ftnn_kv4_attention(&kv, dtype, heads_q, qp, token, head, scale, (int)max_len, y, work, have, st);
        });
        return rc ? PyLong_FromLong(rc) : THPVariable_Wrap(out);
    });
}

#define FTNN_METHOD(name) {#name, reinterpret_cast<PyCFunction>(reinterpret_cast<void*>(name)), METH_FASTCALL, nullptr}
PyMethodDef methods[] = {FTNN_METHOD(mm),          FTNN_METHOD(mm_engine), FTNN_METHOD(mm_expanded), FTNN_METHOD(conv), FTNN_METHOD(conv_prepared),
                         FTNN_METHOD(conv_static), FTNN_METHOD(net_run),   FTNN_METHOD(quantize_rows_i8), FTNN_METHOD(mm_i8), FTNN_METHOD(mm_i8_rows),
                         FTNN_METHOD(kv4_append),  FTNN_METHOD(kv4_read),  FTNN_METHOD(kv4_attention), {nullptr, nullptr, 0, nullptr}};
PyModuleDef module = {PyModuleDef_HEAD_INIT, "_call", "ftnn device calls without ctypes", -1, methods, nullptr, nullptr, nullptr, nullptr};

}  // namespace

PyMODINIT_FUNC PyInit__call(void) {
    PyObject* const m = PyModule_Create(&module);
    // the torch whose tensors it reads: another one's may lie otherwise in memory
    if (m && PyModule_AddStringConstant(m, "torch_version", FTNN_TORCH) < 0) {
        Py_DECREF(m);
        return nullptr;
    }
    return m;
}
