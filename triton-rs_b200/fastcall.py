"""Build recipe for `_b200_call.so`, the compiled edition of `Library.caller`.

A decode step makes a dozen calls of twenty arguments, and converting them in Python and ctypes takes longer than the kernels
run: 7 us a call on the host where the launch itself takes 2.  This writes a C file with one typed call per prototype of
include/b200_kernels.h and one function that converts the arguments, and compiles it against the CPython headers (build.py does so
with the library).  The extension holds no address of its own: `_lib.Library` hands it those of the library it has loaded.  Where
it cannot be built, `Library.caller` does the same in Python.
"""
from __future__ import annotations

import importlib.util
import os
import subprocess
import sysconfig
from pathlib import Path

HERE = Path(__file__).resolve().parent
OUT = HERE / ("_b200_call" + (sysconfig.get_config_var("EXT_SUFFIX") or ".so"))
HEADER = HERE.parent / "include" / "b200_kernels.h"
_CTYPE = {"ptr": "void *", "int": "int", "float": "float", "size_t": "size_t", "b200k_stream": "void *", "uint64_t": "uint64_t", "int64_t": "int64_t"}
_FIELD = {"ptr": "p", "int": "i", "float": "f", "size_t": "u", "b200k_stream": "p", "uint64_t": "u", "int64_t": "i"}
_CODE = {"ptr": "p", "int": "i", "float": "f", "size_t": "u", "b200k_stream": "s", "uint64_t": "u", "int64_t": "l"}
_RET = {"int": "int", "size_t": "size_t"}
EDITION = 2          # of the arguments that the extension's caller() takes

_BODY = r"""
#define PY_SSIZE_T_CLEAN
#include <Python.h>
#include <stddef.h>
#include <stdint.h>
#include <string.h>

typedef union { void *p; long long i; unsigned long long u; float f; } Arg;
typedef long long (*Call)(void *, const Arg *);
%(calls)s
typedef struct { const char *name; const char *types; Call call; } Proto;
static const Proto protos[] = {
%(table)s};
enum { COUNT = sizeof(protos) / sizeof(protos[0]), MOST = %(most)d };

typedef struct {
    PyObject_HEAD
    vectorcallfunc vectorcall;
    const Proto *proto;
    void *address;
    Py_ssize_t count;
    PyTypeObject *tensor;                 /* exact type whose data_ptr() is taken */
    PyObject *pointer, *stream, *error;   /* what Python does with other arguments, and with a status that is not 0 (or None) */
    PyObject *current;                    /* None, or what gives the stream of a call that leaves it out */
} Caller;

static PyObject *s_is_cuda, *s_data_ptr, *s_stream;

static int convert(Caller *c, PyObject *o, Py_ssize_t at, Arg *a) {
    PyObject *v = NULL;
    switch (c->proto->types[at]) {
        case 'i': {
            const long x = PyLong_CheckExact(o) ? PyLong_AsLong(o) : ((v = PyNumber_Long(o)) ? PyLong_AsLong(v) : -1);
            Py_XDECREF(v);
            if (x == -1 && PyErr_Occurred()) return -1;
            a->i = (int)x;
            return 0;
        }
        case 'l':
        case 'u':
            if (!(v = PyNumber_Long(o))) return -1;
            a->u = PyLong_AsUnsignedLongLongMask(v);
            Py_DECREF(v);
            return PyErr_Occurred() ? -1 : 0;
        case 'f': {
            const double x = PyFloat_CheckExact(o) ? PyFloat_AS_DOUBLE(o) : PyFloat_AsDouble(o);
            if (x == -1.0 && PyErr_Occurred()) return -1;
            a->f = (float)x;
            return 0;
        }
        case 's':
            if (o == Py_None) { a->p = NULL; return 0; }
            if (PyLong_CheckExact(o)) break;
            v = PyObject_CallOneArg(c->stream, o);
            if (!v) return -1;
            break;
        default:
            if (o == Py_None) { a->p = NULL; return 0; }
            if (Py_TYPE(o) == c->tensor) {
                PyObject *cuda = PyObject_GetAttr(o, s_is_cuda);
                if (!cuda) return -1;
                const int is = cuda == Py_True;
                Py_DECREF(cuda);
                if (is) {
                    v = PyObject_CallMethodNoArgs(o, s_data_ptr);
                    if (!v) return -1;
                    break;
                }
            } else if (PyLong_CheckExact(o)) {
                break;
            }
            v = PyObject_CallFunction(c->pointer, "nO", at, o);
            if (!v) return -1;
    }
    if ((v ? v : o) == Py_None) a->p = NULL;
    else a->p = PyLong_AsVoidPtr(v ? v : o);
    Py_XDECREF(v);
    return PyErr_Occurred() ? -1 : 0;
}

static PyObject *caller_call(PyObject *self, PyObject *const *args, size_t nargsf, PyObject *kwnames) {
    Caller *c = (Caller *)self;
    const Py_ssize_t n = PyVectorcall_NARGS(nargsf), named = kwnames ? PyTuple_GET_SIZE(kwnames) : 0;
    const int may = c->current != Py_None;
    if (!(n == c->count || (may && n == c->count - 1)) || named > may ||
        (named && PyUnicode_Compare(PyTuple_GET_ITEM(kwnames, 0), s_stream))) {
        if (!PyErr_Occurred())
            PyErr_Format(PyExc_TypeError, "%%s takes %%zd arguments%%s, got %%zd", c->proto->name, c->count, may ? " (the stream may be left out or named)" : "", n);
        return NULL;
    }
    Arg a[MOST];
    for (Py_ssize_t i = 0; i < n; ++i)
        if (convert(c, args[i], i, &a[i])) return NULL;
    if (n < c->count) {
        PyObject *own = named && args[n] != Py_None ? Py_NewRef(args[n]) : PyObject_CallNoArgs(c->current);
        if (!own) return NULL;
        const int bad = convert(c, own, n, &a[n]);
        Py_DECREF(own);
        if (bad) return NULL;
    }
    long long rc;
    Py_BEGIN_ALLOW_THREADS
    rc = c->proto->call(c->address, a);
    Py_END_ALLOW_THREADS
    if (rc && c->error != Py_None) {
        PyObject *r = PyObject_CallFunction(c->error, "L", rc);
        Py_XDECREF(r);
        if (!r) return NULL;
    }
    return PyLong_FromLongLong(rc);
}

static void caller_free(PyObject *self) {
    Caller *c = (Caller *)self;
    Py_CLEAR(c->tensor);
    Py_CLEAR(c->pointer);
    Py_CLEAR(c->stream);
    Py_CLEAR(c->error);
    Py_CLEAR(c->current);
    Py_TYPE(self)->tp_free(self);
}

static PyObject *caller_name(PyObject *self, void *unused) { return PyUnicode_FromString(((Caller *)self)->proto->name); }
static PyObject *caller_doc(PyObject *self, void *unused) {
    return PyUnicode_FromFormat("C ABI `%%s`; see include/b200_kernels.h for the argument list.", ((Caller *)self)->proto->name);
}
static PyGetSetDef caller_has[] = {{"__name__", caller_name}, {"__doc__", caller_doc}, {NULL}};

static PyTypeObject CallerType = {
    PyVarObject_HEAD_INIT(NULL, 0).tp_name = "_b200_call.Caller", .tp_basicsize = sizeof(Caller), .tp_dealloc = caller_free,
    .tp_flags = Py_TPFLAGS_DEFAULT | Py_TPFLAGS_HAVE_VECTORCALL, .tp_vectorcall_offset = offsetof(Caller, vectorcall), .tp_call = PyVectorcall_Call,
    .tp_getset = caller_has};

/* caller(name, types, address, tensor type, pointer, stream, error, current): None when this build has no such prototype */
static PyObject *make_caller(PyObject *self, PyObject *args) {
    const char *name, *types;
    unsigned long long address;
    PyObject *tensor, *pointer, *stream, *error, *current;
    if (!PyArg_ParseTuple(args, "ssKOOOOO", &name, &types, &address, &tensor, &pointer, &stream, &error, &current)) return NULL;
    const size_t count = strlen(types);
    if (current != Py_None && (!count || types[count - 1] != 's')) Py_RETURN_NONE;
    for (int i = 0; i < COUNT; ++i)
        if (!strcmp(protos[i].name, name) && !strcmp(protos[i].types, types) && PyType_Check(tensor)) {
            Caller *c = (Caller *)CallerType.tp_alloc(&CallerType, 0);
            if (!c) return NULL;
            c->vectorcall = caller_call;
            c->proto = &protos[i];
            c->address = (void *)(uintptr_t)address;
            c->count = (Py_ssize_t)count;
            c->tensor = (PyTypeObject *)Py_NewRef(tensor);
            c->pointer = Py_NewRef(pointer);
            c->stream = Py_NewRef(stream);
            c->error = Py_NewRef(error);
            c->current = Py_NewRef(current);
            return (PyObject *)c;
        }
    Py_RETURN_NONE;
}

static PyMethodDef methods[] = {{"caller", make_caller, METH_VARARGS, "A caller for one prototype, or None."}, {NULL, NULL, 0, NULL}};
static struct PyModuleDef module = {PyModuleDef_HEAD_INIT, "_b200_call", "Argument conversion for libb200_kernels.so.", -1, methods};
PyMODINIT_FUNC PyInit__b200_call(void) {
    s_is_cuda = PyUnicode_InternFromString("is_cuda");
    s_data_ptr = PyUnicode_InternFromString("data_ptr");
    s_stream = PyUnicode_InternFromString("stream");
    if (!s_is_cuda || !s_data_ptr || !s_stream || PyType_Ready(&CallerType) < 0) return NULL;
    PyObject *m = PyModule_Create(&module);
    if (m && PyModule_AddIntConstant(m, "EDITION", %(edition)d)) Py_CLEAR(m);
    return m;
}
"""


def types_of(proto) -> str:
    """One letter an argument, the key under which the extension knows a prototype."""
    return "".join(_CODE[ty] for ty, _ in proto)


def source(protos) -> str:
    calls, table, most = [], [], 1
    for name, (ret, args) in protos.items():
        if ret not in _RET:
            continue
        most = max(most, len(args))
        sig = ", ".join(_CTYPE[ty] for ty, _ in args) or "void"
        conv = ", ".join(f"({_CTYPE[ty]})a[{i}].{_FIELD[ty]}" if ty != "float" else f"a[{i}].f" for i, (ty, _) in enumerate(args))
        calls.append(f"static long long call_{name}(void *f, const Arg *a) {{ return (long long)(({_RET[ret]} (*)({sig}))f)({conv}); }}")
        table.append(f'    {{"{name}", "{types_of(args)}", call_{name}}},')
    return _BODY % {"edition": EDITION, "calls": "\n".join(calls), "table": "\n".join(table) + "\n", "most": most}


def build(protos, obj_dir: Path) -> Path | None:
    """Compiles the extension; None (and no exception) where there is no C compiler or no CPython header."""
    src = obj_dir / "b200_call.c"
    src.write_text(source(protos))
    cmd = [os.environ.get("CC", "gcc"), "-O2", "-shared", "-fPIC", "-fvisibility=hidden", "-I", sysconfig.get_paths()["include"], str(src), "-o", str(OUT)]
    try:
        done = subprocess.run(cmd, capture_output=True, text=True)
    except OSError as e:
        print(f"{OUT.name} not built: {e}")
        return None
    if done.returncode:
        print(f"{OUT.name} not built:\n{done.stderr[-2000:]}")
        return None
    return OUT


def load():
    """The extension module, or None."""
    if not OUT.exists():
        return None
    try:
        spec = importlib.util.spec_from_file_location("_b200_call", OUT)
        mod = importlib.util.module_from_spec(spec)
        spec.loader.exec_module(mod)
        return mod if getattr(mod, "EDITION", 1) == EDITION else None
    except ImportError:
        return None
