"""ctypes binding of libb200_kernels.so.

The C prototypes are read from include/b200_kernels.h, so the Python side cannot
drift from the header: every function the header declares is bound with the
argument types written there, and a missing export is an error at load time.
There is no fallback of any kind: if the shared object is absent or a call is made
without a CUDA device, an exception says so.
"""
from __future__ import annotations

import ctypes
import re
from pathlib import Path

try:
    from .fastcall import load as load_calls, types_of
except ImportError:      # loaded by path, without its package (build.py reads the prototypes)
    def load_calls():
        return None

HERE = Path(__file__).resolve().parent
HEADER = HERE.parent / "include" / "b200_kernels.h"
LIB_PATH = HERE / "libb200_kernels.so"

_SCALARS = {
    "int": ctypes.c_int,
    "float": ctypes.c_float,
    "size_t": ctypes.c_size_t,
    "b200k_stream": ctypes.c_void_p,
    "uint64_t": ctypes.c_uint64,
    "int64_t": ctypes.c_int64,
}
# int-returning functions whose value is a count, not a status
_NOT_STATUS = {"b200k_layer_launches_per_forward"}
_RET = {"int": ctypes.c_int, "size_t": ctypes.c_size_t, "const char *": ctypes.c_char_p, "void": None}


class B200KError(RuntimeError):
    def __init__(self, name: str, code: int, message: str):
        super().__init__(f"{name} failed with status {code}: {message}")
        self.code = code
        self.message = message


def parse_header(path: Path = HEADER):
    """-> {name: (restype_key, [(ctype_key, argname), ...])} for every prototype."""
    text = path.read_text()
    text = re.sub(r"/\*.*?\*/", " ", text, flags=re.S)
    text = re.sub(r"//[^\n]*", " ", text)
    text = re.sub(r"^\s*#.*$", " ", text, flags=re.M)
    protos = {}
    pat = re.compile(r"\b(const\s+char\s*\*\s*|int\s+|size_t\s+|void\s+)(\w+)\s*\(([^;{}]*?)\)\s*;", re.S)
    for m in pat.finditer(text):
        ret, name, args = m.group(1), m.group(2), m.group(3)
        ret = "const char *" if "char" in ret else ret.strip()
        parsed = []
        args = " ".join(args.split())
        if args and args != "void":
            for a in args.split(","):
                a = a.strip()
                am = re.match(r"^(.*?)(\w+)$", a)
                ty, an = am.group(1).strip(), am.group(2)
                if "*" in ty:
                    parsed.append(("ptr", an))
                else:
                    ty = ty.replace("const ", "").strip()
                    if ty not in _SCALARS:
                        raise ValueError(f"{name}: unknown C type {ty!r}")
                    parsed.append((ty, an))
        protos[name] = (ret, parsed)
    return protos


class Library:
    def __init__(self, path: Path = LIB_PATH):
        if not path.exists():
            raise FileNotFoundError(
                f"{path} is missing: build it with `python {HERE.name}/build.py` "
                "(nvcc, sm_100a). There is no CPU fallback.")
        self._dll = ctypes.CDLL(str(path), mode=ctypes.RTLD_GLOBAL)
        self.protos = parse_header()
        self._fns = {}
        self._callers = {}
        self._compiled = load_calls()
        missing = []
        for name, (ret, args) in self.protos.items():
            try:
                fn = getattr(self._dll, name)
            except AttributeError:
                missing.append(name)
                continue
            fn.restype = _RET[ret]
            fn.argtypes = [ctypes.c_void_p if t == "ptr" else _SCALARS[t] for t, _ in args]
            self._fns[name] = fn
        if missing:
            raise ImportError(f"{path} does not export: {', '.join(missing)}")

    def last_error(self) -> str:
        return self._fns["b200k_last_error"]().decode()

    def raw(self, name: str):
        return self._fns[name]

    def caller(self, name: str, tensor_type, current=None):
        """A function of `name`'s arguments that does what `call` does, with the conversions written out for its prototype: a
        decode step makes a dozen calls of a few microseconds each, and the loop in `call` takes as long as a kernel.
        `tensor_type` is torch.Tensor (this module does not import torch); anything else goes the way of `call`.  With `current`, a
        function, the stream (the last argument) may be left out or given by name; `current()` then says which."""
        fn = self._callers.get((name, current))
        if fn is None:
            ret, proto = self.protos[name]

            def fail(rc):
                raise B200KError(name, rc, self.last_error())
            status = ret == "int" and name not in _NOT_STATUS
            if self._compiled is not None and ret in ("int", "size_t"):
                fn = self._compiled.caller(name, types_of(proto), ctypes.cast(self._fns[name], ctypes.c_void_p).value, tensor_type,
                                           lambda at, a: self._pointer(name, proto[at][1], a), self._stream, fail if status else None, current)
                if fn is not None:
                    self._callers[(name, current)] = fn
                    return fn
            conv = []
            for ty, an in proto:
                if ty == "ptr":
                    conv.append(f"{an}.data_ptr() if {an}.__class__ is T and {an}.is_cuda else P({an}, {an!r})")
                elif ty == "b200k_stream":
                    conv.append(f"{an} if {an}.__class__ is int and {an} else S({an})")
                elif ty == "float":
                    conv.append(f"{an} if {an}.__class__ is float else float({an})")
                else:
                    conv.append(f"{an} if {an}.__class__ is int else int({an})")
            check = "    if rc: E(rc)\n" if status else ""
            src = f"def caller({', '.join([an for _, an in proto] + ['/'] * bool(proto))}):\n    rc = F({', '.join(conv)})\n{check}    return rc\n"
            space = {"T": tensor_type, "F": self._fns[name], "P": lambda a, an: self._pointer(name, an, a), "S": self._stream, "E": fail}
            exec(compile(src, f"<{name}>", "exec"), space)
            fn = space["caller"]
            if current is not None:
                fn = self._streamed(name, len(proto), fn, current)
            self._callers[(name, current)] = fn
        return fn

    @staticmethod
    def _streamed(name, nargs, call, current):
        def fn(*args, stream=None):
            if len(args) == nargs - 1:
                return call(*args, current() if stream is None else stream)
            return call(*args)
        fn.__name__ = name
        fn.__doc__ = f"C ABI `{name}`; see include/b200_kernels.h for the argument list."
        return fn

    @staticmethod
    def _pointer(name, an, a):
        if a is None:
            return None
        if hasattr(a, "data_ptr"):
            if not a.is_cuda and not an.startswith("host"):
                raise ValueError(f"{name}: argument {an} must be a CUDA tensor (no CPU fallback exists)")
            return a.data_ptr()
        return int(a)

    @staticmethod
    def _stream(a):
        return None if a in (None, 0) else int(getattr(a, "cuda_stream", a))

    def call(self, name: str, *args):
        """Call `name`; torch tensors become device pointers; a non-zero status raises."""
        ret, proto = self.protos[name]
        if len(args) != len(proto):
            raise TypeError(f"{name} takes {len(proto)} arguments ({', '.join(n for _, n in proto)}), got {len(args)}")
        conv = []
        for (ty, an), a in zip(proto, args):
            if ty == "ptr":
                conv.append(self._pointer(name, an, a))
            elif ty == "b200k_stream":
                conv.append(self._stream(a))
            elif ty == "float":
                conv.append(float(a))
            else:
                conv.append(int(a))
        rc = self._fns[name](*conv)
        if ret == "int" and rc != 0 and name not in _NOT_STATUS:
            raise B200KError(name, rc, self.last_error())
        return rc


_LIB = None


def lib() -> Library:
    global _LIB
    if _LIB is None:
        _LIB = Library()
    return _LIB
