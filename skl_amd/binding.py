"""ctypes loader for libskl_gfx950.so."""
import ctypes
import os

import numpy as np

from . import signatures

_HERE = os.path.dirname(os.path.abspath(__file__))
_SUFFIX = "_gfx950"


class LibraryNotBuilt(RuntimeError):
    pass


def library_path():
    return os.path.join(_HERE, "lib", "libskl_gfx950.so")


class _Lib:
    """Holds the CDLL and one Python callable per C entry point."""

    def __init__(self, path):
        if not os.path.exists(path):
            raise LibraryNotBuilt(
                f"{path} is missing: build it with `make -C skl_amd/csrc` (or __graft_entry__.build()); "
                "there is no CPU fallback")
        self.path = path
        self.cdll = ctypes.CDLL(path)
        self.names = []
        for name, (restype, sig) in signatures.RUNTIME.items():
            raw = signatures.bind(self.cdll, name, sig, restype)
            setattr(self, name, _wrap(raw, sig) if "p" in sig else raw)
        for table in (signatures.reference_shared(), signatures.gfx950_only()):
            for stem, sig in table.items():
                cname = stem + _SUFFIX
                raw = signatures.bind(self.cdll, cname, sig)
                setattr(self, cname, _wrap(raw, sig))
                self.names.append(cname)


def _as_pointer(x):
    if x is None:
        return None
    if isinstance(x, DeviceBuffer):
        return x.ptr
    if isinstance(x, np.ndarray):
        return x.ctypes.data
    return x  # integer address


class Epilogue:
    """Fused-epilogue operands of the `skl_gemm_fused_*` entry points: `bias` (n values of C's
    type), `max` (one value of C's type), `activation` (ACT_NONE / ACT_RELU; floating-point C also ACT_SILU / ACT_GELU) and the requantised
    copy `q` (int8, element (i, j) at `i * rsq + j * csq`) made with `q_scale` (one float32, or n
    of them with `q_scale_per_column`) and `q_zero`; `q_only` leaves C unwritten. Every operand
    is a DeviceBuffer, a numpy array or None."""

    ACT_NONE, ACT_RELU, ACT_SILU, ACT_GELU = 0, 1, 2, 3

    Q_INT8, Q_F8E4M3, Q_F8E4M3_SAT, Q_F8E5M2, Q_F8E5M2_SAT = range(5)

    def __init__(self, bias=None, max=None, activation=0, q=None, rsq=0, csq=0, q_scale=None,
                 q_scale_per_column=False, q_zero=0, q_only=False, q_format=0):
        self.bias, self.max, self.activation = bias, max, activation
        self.q, self.rsq, self.csq, self.q_scale = q, rsq, csq, q_scale
        self.q_scale_per_column, self.q_zero, self.q_only, self.q_format = q_scale_per_column, q_zero, q_only, q_format

    def as_struct(self):
        return signatures.EpilogueStruct(_as_pointer(self.bias), _as_pointer(self.max), int(self.activation),
                                         int(bool(self.q_scale_per_column)), int(bool(self.q_only)), int(self.q_zero),
                                         _as_pointer(self.q), int(self.rsq), int(self.csq),
                                         _as_pointer(self.q_scale), int(self.q_format))


class MoeLayer:
    """A mixture-of-experts layer (`skl_gfx950_moe_t`, every member by its name there) for `skl_moe_bf16_mxf4e2m1_f32`. Pointers are
    DeviceBuffers, numpy arrays, integer addresses or None; what they refer to is kept as long as the layer is. The C descriptor is
    made once."""

    def __init__(self, **members):
        fields = dict(signatures.MoeStruct._fields_)
        unknown = set(members) - set(fields)
        if unknown:
            raise TypeError(f"skl_gfx950_moe_t has no member {sorted(unknown)[0]}")
        self.members = members
        self._struct = signatures.MoeStruct(**{name: _as_pointer(v) if fields[name] is ctypes.c_void_p else int(v) for name, v in members.items()})

    def as_struct(self):
        return self._struct


def _descriptor(x, struct):
    """The C structure that an Epilogue or a MoeLayer stands for."""
    made = x.as_struct() if hasattr(x, "as_struct") else None
    if not isinstance(made, struct):
        raise TypeError(f"expected what describes a {struct.__name__}, got {type(x).__name__}")
    return made


def _wrap(raw, sig):
    """A callable that hands its arguments to `raw`: pointers and descriptors by what they stand for, each looked at once, everything else as it is. The
    code is written out per signature: 1.7 us for 16 arguments by address, 2.2 for buffers, where a loop over a list takes 2.6 and 2.4."""
    names = [f"a{i}" for i in range(len(sig))]
    lines, passed = [], []
    for name, ch in zip(names, sig):
        if ch == "p":
            passed.append(f"{name} if type({name}) is int else as_pointer({name})")
        elif ch in signatures.STRUCTS:
            lines.append(f"    if {name} is not None: {name} = descriptor({name}, structs[{ch!r}])")  # alive until the call returns
            passed.append(f"None if {name} is None else addressof({name})")
        else:
            passed.append(name)
    source = "\n".join([
        "def call(*args):",
        "    try:",
        f"        {', '.join(names)}, = args",
        "    except ValueError:",
        f"        raise TypeError(f\"{raw.__name__}: expected {len(sig)} arguments, got {{len(args)}}\") from None",
        *lines,
        f"    return raw({', '.join(passed)})"])
    scope = {"raw": raw, "as_pointer": _as_pointer, "descriptor": _descriptor, "structs": signatures.STRUCTS, "addressof": ctypes.addressof}
    exec(compile(source, f"<{raw.__name__}>", "exec"), scope)
    call = scope["call"]
    call.__name__ = raw.__name__
    call.raw = raw
    return call


_lib = None


def load():
    global _lib
    if _lib is None:
        _lib = _Lib(library_path())
    return _lib


def lib():
    return load()


def check_error():
    """Raises if a kernel entry point recorded an error since the last check."""
    code = load().skl_hip_last_error()
    if code != 0:
        raise RuntimeError(f"skl-gfx950 error {code}: {load().skl_hip_last_error_string().decode()}")


class DeviceBuffer:
    """A device allocation made through the library's shim (skl_hip_malloc)."""

    def __init__(self, nbytes):
        self.nbytes = int(nbytes)
        self.ptr = load().skl_hip_malloc(max(self.nbytes, 1))
        if not self.ptr:
            check_error()
            raise MemoryError(f"skl_hip_malloc({nbytes}) failed")

    @classmethod
    def from_array(cls, arr):
        arr = np.ascontiguousarray(arr)
        buf = cls(arr.nbytes)
        buf.upload(arr)
        return buf

    def upload(self, arr):
        arr = np.ascontiguousarray(arr)
        if arr.nbytes > self.nbytes:
            raise ValueError("array larger than buffer")
        rc = load().skl_hip_memcpy_h2d(self.ptr, arr.ctypes.data, arr.nbytes)
        if rc != 0:
            check_error()

    def download(self, dtype, count=None):
        dtype = np.dtype(dtype)
        if count is None:
            count = self.nbytes // dtype.itemsize
        out = np.empty(count, dtype=dtype)
        rc = load().skl_hip_memcpy_d2h(out.ctypes.data, self.ptr, out.nbytes)
        if rc != 0:
            check_error()
        return out

    def offset(self, nbytes):
        """Address `nbytes` into the buffer (for misalignment tests)."""
        return self.ptr + int(nbytes)

    def free(self):
        if self.ptr:
            load().skl_hip_free(self.ptr)
            self.ptr = None

    def __del__(self):
        try:
            self.free()
        except Exception:
            pass
