"""The library's own objects linked against a CUDA runtime without a GPU (fake_cuda_runtime.cpp): its host code runs, its kernels are noted."""
import ctypes as C
import os
import re
import struct
import subprocess

ROOT = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
CSRC = os.path.join(ROOT, "tenmo_b200", "csrc")
HERE = os.path.dirname(os.path.abspath(__file__))
CUDA = os.environ.get("CUDA_HOME", "/usr/local/cuda")


def build(folder) -> str:
    """Links a library of its own (its state begins anew)."""
    subprocess.run(["make", "-s", "-C", CSRC, "-j", str(min(8, os.cpu_count() or 1))], check=True)
    sources = re.search(r"^SRCS := (.*)$", open(os.path.join(CSRC, "Makefile")).read(), re.M).group(1).split()
    out = os.path.join(str(folder), "libtenmo_on_fake.so")
    subprocess.run(["g++", "-shared", "-fPIC", "-O1", "-std=c++17", "-Wl,-Bsymbolic", f"-I{CUDA}/include", "-o", out,
                    os.path.join(HERE, "fake_cuda_runtime.cpp")] + [os.path.join(CSRC, "build", s[:-3] + ".o") for s in sources] + ["-ldl"],
                   check=True)
    return out


class Fake:
    """What the runtime has noted; ``handle`` is the framework's binding on top of it."""

    def __init__(self, path):
        from tenmo_b200 import TenmoCuda

        self.path = str(path)
        self.lib = C.CDLL(self.path)
        for name, result, args in (("fake_launch_name", C.c_char_p, [C.c_int]), ("fake_misuse_text", C.c_char_p, [C.c_int]),
                                   ("fake_room_behind", C.c_size_t, [C.c_size_t]), ("fake_bytes_alive", C.c_size_t, []),
                                   ("fake_stream_create", C.c_size_t, [C.c_size_t]), ("fake_stream_destroy", None, [C.c_size_t]),
                                   ("fake_capture", None, [C.c_size_t, C.c_int]), ("fake_forget_launches", None, []),
                                   ("cudaMalloc", C.c_int, [C.POINTER(C.c_size_t), C.c_size_t])):
            f = getattr(self.lib, name)
            f.restype, f.argtypes = result, args
        self._types = {}
        self.handle = TenmoCuda(0, path=self.path).require()

    def malloc(self, n: int) -> int:
        p = C.c_size_t()
        assert self.lib.cudaMalloc(C.byref(p), n) == 0
        return p.value

    def watch(self, kernel: str, types: str):
        """Keep the arguments of launches of ``kernel``; ``types`` as in struct, one letter an argument."""
        sizes = [struct.calcsize(t) for t in types]
        self.lib.fake_watch(kernel.encode(), (C.c_int * len(sizes))(*sizes), len(sizes))
        self._types[kernel] = types

    def launches(self):
        """(index, name, arguments or None) in the order of their launch."""
        out = []
        for i in range(self.lib.fake_launches()):
            name, args = self.lib.fake_launch_name(i).decode(), None
            if self.lib.fake_launch_args(i):
                types = next(t for k, t in self._types.items() if k in name)
                buf = C.create_string_buffer(16)
                args = []
                for k, t in enumerate(types):
                    self.lib.fake_launch_arg(i, k, buf)
                    args.append(struct.unpack(t, buf.raw[:struct.calcsize(t)])[0])
            out.append((i, name, args))
        return out

    def captured(self, i: int) -> bool:
        return bool(self.lib.fake_launch_captured(i))

    def comes_before(self, i: int, j: int) -> bool:
        return bool(self.lib.fake_comes_before(i, j))

    def misuse(self):
        return [self.lib.fake_misuse_text(i).decode() for i in range(self.lib.fake_misuse())]
