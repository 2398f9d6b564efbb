"""Which launches the entry points of the 8-bit layers make, seen by a child process in which tests/fake_hip.c stands in for
the HIP calls of a launch (no GPU is needed, nothing is computed)."""
import ctypes as C
import json
import os
import subprocess
import sys
import threading
import time

HERE = os.path.dirname(os.path.abspath(__file__))


class Call(C.Structure):
    _fields_ = [("name", C.c_char_p), ("what", C.c_int64), ("grid", C.c_int64 * 3), ("block", C.c_int64 * 3), ("lds", C.c_int64),
                ("most", C.c_int64)]


def build(folder):
    so = os.path.join(str(folder), "fake_hip.so")
    subprocess.run(["gcc", "-O1", "-shared", "-fPIC", "-o", so, os.path.join(HERE, "fake_hip.c")], check=True)
    return so


def launches(so, calls):
    """calls: dicts of op, M, K, N (H: inner width; gap: values between rows; t, out: element types; act).  A call with "beside",
    another call, is made first, and that one on a second thread while the first is setting its kernel's largest LDS (or when it
    has returned).  -> for each, (return code, [(kernel, grid, block, dynamic LDS, the most that the kernel may have)])"""
    r = subprocess.run([sys.executable, os.path.abspath(__file__), so], input=json.dumps(calls), capture_output=True, text=True)
    assert r.returncode == 0, r.stderr[-2000:]
    return json.loads(r.stdout)


def _child(so):
    fake = C.CDLL(so, mode=C.RTLD_GLOBAL)
    fake.fake_call.restype = C.POINTER(Call)
    sys.path.insert(0, os.path.join(os.path.dirname(HERE), "pose-estimation_amd"))
    from posehip import _ffi
    lib = C.CDLL(_ffi.LIB_PATH)
    for name, (res, args) in _ffi.SYMBOLS.items():
        getattr(lib, name).restype, getattr(lib, name).argtypes = res, args
    at, big = 1 << 20, 1 << 60   # addresses that nothing follows

    def make(c):
        M, K, N, H = c["M"], c["K"], c.get("N", 16), c.get("H", 0)
        rows = _ffi.PhRows((C.c_int64 * 3)(1, 1, M), (C.c_int64 * 3)(0, 0, K + c.get("gap", 0)))
        t, out = c.get("t", _ffi.PH_BF16), c.get("out", _ffi.PH_BF16)
        layer = lambda n, k: _ffi.PhW8Layer(at, at, at, at, n, k, c.get("act", 0))   # noqa: E731
        st = (C.c_int64 * 3)(0, 0, N)
        if c["op"] == "matmul":
            return lib.ph_w8_matmul(0, None, at, rows, at, layer(N, K), at, out, st, at, big)
        if c["op"] == "linear":
            return lib.ph_w8_linear(0, None, at, t, rows, layer(N, K), at, out, st, at, big)
        if c["op"] == "feed_forward":
            return lib.ph_w8_feed_forward(0, None, at, t, rows, layer(H, K), layer(N, H), at, out, st, at, big)
        return lib.ph_w8_quantize_rows(0, None, at, t, rows, K, at, (K + 15) // 16 * 16, at)

    done = []
    for c in json.load(sys.stdin):
        fake.fake_clear()
        if "beside" in c:
            fake.fake_wait(300)
            rcs = []
            first = threading.Thread(target=lambda: rcs.append(make(c)))
            first.start()
            while first.is_alive() and not fake.fake_setters():
                time.sleep(0.001)
            rc = make(c["beside"])
            first.join()
            fake.fake_wait(0)
            rc = rc or rcs[0]
        else:
            rc = make(c)
        seen = [fake.fake_call(i).contents for i in range(fake.fake_calls())]
        done.append((rc, [(s.name.decode() if s.name else "?", list(s.grid), list(s.block), s.lds, s.most) for s in seen if s.what == 0]))
    json.dump(done, sys.stdout)


if __name__ == "__main__":
    _child(sys.argv[1])
