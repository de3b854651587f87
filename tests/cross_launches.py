"""Which kernels a call of rsfa_cross_fwd or rsfa_cross_bwd launches, without a GPU (by tests/launch_recorder.cpp, whose
HIP entry points a child process loads ahead of librsfa.so)."""
import json
import os
import re
import subprocess
import sys

_TESTS = os.path.dirname(os.path.abspath(__file__))
_PKG = os.path.join(os.path.dirname(_TESTS), "ascend-rsfa_amd", "ascend_rsfa")


def variants(shapes, tmp_path, entry="rsfa_cross_fwd"):
    """For each (Z, heads, key heads, T, N, D) the kernels launched: (name, template numbers)."""
    so = os.path.join(str(tmp_path), "librecorder.so")
    if not os.path.exists(so):
        subprocess.run(["g++", "-std=c++17", "-O1", "-shared", "-fPIC", "-DRECORDER_TICKET_OFFSET=0", "-DRECORDER_PAIRS_OFFSET=0",
                        "-o", so, os.path.join(_TESTS, "launch_recorder.cpp")], check=True)
    out = subprocess.run([sys.executable, os.path.abspath(__file__)], text=True, capture_output=True, timeout=120,
                         input=json.dumps({"so": so, "entry": entry, "shapes": [list(s) for s in shapes]}))
    assert out.returncode == 0, out.stderr
    result = []
    for status, lines in json.loads(out.stdout.splitlines()[-1]):
        assert status == 0, status
        names = [(re.search(r"fa_fwd_kernel|cross_\w+?_kernel|sum_parts_kernel", x).group(),
                  tuple(int(n) for n in re.findall(r"L[ib](\d+)E", x))) for x in lines]
        result.append(names)
    return result


def _child():
    import ctypes
    import importlib.util

    spec = json.load(sys.stdin)
    rec = ctypes.CDLL(spec["so"], mode=ctypes.RTLD_GLOBAL)
    rec.recorder_lines.restype = ctypes.c_char_p
    mod = importlib.util.spec_from_file_location("_native", os.path.join(_PKG, "_native.py"))
    native = importlib.util.module_from_spec(mod)
    mod.loader.exec_module(native)
    lib = native.lib()
    results = []
    for Z, Hq, H, T, N, D in spec["shapes"]:
        a = native.CrossArgs() if spec["entry"] == "rsfa_cross_fwd" else native.CrossBwdArgs()
        a.struct_size = ctypes.sizeof(a)
        for name, _ in a._fields_:
            if name.endswith("_stride"):
                getattr(a, name)[:] = (1 << 20, 1 << 14, D, 1)
                setattr(a, name[:-7], 0x1000)
        a.lse = 0x1000
        a.z, a.heads, a.key_heads, a.t, a.n, a.head_dim, a.sm_scale = Z, Hq, H, T, N, D, 0.1
        a.workspace, a.workspace_bytes = 0x1000, 1 << 40
        rec.recorder_clear()
        results.append((getattr(lib, spec["entry"])(ctypes.byref(a), None), rec.recorder_lines().decode().splitlines()))
    print(json.dumps(results))


if __name__ == "__main__":
    _child()
