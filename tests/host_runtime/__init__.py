"""The library on a stand-in for the HIP runtime (runtime.cpp), in a process of its own: `run` executes Python code there, after a prelude that loads both
and opens nothing yet."""
import os
import subprocess
import sys
import tempfile

HERE = os.path.dirname(os.path.abspath(__file__))
ROOT = os.path.dirname(os.path.dirname(HERE))

PRELUDE = """
import ctypes as C, sys
sys.path.insert(0, {root!r})
rt = C.CDLL({lib!r}, mode=C.RTLD_GLOBAL)        # before the library: its soname is the runtime's
rt.hostrt_launches.restype = rt.hostrt_sizes.restype = C.c_long
rt.hostrt_held.restype = C.c_size_t
import numpy as np
import chatterbox_amd as cb
from chatterbox_amd import _lib, synth, t3
L = _lib.load()

def model(dims=synth.TINY, dtype="f32", **kw):
    return cb.load_t3(synth.ensure_checkpoint(dims, 1234), device=0, dtype=dtype, start_speech_token=dims.start_speech_token, stop_speech_token=dims.stop_speech_token, **kw)

def prompt(n, seed=1, dims=synth.TINY):
    return synth.synth_embeds(2, n, dims.hidden_size, seed)

def sizes():
    a = (C.c_size_t * 4096)()
    return list(a[:rt.hostrt_sizes(a, 4096)])
"""

_dir = None


def run(code):
    global _dir
    if _dir is None:
        _dir = tempfile.TemporaryDirectory(prefix="host_runtime_")
        subprocess.check_call(["g++", "-std=c++17", "-O1", "-fPIC", "-shared", "-Wl,-soname,libamdhip64.so.7", os.path.join(HERE, "runtime.cpp"),
                               "-o", os.path.join(_dir.name, "libamdhip64.so.7")])
    prelude = PRELUDE.format(root=ROOT, lib=os.path.join(_dir.name, "libamdhip64.so.7"))
    r = subprocess.run([sys.executable, "-c", prelude + code], capture_output=True, text=True, timeout=300)
    assert r.returncode == 0, r.stdout[-1500:] + r.stderr[-1500:]
    return r.stdout
