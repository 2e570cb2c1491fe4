"""The paged cache's host side: refusals of the C ABI and of its Python form,
and the arithmetic that its formats rest on (no GPU work)."""
import ctypes
import shutil
import subprocess
from pathlib import Path

import numpy as np
import pytest
import torch

from inferq_b200 import kv

ROOT = Path(__file__).resolve().parents[1]


@pytest.fixture(scope="module")
def L():
    return kv._lib_()


def err(L):
    return L.iq_last_error().decode()


@pytest.mark.parametrize("args,code,text", [
    ((8, 2, 256, 64, 4), -4, "cache format"),
    ((24, 2, 96, 64, 4), -4, "head size"),
    ((24, 0, 256, 64, 4), -1, "KV heads"),
    ((24, 257, 256, 64, 4), -1, "KV heads"),
    ((24, 2, 256, 8, 4), -1, "pages of 8"),
    ((24, 2, 256, 48, 4), -1, "pages of 48"),
    ((1, 2, 256, 512, 4), -1, "pages of 512"),
    ((1, 2, 256, 64, 0), -1, "pool of 0"),
    ((1, 2, 256, 64, 1 << 31), -1, "pool of"),
])
def test_create_refuses(L, args, code, text):
    h = ctypes.c_void_p()
    assert L.iq_kv_create(*args, ctypes.byref(h)) == code
    assert text in err(L) and not h.value


def test_null_handles_are_errors(L):
    h, b, at, n = ctypes.c_void_p(), kv._Batch(), kv._Attn(0, 16, 0.0, 0, 0, 0), ctypes.c_size_t()
    assert L.iq_kv_create(24, 2, 256, 64, 4, None) == -1
    assert L.iq_kv_bytes(None, ctypes.byref(ctypes.c_int64())) == -1
    assert L.iq_kv_append(h, b, 0, None, 0, 0, None, 0, 0, None) == -1
    assert L.iq_kv_read(h, b, 0, None, 0, 0, None, 0, 0, None) == -1
    assert L.iq_kv_attend_workspace(h, b, at, ctypes.byref(n)) == -1
    assert L.iq_kv_attend(h, b, at, None, 0, 0, None, 0, 0, None, 0, None) == -1
    assert L.iq_kv_status(h, None) == -1
    L.iq_kv_destroy(None)


def test_python_form_refuses_tensors_of_the_host():
    t, p = torch.zeros(1, 4, dtype=torch.int32), torch.zeros(1, dtype=torch.int32)
    with pytest.raises(ValueError, match="CUDA"):
        kv.KvBatch(t, p)
    with pytest.raises(ValueError, match="int32"):
        kv.KvBatch(t.long(), p)
    with pytest.raises(ValueError, match="dimensions"):
        kv.KvBatch(t[0], p)
    with pytest.raises(ValueError, match="cache format"):
        kv.KvCache(2, 256, 4, format="q4")


def test_an_i8_vector_read_back_as_f32_is_written_to_the_same_codes_and_scale():
    """Export and import of a cache lose nothing: with scale s = rn(a / 127),
    the largest value reads back as rn(127 s), which gives the scale s again
    (every mantissa; s scales by powers of two)."""
    a = (np.arange(1 << 23, dtype=np.uint32) | np.uint32(127 << 23)).view(np.float32)
    s = (a / np.float32(127)).astype(np.float32)
    back = (np.float32(127) * s).astype(np.float32)
    assert np.array_equal((back / np.float32(127)).astype(np.float32), s)


def test_code_borders_are_found_in_f32():
    """The f32 quotient is at most 2^-15 from the real one, so a code that it
    leaves at least that far from a border is the right one."""
    r = np.random.default_rng(0)
    amax = np.exp2(r.uniform(-60, 60, 1 << 20)).astype(np.float32)
    x = (amax * r.uniform(-1, 1, amax.size)).astype(np.float32)
    q = (x * np.float32(127) * (np.float32(1) / amax)).astype(np.float32)
    assert np.abs(q.astype(np.float64) - 127.0 * x.astype(np.float64) / amax).max() < 2.0 ** -15


def _split_cases():
    r = np.random.default_rng(7)
    cases = [  # heads kv_heads page cols rows position window sinks chunk max_rows
        (16, 2, 64, 1, 1, 0, 0, 0, 0, 1), (16, 2, 64, 16, 4, 1000, 0, 0, 0, 4), (16, 2, 16, 5, 80, 0, 0, 0, 64, 0),
        (7, 1, 32, 9, 33, 200, 50, 3, 64, 33), (16, 2, 64, 20, 3, 1270, 1, 0, 64, 3), (16, 2, 64, 4, 5, -3, 0, 0, 64, 5),
        (16, 2, 64, 4, 5, -9, 7, 2, 64, 5), (16, 2, 64, 2, 9, 125, 0, 0, 64, 9), (4, 4, 128, 8, 70, 900, 64, 64, 128, 1),
        (16, 2, 64, 0, 2, 0, 0, 0, 64, 2), (128, 1, 16, 40, 4, 600, 100, 130, 64, 4),
    ]
    most = 2**31 - 1  # the types' ends
    cases += [(16, 2, 64, 9, rows, p, window, sinks, chunk, max_rows) for rows, p in ((1, 300), (5, -2), (70, 300))
              for window, sinks in ((most, 0), (most, most), (1, most), (most, 70)) for chunk in (0, 64, most - 63)
              for max_rows in (0, most)]
    for _ in range(150):
        kv_heads = int(r.choice([1, 2, 3]))
        page, cols, rows = int(r.choice([16, 32, 64, 128, 256])), int(r.integers(1, 12)), int(r.integers(1, 90))
        window = int(r.choice([0, 1, int(r.integers(1, 40)), int(r.integers(1, 700))]))
        cases.append((kv_heads * int(r.choice([1, 2, 7, 8, 16])), kv_heads, page, cols, rows,
                      int(r.integers(-5, max(1, cols * page - rows + 20))), window, int(r.choice([0, 1, 64, int(r.integers(0, 300))])),
                      int(r.choice([0, 64, 128, 256, 192])), int(r.choice([0, 1, rows]))))
    return cases


def test_the_split_covers_every_visible_token_once(tmp_path):
    """kv_split.cuh compiled for the host: brute force over rows and tokens."""
    nvcc = next((c for c in ("/usr/local/cuda/bin/nvcc", shutil.which("nvcc")) if c and Path(c).exists()), None)
    if nvcc is None:
        pytest.skip("nvcc not found")
    exe = tmp_path / "kv_split_check"
    build = subprocess.run([nvcc, "-std=c++17", "-O1", "-gencode", "arch=compute_100a,code=sm_100a", "--expt-relaxed-constexpr",
                            "-I" + str(ROOT / "inferq_b200" / "csrc"), "-I" + str(ROOT / "include"),
                            str(ROOT / "tests" / "native" / "kv_split_check.cu"), "-o", str(exe)],
                           capture_output=True, text=True, timeout=600)
    assert build.returncode == 0, build.stderr
    for case in _split_cases():
        run = subprocess.run([str(exe), *map(str, case)], capture_output=True, text=True, timeout=60)
        assert run.returncode == 0, (case, run.stdout)
