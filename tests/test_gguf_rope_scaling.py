"""What the GGUF reader makes of a file whose rotary positions are stretched (rope.scaling.*, rope.scale_linear, rope_freqs.weight).
Needs no GPU."""
import os
import struct
import subprocess

import numpy as np
import pytest

from litenn_b200 import capi
from test_gguf_reader import FIXTURE, HERE, ROOT, fixture


@pytest.fixture(scope="module")
def parse(qmm_lib, tmp_path_factory):
    where = tmp_path_factory.mktemp("gguf_rope")
    gxx = "/usr/bin/g++" if os.path.exists("/usr/bin/g++") else "g++"
    cuda, exe, lib = os.environ.get("CUDA_HOME", "/usr/local/cuda"), str(where / "gguf_rope_test"), os.path.join(ROOT, "litenn_b200")
    subprocess.run([gxx, "-std=c++17", "-O1", "-Wall", "-I", os.path.join(cuda, "include"), "-o", exe,
                    os.path.join(HERE, "native", "gguf_rope_test.cpp"), "-L", lib, "-lqmm_b200", "-L", os.path.join(cuda, "lib64"),
                    "-lcudart", "-Wl,-rpath," + lib, "-Wl,-rpath," + os.path.join(cuda, "lib64")], check=True)

    def run(meta=(), tensor=None, path=None):
        """A file with the given keys of `llama.rope.` and one tensor (type, shape, bytes) rope_freqs.weight."""
        if path is None:
            kvs = [fixture.kv("general.architecture", fixture.V_STR, fixture.gstr("llama")),
                   fixture.kv("general.alignment", fixture.V_U32, struct.pack("<I", fixture.ALIGN)),
                   fixture.kv("llama.context_length", fixture.V_U32, struct.pack("<I", 128))]
            for key, value in meta:
                kvs.append(fixture.kv("llama.rope." + key, fixture.V_STR, fixture.gstr(value)) if isinstance(value, str) else
                           fixture.kv("llama.rope." + key, fixture.V_U32, struct.pack("<I", value)) if isinstance(value, int) else
                           fixture.kv("llama.rope." + key, fixture.V_F32, struct.pack("<f", value)))
            directory, data = b"", b""
            if tensor:
                kind, shape, data = tensor
                directory = fixture.gstr("rope_freqs.weight") + struct.pack("<I", len(shape)) + \
                    b"".join(struct.pack("<Q", n) for n in reversed(shape)) + struct.pack("<IQ", kind, 0)
                data += b"\0" * (-len(data) % fixture.ALIGN)
            head = b"GGUF" + struct.pack("<IQQ", 3, 1 if tensor else 0, len(kvs)) + b"".join(kvs) + directory
            path = where / "f.gguf"
            path.write_bytes(head + b"\0" * (-len(head) % fixture.ALIGN) + data)
        r = subprocess.run([exe, str(path)], capture_output=True, text=True)
        if r.returncode == 3:
            return r.stdout.strip()
        assert r.returncode == 0, r.stdout + r.stderr
        v = r.stdout.split()
        return int(v[0]), [float(x) for x in v[1:5]], np.array(v[5:], dtype=np.float32)

    return run


def test_files_that_are_not_stretched(parse):
    for answer in (parse(path=FIXTURE), parse(), parse([("scaling.type", "none"), ("scaling.factor", 4.0)]), parse([("scale_linear", 1.0)])):
        kind, (factor, _, _, _), factors = answer
        assert kind == capi.ROPE_SCALE_NONE and len(factors) == 0


def test_linear(parse):
    for answer in (parse([("scaling.type", "linear"), ("scaling.factor", 4.0)]), parse([("scale_linear", 4.0)])):
        assert answer[0] == capi.ROPE_SCALE_LINEAR and answer[1][0] == 4.0


def test_yarn(parse):
    kind, values, _ = parse([("scaling.type", "yarn"), ("scaling.factor", 8.0), ("scaling.original_context_length", 4096)])
    assert kind == capi.ROPE_SCALE_YARN and values == [8.0, 4096.0, 32.0, 1.0]
    kind, values, _ = parse([("scaling.type", "yarn"), ("scaling.factor", 8.0), ("scaling.yarn_beta_fast", 16.0),
                             ("scaling.yarn_beta_slow", 2.0)])
    assert values == [8.0, 128.0, 16.0, 2.0]  # trained on what the file names as its context
    capi.rope_frequencies(64, 10000.0, scaling=capi.RopeScaling(kind, *values))


def test_frequency_factors(parse):
    f = np.linspace(1, 8, 32).astype(np.float32)
    kind, _, factors = parse(tensor=(fixture.T_F32, (32,), f.tobytes()))
    assert kind == capi.ROPE_SCALE_NONE
    np.testing.assert_array_equal(factors, f)


def test_what_is_not_known_is_refused(parse):
    assert "longrope" in parse([("scaling.type", "longrope"), ("scaling.factor", 4.0)])
    assert "scaling.factor" in parse([("scaling.type", "linear")])
    assert "rope_freqs" in parse(tensor=(fixture.T_F32, (4, 8), bytes(128)))
    assert "rope_freqs" in parse(tensor=(fixture.T_Q8_0, (32,), bytes(34)))
