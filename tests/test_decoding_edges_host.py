"""Host side of the cached-decoding operators, edges, without a GPU."""

import pytest
import torch

from voyager_b200 import fp8block


def test_quantize_weight_of_a_block_whose_scale_underflows():
    """A block whose largest magnitude over 448 is 0 in float32 counts as a
    block of zeros (scale 1, codes 0), as quantize takes it; the least scale
    that is not 0 is used."""
    w = torch.zeros(130, 260)
    w[0, 0] = 2.0 ** -142      # / 448 is below half of the least float32, 2^-149
    w[3, 130] = 2.0 ** -140    # / 448 = 1.14 * 2^-149
    w[129, 259] = -1.0
    codes, scale = fp8block.quantize_weight(w)
    f = codes.float()
    assert not bool(f.isnan().any())
    assert scale[0, 0] == 1 and not bool(f[:128, :128].any())
    assert scale[0, 1] == 2.0 ** -149 and f[3, 130] == 448  # 2^9 saturates
    assert scale[1, 2] == 1 / 448 and f[129, 259] == -448
    assert scale[0, 2] == 1 and scale[1, 0] == 1 and scale[1, 1] == 1


def test_a_norm_needs_its_weight():
    """Without a weight there is no norm to compute: None is refused, not taken
    as `quantize`."""
    for residual in (None, torch.ones(2, 128)):
        with pytest.raises(TypeError, match="weight"):
            fp8block.rmsnorm_quantize(torch.ones(2, 128), None, 1e-5, residual)


def test_the_binding_is_built_again_for_another_torch_or_python(tmp_path, monkeypatch):
    """_decode.so is up to date only for the torch, the Python and the command
    that it was built with; a build that fails leaves no record."""
    import os
    import subprocess

    import torch as real
    from voyager_b200 import build

    runs = []

    def run(cmd, **kw):
        runs.append(cmd)
        if fails:
            return subprocess.CompletedProcess(cmd, 1, "", "no")
        open(cmd[cmd.index("-o") + 1], "w").close()
        return subprocess.CompletedProcess(cmd, 0, "", "")

    fails = False
    monkeypatch.setattr(build, "PY_OUT", str(tmp_path / "_decode.so"))
    monkeypatch.setattr(build, "BUILD", str(tmp_path))
    monkeypatch.setattr(build.subprocess, "run", run)

    def builds():
        n = len(runs)
        build._build_binding(False)
        return len(runs) - n

    assert builds() == 1 and builds() == 0
    monkeypatch.setattr(real, "__version__", "9.9.9")
    assert builds() == 1 and builds() == 0
    monkeypatch.setattr(build.sysconfig, "get_config_var", lambda name: "cpython-399-" + name)
    assert builds() == 1 and builds() == 0
    monkeypatch.setattr(real, "compiled_with_cxx11_abi", lambda: False)
    assert builds() == 1 and builds() == 0
    assert "-D_GLIBCXX_USE_CXX11_ABI=0" in runs[-1]
    os.utime(build.PY_OUT, (1, 1))  # older than its source
    assert builds() == 1 and builds() == 0
    fails = True
    monkeypatch.setattr(real, "__version__", "9.9.10")
    for _ in range(2):
        with pytest.raises(RuntimeError, match="g\\+\\+ failed"):
            build._build_binding(False)
    fails = False
    assert builds() == 1 and builds() == 0
    os.remove(build.PY_OUT)
    assert builds() == 1


@pytest.mark.parametrize("page", [32, 64, 128])
def test_attention_refuses_tables_whose_keys_leave_31_bits(page):
    """Keys are counted in 31 bits, up to 2^14 past a table's end (the block
    table is read two batches of tiles ahead): a longer table is refused before
    any launch."""
    import ctypes

    from voyager_b200 import _lib

    lib = _lib.load()
    P = 0x1000  # never dereferenced

    def go(width):
        floats, counters = ctypes.c_int64(), ctypes.c_int64()
        st = lib.vq_attn_kv8_workspace(1, 1, 1, 1, 128, page, width, ctypes.byref(floats), ctypes.byref(counters))
        assert st in (0, 1)
        floats.value, counters.value = 1 << 40, 1 << 40
        strides = (ctypes.c_int64 * 3)(128, 128, 128)
        return lib.vq_attn_kv8(P, strides, 1, 1, 1, 1, 128, P, P, P, P, 1, page, P, width, P, None, 1.0, P, floats.value,
                               P, counters.value, P, None)

    top = (1 << 31) // page
    for width in (top, top - 1, top - (1 << 14) // page + 1, 1 << 62):
        assert go(width) == 1, width
