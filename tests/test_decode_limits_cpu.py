"""What the decode operators refuse or hold without a GPU: buffers smaller than
their objects say."""
import pytest

from aps2026_b200 import decode, ops


def _table():
    import torch

    return torch.zeros(1, 2, dtype=torch.int32)


@pytest.mark.parametrize("change", [dict(pages=3), dict(pages=2 ** 32 - 2), dict(page_size=16), dict(kv_heads=2), dict(head_dim=128),
                                    dict(data=slice(1)), dict(data=(slice(None), slice(0, None, 2)))])
def test_a_cache_smaller_than_it_says_is_refused(change):
    import torch

    cache = decode.KVCache4(2, 8, 1, 64, "cpu")
    if "data" in change:
        change = dict(data=cache.data[change["data"]])
    for name, value in change.items():
        setattr(cache, name, value)
    k, i = torch.zeros(1, cache.kv_heads, cache.head_dim), torch.zeros(1, dtype=torch.int32)
    ws = type("Workspace", (), dict(buf=torch.zeros(8), bytes=32))()
    for call in (lambda: decode.kv4_append_gpu(k, k, i, i, cache, _table()),
                 lambda: decode.kv4_read_gpu(cache, _table(), i, i, k, k),
                 lambda: decode.attention_kv4_gpu(k, cache, _table(), i, k, ws=ws)):
        with pytest.raises(ops.InvalidArgument, match="cache: expected"):
            call()


# Experts with fp32 activations, error of the output relative to its size: a
# product is off by 2^-22 of itself three times at most (either operand's last
# part, the product of the low parts), apart from each other in sign; the
# gate, the up and the down product add up to three such sums.
EXPERTS = 2.0 ** -19


def _experts(x, gate_up, down, cut=lambda t: t):
    """One expert in 64 bits; cut: what its activations are held as."""
    import torch

    gate, up = (cut(x) @ gate_up.t()).chunk(2, 1)
    return cut(gate * torch.sigmoid(gate) * up) @ down.t()


@pytest.mark.parametrize("H,I", [(256, 40), (4096, 448), (1001, 333)])
def test_the_experts_bound_tells_16_bits_from_24(H, I):
    """What the bound is for: operands held to 24 bits pass it, to 16 or 17 do not."""
    import torch

    def held_to(bits):
        drop = 53 - bits
        return lambda t: (t.contiguous().view(torch.int64) >> drop << drop).view(torch.float64)

    g = torch.Generator().manual_seed(H)
    rand = lambda *s: torch.randn(s, generator=g, dtype=torch.float64)  # noqa: E731
    x, gate_up, down = rand(9, H), rand(2 * I, H) / H ** 0.5, rand(H, I) / I ** 0.5
    want = _experts(x, gate_up, down)
    off = lambda bits: float((_experts(x, gate_up, down, held_to(bits)) - want).norm() / want.norm())  # noqa: E731
    assert off(24) < EXPERTS and off(22) < EXPERTS
    assert off(17) > EXPERTS and off(16) > EXPERTS


@pytest.fixture
def pyext_builds(monkeypatch, tmp_path):
    """The extension module's builds, made by a compiler that only writes its output."""
    from aps2026_b200 import build

    runs = []

    def compile_(cmd, **_):
        runs.append(cmd)
        open(cmd[cmd.index("-o") + 1], "w").close()
        return type("Result", (), dict(returncode=0, stdout="", stderr=""))

    monkeypatch.setattr(build, "PYEXT_LIB", tmp_path / "_decode_calls.so")
    monkeypatch.setattr(build, "BUILD", tmp_path)
    monkeypatch.setattr(build.subprocess, "run", compile_)
    return runs


def test_the_extension_is_built_anew_for_another_torch(pyext_builds, monkeypatch):
    from aps2026_b200 import build

    build._build_pyext()
    build._build_pyext()
    assert len(pyext_builds) == 1
    monkeypatch.setattr(build.metadata, "version", lambda name: "0.0.1")
    build._build_pyext()
    build._build_pyext()
    assert len(pyext_builds) == 2


def test_the_library_is_built_without_torch(pyext_builds, monkeypatch, capsys):
    """A C program's user needs the library alone."""
    from aps2026_b200 import build

    def version(name):
        raise build.metadata.PackageNotFoundError(name)

    monkeypatch.setattr(build.metadata, "version", version)
    build._build_pyext()
    assert pyext_builds == [] and not build.PYEXT_LIB.exists()
    assert "torch" in capsys.readouterr().err


def test_experts_without_a_workspace_refuse_what_is_no_tensor():
    import torch

    x = torch.zeros(2, 8)
    for bad in (None, "x", [1.0]):
        with pytest.raises(ops.InvalidArgument):
            decode.moe_decode_gpu(bad, x, x, x.view(2, 2, 4), x)
        with pytest.raises(ops.InvalidArgument):
            decode.moe_decode_gpu(x, x, x, bad, x)
