"""The paged-cache operators' argument checks, without a GPU (nothing is launched)."""

import ctypes

import pytest
import torch

from liteweight_b200 import _native as nat
from liteweight_b200 import build as lwbuild
from liteweight_b200 import kernels
from liteweight_b200.kernels import paged

FAKE = 0x1000   # never dereferenced: validation fails first


@pytest.fixture(scope="module")
def lib():
    lwbuild.build()
    return nat.lib()


def cache_args(**kw):
    d = dict(k_pages=FAKE, v_pages=FAKE, k_strides=(8192, 2048, 128), v_strides=(8192, 2048, 128), n_pages=4,
             page_size=16, n_kv_heads=4, head_dim=128, dtype=0, batch=2, page_table=FAKE, table_stride=4,
             table_width=4, kv_lens=FAKE)
    d.update(kw)
    return paged.PagedCacheArgs(**d)


def attn_args(cache=None, **kw):
    d = dict(cache=cache or cache_args(), q=FAKE, q_strides=(1024, 128), out=FAKE, out_strides=(1024, 128), tokens=2,
             n_q_heads=8, q_offsets=None, window=0, sinks=0, scale=1.0)
    d.update(kw)
    return paged.PagedAttentionArgs(**d)


def rope_args(cache=None, **kw):
    d = dict(cache=cache or cache_args(), q=FAKE, k=FAKE, v=FAKE, q_strides=(1024, 128), k_strides=(512, 128),
             v_strides=(512, 128), q_out=FAKE, out_strides=(1024, 128), tokens=2, n_q_heads=8, rope_cos=FAKE,
             rope_sin=FAKE, rope_stride=128, rope_dtype=2, rope_rows=64, eps=1e-6)
    d.update(kw)
    return paged.QkNormRopeArgs(**d)


LONG = cache_args(table_width=1 << 16, table_stride=1 << 16)   # long enough that its decode needs scratch

BAD_CACHE = [
    (dict(page_size=24), 2), (dict(page_size=0), 2), (dict(page_size=8), 5), (dict(page_size=512), 5),
    (dict(head_dim=80), 5), (dict(dtype=2), 5), (dict(dtype=7), 5), (dict(n_kv_heads=0), 2), (dict(batch=-1), 2),
    (dict(k_pages=None), 1), (dict(v_pages=None), 1), (dict(kv_lens=None), 1), (dict(page_table=None), 1),
    (dict(k_pages=FAKE + 2), 4), (dict(v_strides=(8192, 2048, 129), ), 4), (dict(k_strides=(8192, 2048, -128)), 4),
    (dict(kv_lens=FAKE + 2), 4), (dict(table_width=1 << 27, page_size=64), 5),
]


@pytest.mark.parametrize("kw,status", BAD_CACHE)
def test_bad_caches_are_refused(lib, kw, status):
    bad = cache_args(**kw)
    assert lib.lw_qk_norm_rope(ctypes.byref(rope_args(bad)), None) == status
    assert lib.lw_paged_attention(ctypes.byref(attn_args(bad)), None) == status
    assert lib.lw_paged_attention_workspace_size(ctypes.byref(attn_args(bad))) == 0


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(out=None), 1), (dict(tokens=3), 2), (dict(n_q_heads=6), 2), (dict(n_q_heads=0), 2),
    (dict(sinks=-1), 2), (dict(scale=0.0), 2), (dict(scale=-1.0), 2), (dict(scale=float("nan")), 2),
    (dict(scale=float("inf")), 2), (dict(q=FAKE + 8), 4), (dict(out_strides=(1024, 130)), 4), (dict(tokens=-1), 2),
    (dict(cache=LONG, workspace=None), 7), (dict(cache=LONG, workspace=FAKE, workspace_bytes=256), 7),
    (dict(cache=LONG, workspace=FAKE + 16, workspace_bytes=1 << 30), 4),
    (dict(q_offsets=FAKE + 2), 4), (dict(q_offsets=FAKE, n_q_heads=4 * 65), 5),
])
def test_bad_attention_arguments_are_refused(lib, kw, status):
    assert lib.lw_paged_attention(ctypes.byref(attn_args(**kw)), None) == status


@pytest.mark.parametrize("kw,status", [
    (dict(q=None), 1), (dict(k=None), 1), (dict(v=None), 1), (dict(q_out=None), 1), (dict(rope_cos=None), 1),
    (dict(q_weight=FAKE), 1), (dict(k_weight=FAKE), 1), (dict(rope_dtype=1), 5), (dict(tokens=1), 2),
    (dict(rope_rows=-1), 2), (dict(k=FAKE + 4), 4), (dict(v_strides=(512, 4)), 4), (dict(rope_stride=12), 4),
    (dict(rope_sin=FAKE + 4), 4),
])
def test_bad_rope_arguments_are_refused(lib, kw, status):
    assert lib.lw_qk_norm_rope(ctypes.byref(rope_args(**kw)), None) == status


def test_empty_calls_do_nothing(lib):
    empty = cache_args(batch=0, kv_lens=None, page_table=None)
    assert lib.lw_paged_attention(ctypes.byref(attn_args(empty, tokens=0, q=None, out=None)), None) == 0
    assert lib.lw_qk_norm_rope(ctypes.byref(rope_args(empty, tokens=0, q=None)), None) == 0
    assert lib.lw_paged_attention(None, None) == 1
    assert lib.lw_qk_norm_rope(None, None) == 1


def test_status_string(lib):
    assert lib.lw_status_string(9) == b"page id, position or length out of range"


def test_bindings_mirror_the_structs(lib):
    for which, cls in ((5, paged.PagedCacheArgs), (6, paged.QkNormRopeArgs), (7, paged.PagedAttentionArgs)):
        assert lib.lw_struct_size(which) == ctypes.sizeof(cls)


def tensors(**kw):
    d = dict(q=torch.zeros(2, 8, 128, dtype=torch.float16), k_pages=torch.zeros(4, 4, 16, 128, dtype=torch.float16),
             v_pages=torch.zeros(4, 4, 16, 128, dtype=torch.float16),
             page_table=torch.zeros(2, 3, dtype=torch.int32), kv_lens=torch.zeros(2, dtype=torch.int32))
    d.update(kw)
    return d


@pytest.mark.parametrize("kw", [
    dict(q=torch.zeros(2, 8, 128)), dict(q=torch.zeros(2, 8 * 128, dtype=torch.float16)),
    dict(q=torch.zeros(3, 8, 128, dtype=torch.float16)), dict(q=torch.zeros(2, 6, 128, dtype=torch.float16)),
    dict(q=torch.zeros(2, 8, 64, dtype=torch.float16)),
    dict(q=torch.zeros(2, 128, 8, dtype=torch.float16).transpose(1, 2)),
    dict(v_pages=torch.zeros(4, 4, 32, 128, dtype=torch.float16)), dict(v_pages=torch.zeros(4, 4, 16, 128)),
    dict(k_pages=torch.zeros(4, 4, 16, 128), v_pages=torch.zeros(4, 4, 16, 128)),
    dict(page_table=torch.zeros(2, 3, dtype=torch.int64)), dict(kv_lens=torch.zeros(2, dtype=torch.int64)),
    dict(page_table=torch.zeros(3, 3, dtype=torch.int32)), dict(kv_lens=torch.zeros(4, dtype=torch.int32)[::2]),
    dict(page_table=torch.zeros(3, 2, dtype=torch.int32).t()), dict(window=0), dict(window=-3), dict(sinks=-1),
    dict(out=torch.zeros(2, 8, 64, dtype=torch.float16)), dict(out=torch.zeros(2, 8, 128)),
])
def test_attention_asserts(kw):
    with pytest.raises(AssertionError):
        kernels.paged_attention(**tensors(**kw))


@pytest.mark.parametrize("kw", [dict(window=2.5), dict(sinks="4"), dict(scale="x"), dict(q=None), dict(kv_lens=[1, 2])])
def test_attention_types(kw):
    with pytest.raises(TypeError):
        kernels.paged_attention(**tensors(**kw))


def test_prompt_attention_asserts():
    for off in (None, torch.zeros(3, dtype=torch.int64), torch.zeros(4, dtype=torch.int32),
                torch.zeros(6, dtype=torch.int32)[::2]):
        with pytest.raises(AssertionError):
            kernels.prompt_attention(q_offsets=off, **tensors())


def test_no_cpu_fallback():
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.paged_attention(**tensors())
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.prompt_attention(q_offsets=torch.zeros(3, dtype=torch.int32), **tensors())


def test_rope_asserts():
    base = tensors()
    q = base.pop("q")
    good = dict(q=q, k=q[:, :4], v=q[:, :4], cos=torch.zeros(9, 128), sin=torch.zeros(9, 128), **base)
    with pytest.raises(RuntimeError, match="CUDA"):
        kernels.qk_norm_rope(**good)
    w = torch.ones(128, dtype=torch.float16)
    for kw in (dict(k=q), dict(v=q[:, :2]), dict(cos=torch.zeros(9, 64)), dict(sin=torch.zeros(8, 128)),
               dict(cos=torch.zeros(9, 128, dtype=torch.float64), sin=torch.zeros(9, 128, dtype=torch.float64)),
               dict(cos=torch.zeros(9, 128, dtype=torch.bfloat16), sin=torch.zeros(9, 128, dtype=torch.bfloat16)),
               dict(q_weight=w), dict(k_weight=w), dict(q_weight=w.float(), k_weight=w.float()),
               dict(q_weight=w[:64], k_weight=w[:64]), dict(k=q[:1, :4], v=q[:1, :4]),
               dict(out=torch.zeros(2, 4, 128, dtype=torch.float16)),
               dict(q_offsets=torch.zeros(2, dtype=torch.int32))):
        with pytest.raises(AssertionError):
            kernels.qk_norm_rope(**{**good, **kw})


STUB_USE = """
from liteweight_b200 import _native as nat
import liteweight_b200.engine
try:
    nat.bind()
    print("bound")
except RuntimeError as e:
    print("refused:", e)
"""


@pytest.mark.parametrize("abi,grow,want", [(0, 0, "bound"), (1, 0, "refused"), (-1, 0, "refused"), (0, 8, "refused")])
def test_the_extension_module_takes_only_the_library_it_was_built_for(lib, tmp_path, abi, grow, want):
    """Against a stand-in library whose version, or one of whose structs, differs."""
    import os
    import subprocess
    import sys
    from pathlib import Path

    import liteweight_b200.engine  # noqa: F401  (registers the engine entry points)
    sizes = [lib.lw_struct_size(i) for i in range(8)]
    sizes[7] += grow
    src = tmp_path / "stub.c"
    src.write_text("".join(f"long {f}() {{ return 0; }}\n" for f in nat.declared_symbols()
                           if f not in ("lw_abi_version", "lw_struct_size")) +
                   f"int lw_abi_version(void) {{ return {lib.lw_abi_version() + abi}; }}\n"
                   f"unsigned long lw_struct_size(int i) {{ static unsigned long s[] = {{{', '.join(map(str, sizes))}}};"
                   " return s[i]; }\n")
    out = tmp_path / "stub.so"
    subprocess.run(["gcc", "-shared", "-fPIC", "-o", str(out), str(src)], check=True)
    got = subprocess.run([sys.executable, "-c", STUB_USE], env={**os.environ, "LW_B200_LIB": str(out)}, text=True,
                         capture_output=True, timeout=300, cwd=Path(__file__).resolve().parent.parent)
    assert got.stdout.startswith(want), got.stdout + got.stderr


def test_the_c_library_is_built_without_the_extension_module(tmp_path, monkeypatch):
    """A compiler or a torch that the Python module cannot be built with does not cost
    the C library, which needs neither; what failed is still raised, and built next time."""
    (tmp_path / "csrc").mkdir()
    src = tmp_path / "csrc" / "one.cu"
    src.write_text('extern "C" int lw_one(void) { return 1; }\n')
    monkeypatch.setattr(lwbuild, "CSRC", tmp_path / "csrc")
    monkeypatch.setattr(lwbuild, "LIB_DIR", tmp_path / "lib")
    for name, file in (("LIB", "liblw_b200.so"), ("BIND", "lw_bind.so"), ("STAMP", "liblw_b200.sha"),
                       ("BIND_STAMP", "lw_bind.sha")):
        monkeypatch.setattr(lwbuild, name, tmp_path / "lib" / file, raising=False)

    def no_torch(out):
        raise ImportError("no torch")

    for command in (lambda out: ["false"], no_torch, lambda out: ["/nonexistent/g++"]):
        monkeypatch.setattr(lwbuild, "_bind_command", command)
        lwbuild.LIB.unlink(missing_ok=True)
        with pytest.raises(RuntimeError, match="bind_paged.cpp"):
            lwbuild.build()
        assert ctypes.CDLL(str(lwbuild.LIB)).lw_one() == 1
        assert not lwbuild.BIND.exists() and not lwbuild.up_to_date()
    made = lwbuild.LIB.stat().st_mtime_ns
    monkeypatch.setattr(lwbuild, "_bind_command", lambda out: ["cp", str(src), str(out)])
    lwbuild.build()
    assert lwbuild.BIND.exists() and lwbuild.up_to_date()
    assert lwbuild.LIB.stat().st_mtime_ns == made   # not built again


def test_scales_are_finite_times_log2_e(lib):
    """The kernels' exponentials are of base 2: a scale that log2(e) takes past fp32 is refused too."""
    for scale, status in ((3.4e38, 2), (3.0e38, 2), (2.4e38, 2), (2.3e38, 1)):   # 1: goes on to q's pointer
        assert lib.lw_paged_attention(ctypes.byref(attn_args(scale=scale, q=None)), None) == status
