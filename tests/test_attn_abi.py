"""The attention entry points on the CPU: struct layouts, host-side refusals (made
before any device call), workspace sizes, the binding's checks and streams, and
what a call launches."""
from __future__ import annotations

import ctypes
import inspect
import math
import pathlib
import shutil
import subprocess
import types
from functools import partial

import pytest

import launch_record
from r9v_amd import attn, ffi

torch = pytest.importorskip("torch")
from test_fp8_abi import ALIGN, FAKE, INVALID, NULL, UNSUPPORTED, WORKSPACE, lib, refused  # noqa: E402
from test_streams import spy, stream  # noqa: E402, F401

ROOT = pathlib.Path(__file__).resolve().parent.parent
STRUCTS = {"r9vx_rope_kv_static": ffi.RopeKvStatic, "r9vx_rope_kv_args": ffi.RopeKvArgs, "r9vx_attn_static": ffi.AttnStatic,
           "r9vx_attn_args": ffi.AttnArgs}


def test_struct_layouts(tmp_path):
    lines = ["#include <stdio.h>", "#include <stddef.h>", '#include "r9vx_attn.h"', "int main(void){"]
    for name, cls in STRUCTS.items():
        lines.append(f'printf("%zu\\n", sizeof({name}));')
        lines += [f'printf("%zu\\n", offsetof({name}, {f}));' for f, _ in cls._fields_]
    (tmp_path / "s.c").write_text("\n".join([*lines, "return 0;}"]))
    subprocess.run(["gcc", "-std=c11", "-I", str(ROOT / "include"), str(tmp_path / "s.c"), "-o", str(tmp_path / "s")], check=True)
    got = [int(v) for v in subprocess.run([str(tmp_path / "s")], capture_output=True, text=True, check=True).stdout.split()]
    want = []
    for cls in STRUCTS.values():
        want += [ctypes.sizeof(cls), *(getattr(cls, f).offset for f, _ in cls._fields_)]
    assert got == want


@pytest.mark.parametrize("cls,pointers,rest", [(ffi.RopeKvArgs, attn._ROPE_POINTERS, attn._ROPE_REST), (ffi.AttnArgs, attn._ATTN_POINTERS, attn._ATTN_REST)])
def test_packed_arguments_are_the_struct(cls, pointers, rest):
    values = list(range(1, 1 + sum(getattr(t, "_length_", 1) for _, t in cls._fields_)))
    n = len(pointers.unpack(bytes(pointers.size)))
    data = pointers.pack(*values[:n]) + rest.pack(*values[n:])
    assert len(data) == ctypes.sizeof(cls)
    s = cls.from_buffer_copy(data)
    got = []
    for name, _ in cls._fields_:
        v = getattr(s, name)
        got += list(v) if isinstance(v, ctypes.Array) else [v]
    assert got == values


APART = {n: FAKE + (i << 32) for i, n in enumerate(("q", "k", "v", "positions", "freqs", "q_out", "k_cache", "v_cache", "slots", "status"))}


def rope(**kw):
    st = dict(heads=8, kv_heads=2, head_dim=128, rot=64, interleaved=0, page_size=16, in_dtype=ffi.BF16, out_dtype=ffi.BF16,
              amplitude_bits=attn._bits(1.0))
    a = dict(APART, status=None, q_stride=(1536, 128), k_stride=(1536, 128), v_stride=(1536, 128), q_out_stride=(1024, 128),
             k_cache_stride=(4096, 256, 128), v_cache_stride=(4096, 256, 128), pages=10, t=4)
    for name, v in kw.items():
        (st if name in st else a)[name] = v
    return ffi.RopeKvStatic(**st), ffi.RopeKvArgs(**a)


NO_CACHE = dict(kv_heads=0, k=None, v=None, k_cache=None, v_cache=None, slots=None)


@pytest.mark.parametrize("kw,code,text", [
    (dict(heads=0), INVALID, "heads=0"), (dict(heads=1025), INVALID, "heads"), (dict(head_dim=132), UNSUPPORTED, "multiple of 8"),
    (dict(head_dim=520), UNSUPPORTED, "at most 512"), (dict(rot=0), INVALID, "rot=0"), (dict(rot=24), INVALID, "rot=24"), (dict(rot=144), INVALID, "rot=144"),
    (dict(interleaved=2), INVALID, "interleaved"), (dict(page_size=24), UNSUPPORTED, "page_size=24"), (dict(page_size=0), UNSUPPORTED, "page_size"),
    (dict(in_dtype=ffi.I8), UNSUPPORTED, "in_dtype"), (dict(out_dtype=ffi.F16), UNSUPPORTED, "out_dtype"), (dict(out_dtype=ffi.F32), UNSUPPORTED, "out_dtype"),
    (dict(amplitude_bits=attn._bits(math.inf)), INVALID, "amplitude"), (dict(t=(1 << 23) + 1), UNSUPPORTED, "2^23"),
    (dict(q=None), NULL, "q, q_out"), (dict(freqs=None), NULL, "freqs"), (dict(k=None), NULL, "k, v"), (dict(slots=None), NULL, "slots"),
    (dict(NO_CACHE, slots=FAKE), INVALID, "without kv_heads"), (dict(q=FAKE + 8), ALIGN, "16-byte"), (dict(slots=APART["slots"] + 4), ALIGN, "8-byte"),
    (dict(positions=APART["positions"] + 2), ALIGN, "4-byte"), (dict(q_stride=(1537, 128)), ALIGN, "q: a stride of 1537"),
    (dict(k_cache_stride=(4096, 260, 128)), ALIGN, "k_cache: a stride of 260"), (dict(v_stride=(1 << 41, 128)), INVALID, "2^40"),
    (dict(q_out=APART["q"]), INVALID, "q_out must not overlap q"), (dict(q_out=APART["k"]), INVALID, "overlap k or v"),
    (dict(q_out=APART["q"], q_out_stride=(1536, 128), in_dtype=ffi.F32), INVALID, "q_out must not overlap q"),
    (dict(k_cache=APART["q"] + 4096), INVALID, "cache must not overlap"), (dict(v_cache=APART["q_out"]), INVALID, "cache must not overlap"),
    (dict(v_cache=APART["slots"]), INVALID, "cache must not overlap positions"), (dict(q_out=APART["freqs"]), INVALID, "positions, freqs or slots"),
    (dict(q_out_stride=(0, 128)), INVALID, "rows of q_out overlap"), (dict(k_cache_stride=(4096, 128, 128)), INVALID, "rows of the cache overlap"),
    (dict(v_cache_stride=(2048, 256, 128)), INVALID, "rows of the cache overlap"), (dict(v_cache=APART["k_cache"]), INVALID, "rows of the cache overlap")])
def test_rope_refusals(kw, code, text):
    refused(lib.r9vx_rope_kv_launch, *rope(**kw), code=code, text=text)


def test_rope_without_rows():
    for kw in (dict(t=0), dict(NO_CACHE, t=0), dict(t=0, q=None, k=None)):
        st, a = rope(**kw)
        assert lib.r9vx_rope_kv_launch(ctypes.byref(st), ctypes.byref(a), None) == 0
    assert lib.r9vx_rope_kv_launch(None, None, None) == NULL


ATTN = {n: FAKE + (i << 36) for i, n in enumerate(("q", "k_cache", "v_cache", "table", "lengths", "offsets", "starts", "prefix", "slopes", "out",
                                                   "workspace", "status"))}


def attention(decode, **kw):
    st = dict(b_bucket=4, t_bucket=2 if decode else 100, len_bucket=500, heads=8, kv_heads=2, head_dim=128, page_size=16, dtype=ffi.BF16, causal=1,
              window=0, scale_bits=attn._bits(0.1), softcap_bits=0)
    a = dict(ATTN, starts=None, prefix=None, slopes=None, status=None, offsets=None if decode else ATTN["offsets"], q_stride=(2048, 1024, 128),
             out_stride=(2048, 1024, 128), k_stride=(4096, 256, 128), v_stride=(4096, 256, 128), table_stride=40, pages=1000, b=3, t=0 if decode else 70)
    for name, v in kw.items():
        (st if name in st else a)[name] = v
    return ffi.AttnStatic(**st), ffi.AttnArgs(**a)


BOTH = [
    (dict(heads=9), INVALID, "multiple of kv_heads"), (dict(kv_heads=0), INVALID, "kv_heads=0"), (dict(heads=2048), UNSUPPORTED, "1024"),
    (dict(head_dim=80), UNSUPPORTED, "head_dim=80"), (dict(head_dim=0), UNSUPPORTED, "head_dim"), (dict(page_size=48), UNSUPPORTED, "page_size"),
    (dict(page_size=4), UNSUPPORTED, "page_size"), (dict(dtype=ffi.F32), UNSUPPORTED, "dtype"), (dict(causal=2), INVALID, "causal"),
    (dict(scale_bits=attn._bits(math.nan)), INVALID, "scale"), (dict(softcap_bits=attn._bits(-1.0)), INVALID, "softcap"),
    (dict(softcap_bits=attn._bits(math.inf)), INVALID, "softcap"), (dict(softcap_bits=attn._bits(1e-45)), INVALID, "scale / softcap"),
    (dict(len_bucket=(1 << 30) + 1), UNSUPPORTED, "2^30"), (dict(b_bucket=1 << 16), UNSUPPORTED, "2^16"), (dict(b=5), INVALID, "b=5"),
    (dict(q=None), NULL, "q, k_cache"), (dict(out=None), NULL, "out"), (dict(table=None), NULL, "table"), (dict(lengths=None), NULL, "lengths"),
    (dict(pages=0), INVALID, "no page"), (dict(pages=(1 << 31) + 1), UNSUPPORTED, "2^31"), (dict(k_cache=ATTN["k_cache"] + 8), ALIGN, "16-byte"),
    (dict(table=ATTN["table"] + 1), ALIGN, "4-byte"), (dict(status=ATTN["status"] + 2), ALIGN, "4-byte"),
    (dict(q_stride=(2048, 1028, 128)), ALIGN, "q: a stride"), (dict(out_stride=(2048, 1024, 1)), ALIGN, "out: a stride"),
    (dict(v_stride=(4097, 256, 128)), ALIGN, "v_cache: a stride"), (dict(k_stride=(4096, 1 << 27, 128)), UNSUPPORTED, "2^27 elements"), (dict(workspace=None, len_bucket=4096, table_stride=256), WORKSPACE, "workspace"),
    (dict(workspace=ATTN["workspace"] + 16), ALIGN, "256-byte"), (dict(table_stride=31), INVALID, "columns apart"),
    (dict(out=ATTN["q"]), INVALID, "out must not overlap"), (dict(out=ATTN["v_cache"] + 4096), INVALID, "out must not overlap"),
    (dict(out=ATTN["lengths"]), INVALID, "out must not overlap"), (dict(workspace=ATTN["out"], len_bucket=600), INVALID, "workspace must not overlap"),
    (dict(workspace=ATTN["table"], len_bucket=600), INVALID, "workspace must not overlap"),
    (dict(out_stride=(2048, 0, 128)), INVALID, "rows of out overlap"), (dict(out_stride=(2048, 1024, 120)), INVALID, "rows of out overlap")]
DECODE = [(dict(t_bucket=0), UNSUPPORTED, "1 to 8"), (dict(t_bucket=9), UNSUPPORTED, "1 to 8"), (dict(causal=0), INVALID, "causal"), (dict(t=2), INVALID, "t=2"),
          (dict(offsets=ATTN["offsets"]), INVALID, "prefill's"), (dict(prefix=ATTN["prefix"]), INVALID, "prefill's"),
          (dict(b_bucket=65535, heads=1024, kv_heads=512), UNSUPPORTED, "more tiles than a launch"),
          (dict(b_bucket=65535, t_bucket=8, heads=256, kv_heads=1, len_bucket=1 << 23), UNSUPPORTED, "more rows to join"),
          (dict(out_stride=(0, 1024, 128)), INVALID, "rows of out overlap"), (dict(out_stride=(1024, 1024, 128)), INVALID, "rows of out overlap")]
PREFILL = [(dict(t_bucket=(1 << 24) + 1), UNSUPPORTED, "2^24"), (dict(t=101), INVALID, "t=101"), (dict(offsets=None), NULL, "offsets"),
           (dict(causal=0, prefix=ATTN["prefix"]), INVALID, "prefix without"), (dict(t_bucket=1 << 24, heads=1024, kv_heads=4), UNSUPPORTED, "more tiles")]


@pytest.mark.parametrize("decode,kw,code,text", [(d, *x) for d in (True, False) for x in BOTH] + [(True, *x) for x in DECODE] + [(False, *x) for x in PREFILL])
def test_attention_refusals(decode, kw, code, text):
    refused(lib.r9vx_attn_decode_launch if decode else lib.r9vx_attn_prefill_launch, *attention(decode, **kw), code=code, text=text)


def test_attention_without_rows():
    for decode, kw in ((True, dict(b=0)), (False, dict(b=0)), (False, dict(t=0)), (True, dict(b=0, q=None, out=None, table=None, pages=0))):
        st, a = attention(decode, **kw)
        assert (lib.r9vx_attn_decode_launch if decode else lib.r9vx_attn_prefill_launch)(ctypes.byref(st), ctypes.byref(a), None) == 0
    assert lib.r9vx_attn_decode_launch(None, None, None) == NULL and lib.r9vx_attn_prefill_launch(None, None, None) == NULL


def test_workspace_sizes():
    """Parts only where the rows do not fill the card, and none of a static that is refused."""
    def size(decode, **kw):
        return (attn.decode_workspace_bytes if decode else attn.prefill_workspace_bytes)(attention(decode, **kw)[0])

    for decode in (True, False):
        assert size(decode, len_bucket=16) == 0
        one = size(decode, b_bucket=1, len_bucket=1 << 17)
        rows = 2 * 8 if decode else 100 * 8
        assert one > 0 and one % (rows * (4 * 128 + 8)) == 0
        assert size(decode, head_dim=100) == 0
    assert size(True, b_bucket=2000) == 0 and size(False, t_bucket=100000) == 0
    assert lib.r9vx_attn_decode_workspace_bytes(None) == 0 and lib.r9vx_attn_prefill_workspace_bytes(None) == 0


# ------------------------------------------------------------------ the binding

def z(*shape, dtype=torch.float32):
    return torch.zeros(shape, dtype=dtype)


B, I, L, D = torch.bfloat16, torch.int32, torch.int64, torch.float64
CACHE = [z(9, 16, 2, 64, dtype=B) for _ in range(2)]
CALLS = {
    "rope_kv": partial(attn.rope_kv, z(4, 8, 64, dtype=B), z(4, 2, 64, dtype=B), z(4, 2, 64, dtype=B), z(4, dtype=I), z(16, dtype=D), *CACHE, z(4, dtype=L)),
    "rope": partial(attn.rope, z(4, 8, 64), z(4, dtype=I), z(16, dtype=D)),
    "decode": partial(attn.decode, z(3, 1, 8, 64, dtype=B), *CACHE, z(3, 4, dtype=I), z(3, dtype=I)),
    "prefill": partial(attn.prefill, z(30, 8, 64, dtype=B), *CACHE, z(3, 4, dtype=I), z(3, dtype=I), z(4, dtype=I)),
}


@pytest.fixture
def on_cpu(spy, monkeypatch):  # noqa: F811
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 0)
    return spy


@pytest.mark.parametrize("name", CALLS)
def test_memory_of_a_call_belongs_to_its_stream(name, on_cpu, monkeypatch):
    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    with on_cpu:
        CALLS[name]()
    assert on_cpu.seen and {s for _, s in on_cpu.seen} == {0} and on_cpu.kept == []
    del on_cpu.seen[:]
    with on_cpu:
        out = CALLS[name](stream=stream(7))
    assert on_cpu.seen and {s for _, s in on_cpu.seen} == {7}
    assert (out.data_ptr(), 0) in on_cpu.kept


def test_every_call_with_a_stream_is_here():
    names = {n for n, f in inspect.getmembers(attn, inspect.isfunction)
             if f.__module__ == attn.__name__ and not n.startswith("_") and "stream" in inspect.signature(f).parameters}
    assert names == set(CALLS)


def meta(*shape, dtype=torch.float32):
    return torch.empty(shape, dtype=dtype, device="meta")


@pytest.mark.parametrize("name,args,kw,text", [
    ("decode", {0: z(3, 8, 64, dtype=B)}, {}, "dimensions"), ("decode", {0: z(3, 1, 8, 64)}, {}, "q is torch.float32"), ("decode", {0: z(3, 1, 8, 96, dtype=B)}, {}, "q has shape"),
    ("decode", {2: z(9, 16, 2, 96, dtype=B)}, {}, "v_cache has shape"), ("decode", {1: z(9, 16, 2, 64)}, {}, "k_cache is"), ("decode", {1: z(9, 16, 64, 2, dtype=B).transpose(2, 3)}, {}, "dense"),
    ("decode", {3: z(2, 4, dtype=I)}, {}, "2 rows"), ("decode", {3: z(3, 4, dtype=L)}, {}, "table is"), ("decode", {}, dict(len_bucket=65), "len_bucket=65"),
    ("decode", {}, dict(out=z(3, 1, 8, 64)), "out is"), ("decode", {}, dict(out=z(3, 2, 8, 64, dtype=B)), "out has shape"),
    ("decode", {}, dict(workspace=z(16, dtype=torch.uint8)), "workspace of 16"), ("decode", {}, dict(window=1 << 32), "32 bits"), ("decode", {}, dict(window=-1), "32 bits"),
    ("decode", {}, dict(b_bucket=1 << 32), "32 bits"), ("decode", {}, dict(scale=1e300), "no f32"), ("decode", {}, dict(scale=z(1)), "no number"),
    ("prefill", {0: z(30, 8, 64)}, {}, "q is"), ("prefill", {}, dict(t_bucket=1 << 32), "32 bits"), ("prefill", {}, dict(softcap="a"), "no number"), ("prefill", {5: None}, {}, "offsets are required"),
    ("rope_kv", {1: z(4, 2, 64)}, {}, "k is torch.float32"), ("rope_kv", {2: z(4, 3, 64, dtype=B)}, {}, "v has shape"), ("rope_kv", {0: z(4, 8, 96, dtype=B)}, {}, "head_dim is 64"), ("rope_kv", {1: z(4, 3, 64, dtype=B)}, {}, "k has shape"),
    ("rope_kv", {}, dict(q_out=z(4, 8, 64)), "q_out is"), ("rope", {0: z(4, 8, 64, dtype=D)}, {}, "x is torch.float64"), ("rope", {}, dict(out=z(4, 8, 64, dtype=B)), "out is")])
def test_binding_refusals(name, args, kw, text, on_cpu, monkeypatch):
    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    call = CALLS[name]
    values = list(call.args)
    for i, v in args.items():
        values[i] = v
    with pytest.raises(ffi.R9vxError, match=text):
        call.func(*values, **kw)


def test_operands_of_another_device(on_cpu, monkeypatch):
    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    monkeypatch.setattr(torch.Tensor, "get_device", lambda t: 1 if t is CACHE[1] else 0)
    for name in ("decode", "prefill", "rope_kv"):
        with pytest.raises(ffi.R9vxError, match="v_cache is on cuda:1"):
            CALLS[name]()


@pytest.mark.parametrize("name", CALLS)
def test_a_stream_of_another_device_is_refused(name, on_cpu, monkeypatch):
    import test_streams

    monkeypatch.setattr(attn.ffi, "_fp8_operands", lambda *o: 0)
    monkeypatch.setattr(ffi, "_raw_stream", test_streams.RAW_STREAM)
    other = stream(8)
    other.device = torch.device("cuda", 1)
    with pytest.raises(ffi.R9vxError, match="stream is of cuda:1"):
        CALLS[name](stream=other)


def test_frequencies():
    f, a = attn.rope_freqs(64, base=1e4, device="cpu")
    assert f.dtype is torch.float64 and a == 1.0
    assert torch.allclose(f, torch.tensor([1e4 ** (-i / 32) for i in range(32)], dtype=torch.float64), rtol=1e-15)
    g, a = attn.rope_freqs(64, base=1e4, scaling="linear", factor=4.0, device="cpu")
    assert torch.equal(g, f / 4) and a == 1.0
    g, a = attn.rope_freqs(64, base=1e4, scaling="yarn", factor=8.0, original_length=4096, device="cpu")
    assert a == 1.0 + 0.1 * math.log(8.0)
    turns = 4096 * f / (2 * math.pi)
    # whole pairs beside the ramp's ends: it starts at the pair below that of 32 turns and ends at the one above that of 1
    assert torch.equal(g[turns > 45], f[turns > 45]) and torch.equal(g[turns < 0.7], f[turns < 0.7] / 8)
    between = g / f
    assert ((between[1:] - between[:-1]) <= 0).all()
    d = [1.0 + i for i in range(32)]
    g, _ = attn.rope_freqs(64, base=1e4, factors=d, device="cpu")
    assert torch.allclose(g, f / torch.tensor(d, dtype=torch.float64), rtol=1e-15)
    for kw, text in ((dict(rot=20), "rot=20"), (dict(rot=64, base=1.0), "base"), (dict(rot=64, scaling="other"), "scaling"), (dict(rot=64, factor=0.5), "factor"),
                     (dict(rot=64, scaling="yarn", factor=2.0), "original_length"), (dict(rot=64, factors=[1.0]), "1 factors")):
        with pytest.raises(ffi.R9vxError, match=text):
            attn.rope_freqs(device="cpu", **kw)


# ------------------------------------------------------------------ launches

CHILD = '''
def attn(decode, threads=None, **kw):
    st = dict(b_bucket=4, t_bucket=1 if decode else 100, len_bucket=4096, heads=8, kv_heads=2, head_dim=128, page_size=16, dtype=ffi.BF16, causal=1,
              window=0, scale_bits=0x3F800000, softcap_bits=0)
    st.update(kw)
    token = st["heads"] * st["head_dim"]
    rows = (st["t_bucket"] * token, token, st["head_dim"])
    a = ffi.AttnArgs(*APART[:5], None if decode else APART[5], None, None, None, APART[6], APART[7], None, rows, rows,
                     (4096, 256, 128), (4096, 256, 128), 1 << 20, 1000, st["b_bucket"], 0 if decode else st["t_bucket"], 0)
    f = L.r9vx_attn_decode_launch if decode else L.r9vx_attn_prefill_launch
    return f(ctypes.byref(ffi.AttnStatic(**st)), ctypes.byref(a), None)
'''


@pytest.mark.skipif(not launch_record.LIB.exists() or shutil.which("gcc") is None, reason="needs the built libr9vx.so and gcc")
def test_launches(tmp_path, monkeypatch):
    """Parts and their join where the rows are few; a grid whose threads 32 bits count."""
    monkeypatch.setattr(launch_record, "CHILD", launch_record.CHILD.replace("out = []\n", CHILD + "out = []\n", 1))
    runtime = launch_record.build(tmp_path)
    calls = [("attn", dict(decode=True)), ("attn", dict(decode=True, b_bucket=20000)), ("attn", dict(decode=True, len_bucket=100)), ("attn", dict(decode=False)),
             ("attn", dict(decode=False, t_bucket=100000)), ("attn", dict(decode=True, t_bucket=8)), ("attn", dict(decode=False, t_bucket=1 << 23, heads=128, kv_heads=8)),
             ("attn", dict(decode=True, b_bucket=65535, heads=224, kv_heads=224)), ("attn", dict(decode=True, b_bucket=1, len_bucket=131072)),
             ("attn", dict(decode=True, t_bucket=5, b_bucket=8, head_dim=256, len_bucket=16384))]
    out = launch_record.record(runtime, calls)
    names = [[n.split("<")[0] for n, _, _ in ls] for _, _, ls in out]
    assert all(rc == 0 for rc, _, _ in out), [msg for rc, msg, _ in out if rc]
    d, p, j, few = "attn_decode_kernel", "attn_prefill_kernel", "attn_join_kernel", "attn_join_few_kernel"
    assert names == [[d, j], [d], [d], [p, few], [p], [d, j], [p], [d], [d, j], [d, few]]
    for _, _, ls in out:
        for _, grid, block in ls:
            assert grid[0] * grid[1] * grid[2] * block[0] < 1 << 32 and grid[1] < 1 << 16 and grid[2] < 1 << 16
