"""The paged entry points' refusals, on the CPU: the C ABI's with addresses that
are never followed, the package's with CPU tensors let past the device check.
Nothing here launches a kernel."""

from __future__ import annotations

import re
import struct
from pathlib import Path

import pytest
import torch

from ssalaad_amd import _lib, logprobs, paged

ROOT = Path(__file__).resolve().parents[1]
FAKE = 256
POOLS = [FAKE, FAKE, 0, 4096, 2048, 64, 1, 9, 2, 16, 64]  # k … head_dim
GRID = [FAKE, 5, 3, 5]  # table, stride, seqs, cols


def _fields(name):
    text = re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "ssalaad_amd.h").read_text(), flags=re.S)
    body = re.search(r"typedef struct \{([^}]*)\} " + name + ";", text).group(1)
    names = []
    for decl in filter(str.strip, body.split(";")):
        for part in decl.split(","):
            names.append(re.sub(r"[^a-z0-9_ ]", " ", part).split()[-1])
    return names


@pytest.mark.parametrize("name,st", [("ssl_paged_append_args", paged._APPEND),
                                     ("ssl_paged_attention_args", paged._ATTENTION),
                                     ("ssl_pages_args", paged._PAGES),
                                     ("ssl_token_logprobs_args", logprobs._ARGS)])
def test_packed_arguments_have_the_headers_fields(name, st):
    fields = _fields(name)
    if fields[0] == "cache":
        fields[:1] = _fields("ssl_paged_cache")
    assert fields[0] == "bytes" and st.size == 8 * len(fields)
    codes = re.sub(r"(\d+)([qd])", lambda m: m[2] * int(m[1]), st.format.lstrip("="))
    assert [f for f, c in zip(fields, codes) if c == "d"] == [
        f for f in fields if f in ("eps", "scale")]


def _try(fn, st, base, **change):
    fields = list(base)
    for k, v in change.items():
        fields[int(k[1:])] = v
    return getattr(_lib.load(), fn)(st.pack(*fields), None)


def test_cache_descriptions_are_checked_before_any_launch():
    st = paged._ATTENTION
    base = [st.size, *POOLS, *GRID, _lib.SSL_BF16, FAKE, 128, 64, FAKE, FAKE, FAKE, 7, 4, 0, 0, 0.1,
            7, 80, FAKE, 1 << 30]
    call = lambda **kw: _try("ssl_paged_attention", st, base, **kw)  # noqa: E731
    assert call(_23=0) == 0  # no tokens: nothing to do
    assert call(_0=8) == 1 and b"struct" in _lib.load().ssl_last_error()
    assert call(_1=0) == 1 and call(_2=FAKE + 8) == 1  # no pool, a misaligned one
    assert call(_4=4095) == 1 and call(_6=32) == 1  # an odd stride, overlapping positions
    assert call(_8=0) == 1 and call(_9=0) == 1  # no pages, no heads
    assert call(_10=8) == 2 and call(_10=48) == 2 and call(_10=2048) == 2
    assert call(_11=96) == 2 and b"head_dim" in _lib.load().ssl_last_error()
    assert call(_12=0) == 1 and call(_13=4) == 1 and call(_14=-1) == 1 and call(_15=-1) == 1
    assert call(_13=1 << 40, _15=1 << 30) == 1  # positions past 31 bits
    assert call(_16=7) == 2
    assert call(_17=0) == 1 and call(_17=FAKE + 2) == 1 and call(_18=127) == 1
    assert call(_20=0) == 1 and call(_21=0) == 1
    assert call(_23=-1) == 1 and call(_24=3) == 1 and call(_24=0) == 1
    assert call(_25=-1) == 1 and call(_26=-1) == 1
    assert call(_22=0) == 1  # 7 tokens, one a sequence, for 3 sequences
    assert _lib.load().ssl_paged_attention(None, None) == 1


@pytest.mark.parametrize("dt,tokens", [(_lib.SSL_BF16, 2048), (_lib.SSL_BF16, 4096), (_lib.SSL_F16, 4096)])
def test_whole_prompts_that_fill_the_device_are_not_split(dt, tokens):
    """16 heads of 64, a workgroup and more a compute unit: no parts, no workspace."""
    st = paged._ATTENTION
    pools = [FAKE, FAKE, 0, 16 * 16 * 64, 16 * 64, 64, 1, 300, 16, 16, 64]
    args = st.pack(st.size, *pools, FAKE, 300, 1, 300, dt, FAKE, 1024, 64, FAKE, FAKE, FAKE, tokens, 16,
                   0, 0, 0.125, tokens, tokens, 0, 0)
    assert _lib.load().ssl_paged_attention_workspace_size(args) == 0


def test_append_arguments_are_checked_before_any_launch():
    st = paged._APPEND
    base = [st.size, *POOLS, *GRID, _lib.SSL_BF16, FAKE, 256, 64, FAKE, 128, 64, FAKE, 128, 64,
            FAKE, FAKE, 32, 32, 100, 0, 0, 1e-6, FAKE, FAKE, FAKE, 2, 4]
    call = lambda **kw: _try("ssl_paged_append", st, base, **kw)  # noqa: E731
    assert call(_37=0) == 0
    assert call(_0=0) == 1 and call(_37=-1) == 1 and call(_38=0) == 1
    for i in (17, 20, 23, 26, 27, 34, 35, 36):
        assert call(**{f"_{i}": 0}) == 1, i
    for i in (17, 20, 23, 26, 27, 36):
        assert call(**{f"_{i}": FAKE + 4}) == 1, i
    for i in (18, 19, 21, 22, 24, 25):
        assert call(**{f"_{i}": 65}) == 1, i
    assert call(_28=33) == 1 and call(_30=0) == 1 and call(_31=FAKE + 4) == 1


def test_page_arguments_are_checked_before_any_launch():
    st, lib = paged._PAGES, _lib.load()
    base = [st.size, *POOLS, *GRID, _lib.SSL_BF16, FAKE, FAKE, FAKE, FAKE, 2, FAKE, FAKE, FAKE, FAKE,
            FAKE, FAKE, 1 << 20]
    for fn, needed in (("ssl_pages_free", (17, 18, 20, 22, 23, 24)),
                       ("ssl_pages_fork", (1, 17, 18, 19, 20, 22, 23, 24, 25)),
                       ("ssl_pages_compact", (1, 18, 22, 24, 26))):
        assert _try(fn, st, base, _0=1) == 1 and _try(fn, st, base, _21=-1) == 1
        assert _try(fn, st, base, _8=0) == 1 and getattr(lib, fn)(None, None) == 1
        for i in needed:
            assert _try(fn, st, base, **{f"_{i}": 0}) == 1, (fn, i)
    need = lib.ssl_pages_fork_workspace_size(2)
    assert need > 0 and lib.ssl_pages_fork_workspace_size(0) == 0
    assert _try("ssl_pages_fork", st, base, _28=need - 1) == 3 and _try("ssl_pages_fork", st, base, _27=0) == 3
    need = lib.ssl_pages_compact_workspace_size(9)
    assert need > 0 and _try("ssl_pages_compact", st, base, _28=need - 1) == 3
    assert _try("ssl_pages_compact", st, base, _27=0) == 3


def test_logprob_arguments_are_checked_before_any_launch():
    st = logprobs._ARGS
    base = [st.size, FAKE, 100, 3, 100, FAKE, 5, FAKE, FAKE, FAKE, FAKE, _lib.SSL_F32]
    call = lambda **kw: _try("ssl_token_logprobs", st, base, **kw)  # noqa: E731
    assert call(_3=0) == 0
    assert call(_0=4) == 1 and call(_2=99) == 1 and call(_3=-1) == 1 and call(_4=0) == 1
    assert call(_6=-1) == 1 and call(_6=101) == 1 and call(_6=65) == 1 and call(_11=5) == 2
    for i in (1, 5, 7, 8, 9, 10):
        assert call(**{f"_{i}": 0}) == 1, i
    assert _lib.load().ssl_token_logprobs(None, None) == 1


# ------------------------------------------------------- the package's own --
class _Launched(Exception):
    pass


@pytest.fixture
def on_cpu(monkeypatch):
    """CPU tensors pass the device check; a call that would launch raises."""
    def call(name, args, device):
        raise _Launched(name)

    monkeypatch.setattr(paged, "_on_gpu", lambda t, name: t.device)
    monkeypatch.setattr(paged, "_call", call)


def _t(*shape, dtype=torch.bfloat16):
    return torch.zeros(*shape, dtype=dtype)


def _i(*shape):
    return torch.zeros(*shape, dtype=torch.int32)


def _refused(fn, good, **bad):
    with pytest.raises(_Launched):
        fn(**good)
    for name, (value, error) in bad.items():
        name = name.split("__")[0]
        with pytest.raises(error):
            fn(**{**good, name: value})


def test_attention_refusals(on_cpu):
    good = dict(q=_t(3, 4, 64), k_pool=_t(9, 2, 16, 64), v_pool=_t(9, 2, 16, 64), table=_i(3, 5),
                lengths=_i(3))
    bad = dict(
        q=(_t(3, 4, 128), ValueError), q__2=(_t(3, 3, 64), ValueError),
        q__3=(_t(3, 4, 64, dtype=torch.float16), TypeError), q__4=(_t(3, 256), ValueError),
        q__6=(_t(3, 0, 64), ValueError),
        k_pool=(_t(9, 2, 16, 128), ValueError), k_pool__2=(_t(2, 16, 64), ValueError),
        k_pool__3=(_t(9, 2, 16, 64, dtype=torch.int8), TypeError),
        k_pool__4=(_t(1, 9, 2, 16, 64), ValueError),
        v_pool=(_t(9, 2, 16, 64, dtype=torch.float16), TypeError),
        v_pool__2=(_t(9, 16, 2, 64).transpose(1, 2), ValueError),
        table=(_i(3, 5).long(), TypeError), table__2=(_i(15), ValueError),
        lengths=(_i(2), ValueError), lengths__2=(_i(3).long(), TypeError),
        window=(-1, ValueError), sinks=(-1, ValueError), max_length=(-1, ValueError))
    _refused(paged.paged_decode_attention, good, q__5=(_t(2, 4, 64), ValueError), **bad)
    good = dict(good, q=_t(7, 4, 64), cu=_i(4))
    _refused(paged.paged_prompt_attention, good, cu=(_i(3), ValueError), cu__2=(None, TypeError),
             cu__3=(_i(4).long(), TypeError), max_tokens=(-1, ValueError), **bad)


def test_attention_of_no_tokens_launches_nothing(on_cpu):
    out = paged.paged_prompt_attention(_t(0, 4, 64), _t(9, 2, 16, 64), _t(9, 2, 16, 64), _i(3, 5),
                                       _i(3), _i(4))
    assert out.shape == (0, 4, 64)


def test_append_refusals(on_cpu):
    f32 = torch.float32
    good = dict(q=_t(7, 4, 64), k=_t(7, 2, 64), v=_t(7, 2, 64), cos=_t(50, 32, dtype=f32),
                sin=_t(50, 32, dtype=f32), k_pool=_t(9, 2, 16, 64), v_pool=_t(9, 2, 16, 64),
                table=_i(3, 5), seqs=_i(7), positions=_i(7), q_norm=_t(64))
    _refused(paged.paged_append, good, k=(_t(7, 3, 64), ValueError), v=(_t(6, 2, 64), ValueError),
             q=(_t(7, 4, 64, dtype=f32), TypeError), q__2=(_t(7, 256), ValueError),
             cos=(_t(50, 64, dtype=f32), ValueError), cos__2=(_t(50, 32), TypeError),
             sin=(_t(49, 32, dtype=f32), ValueError), seqs=(_i(6), ValueError),
             positions=(_i(7).long(), TypeError), q_norm=(_t(32), ValueError),
             k_norm=(_t(64, dtype=f32), TypeError))


def test_page_refusals(on_cpu):
    state = dict(table=_i(3, 5), lengths=_i(3), refs=_i(9))
    pools = dict(k_pool=_t(4, 9, 2, 16, 64), v_pool=_t(4, 9, 2, 16, 64))
    bad = dict(table=(_i(3, 5).long(), TypeError), refs=(_i(0), ValueError),
               refs__2=(_i(9).long(), TypeError))
    _refused(paged.free_pages, dict(state, seqs=_i(2)), lengths=(_i(4), ValueError),
             seqs=(_i(2, 1), ValueError), seqs__2=(_i(2).long(), TypeError), **bad)
    _refused(paged.fork_pages, dict(state, **pools, src=_i(2), dst=_i(2)), refs__3=(_i(8), ValueError),
             dst=(_i(3), ValueError), src=(_i(2, 1), ValueError), lengths=(_i(4), ValueError),
             k_pool=(_t(9, 2, 16, 64), ValueError), **bad)
    _refused(paged.compact_pages, dict(table=_i(3, 5), refs=_i(9), **pools),
             refs__3=(_i(8), ValueError), v_pool=(_t(4, 9, 2, 16, 128), ValueError), **bad)


def test_there_is_no_cpu_path():
    with pytest.raises(ValueError, match="ROCm GPU"):
        paged.paged_decode_attention(_t(3, 4, 64), _t(9, 2, 16, 64), _t(9, 2, 16, 64), _i(3, 5), _i(3))
    with pytest.raises(ValueError, match="ROCm GPU"):
        paged.free_pages(_i(3, 5), _i(3), _i(9), _i(1))
    with pytest.raises(ValueError, match="ROCm GPU"):
        logprobs.token_logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64))


def test_struct_sizes_are_whole_words():
    for st in (paged._APPEND, paged._ATTENTION, paged._PAGES, logprobs._ARGS):
        assert isinstance(st, struct.Struct) and st.size % 8 == 0


# ------------------------------------------------------ the compiled path --
def test_the_compiled_path_leaves_cpu_tensors_to_python():
    """None for every function: nothing is launched, the Python checks decide."""
    tc = _lib.tensorcall()
    pool = _t(9, 2, 16, 64)
    assert tc.append(*[_t(1, 2, 64)] * 3, _t(9, 32), _t(9, 32), pool, pool, _i(1, 4), _i(1), _i(1),
                     None, None, 1e-6) is None
    assert tc.attention(_t(3, 2, 64), pool, pool, _i(3, 5), _i(3), None, 0, 0, None, 1, None) is None
    assert tc.free(_i(3, 5), _i(3), _i(9), _i(1)) is None
    assert tc.fork(_i(3, 5), _i(3), _i(9), pool, pool, _i(1), _i(1)) is None
    assert tc.compact(_i(3, 5), _i(9), pool, pool) is None
    assert tc.logprobs(torch.zeros(2, 9), torch.zeros(2, dtype=torch.int64), 1) is None
    for fn in (tc.append, tc.attention, tc.free, tc.fork, tc.compact, tc.logprobs):
        assert fn() is None and fn(None) is None and fn(*[object()] * 7) is None
    with pytest.raises(TypeError):
        tc.bind(None)
    with pytest.raises(ValueError):
        tc.bind(None, *[0] * 9)


def test_a_status_becomes_the_exception_of_the_c_abi():
    with pytest.raises(ValueError):
        _lib.completed(_lib.SSL_ERR_INVALID, "call")
    with pytest.raises(TypeError):
        _lib.completed(_lib.SSL_ERR_UNSUPPORTED, "call")
    with pytest.raises(RuntimeError):
        _lib.completed(_lib.SSL_ERR_HIP, "call")
    t = torch.zeros(1)
    assert _lib.completed(t, "call") is t


def test_the_paged_engine_needs_a_gpu_and_a_known_model():
    from transformers import LlamaConfig, LlamaForCausalLM

    from ssalaad_amd import PagedEngine

    kw = dict(vocab_size=32, hidden_size=128, intermediate_size=64, num_hidden_layers=1,
              num_attention_heads=2, num_key_value_heads=1, max_position_embeddings=32)
    with pytest.raises(ValueError, match="ROCm GPU"):
        PagedEngine(LlamaForCausalLM(LlamaConfig(**kw)), max_seqs=1, pages=4)
    with pytest.raises(ValueError, match="activation"):
        PagedEngine(LlamaForCausalLM(LlamaConfig(**kw, hidden_act="gelu")), max_seqs=1, pages=4)
    with pytest.raises(ValueError, match="positive"):
        PagedEngine(LlamaForCausalLM(LlamaConfig(**kw)), max_seqs=0, pages=4)
