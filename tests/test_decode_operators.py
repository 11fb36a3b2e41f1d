"""The decode-step operators without a GPU: argument checks of the C ABI and the host's gate layout."""

from __future__ import annotations

import ctypes
import re
from pathlib import Path

import pytest
import torch

import metile_amd as mt
from metile_amd import _lib, norms
from tests import paged_reference as ref

BUF = ctypes.c_void_p(256)  # never dereferenced (nor any 256 below): every case fails its checks


def test_argument_blocks_are_laid_out_as_the_header_says():
    """The struct formats against the header's declarations, field by field."""
    header = (Path(__file__).resolve().parents[1] / "include" / "metile_amd.h").read_text()
    for name, packer in (("mt_paged_tables_args", _lib.PAGED_TABLES_ARGS),
                         ("mt_paged_append_args", _lib.PAGED_APPEND_ARGS),
                         ("mt_paged_attention_args", _lib.PAGED_ATTENTION_ARGS),
                         ("mt_residual_norm_args", _lib.RESIDUAL_NORM_ARGS)):
        body = re.search(r"typedef struct %s \{(.*?)\}" % name, header, re.S).group(1)
        letters = ""
        for line in body.strip().split(";")[:-1]:
            kind, names = re.match(r"\s*(?:const )?(\w+)(.*)", line, re.S).groups()
            for field in names.split(","):
                count = int(re.search(r"\[(\d)\]", field).group(1)) if "[" in field else 1
                letters += ("P" if "*" in field else
                            {"int64_t": "q", "int": "i", "float": "f"}[kind]) * count
        assert packer.format == "@" + letters + "0P", name


def cache(**changes):
    fields = dict(key=256, value=256, key_strides=(ctypes.c_int64 * 3)(2048, 128, 128),
                  value_strides=(ctypes.c_int64 * 3)(2048, 128, 128), pages=4, page_size=16, heads=1,
                  dim=128, dtype=_lib.MT_BF16, key_scale=1.0, value_scale=1.0)
    for name, value in changes.items():
        fields[name] = (ctypes.c_int64 * 3)(*value) if name.endswith("strides") else value
    return ctypes.byref(_lib.PagedCacheDesc(**fields))


BAD_CACHES = [(dict(dtype=2), "dtype"), (dict(pages=0), "pages"), (dict(page_size=0), "pages"),
              (dict(pages=1 << 20, page_size=1 << 11), "2^31"), (dict(heads=0), "heads"),
              (dict(dim=24), "multiple of 16"), (dict(dim=272), "multiple of 16"),
              (dict(key_strides=(2048, 12, 128)), "16 bytes"),
              (dict(value_strides=(2048, -128, 128)), "16 bytes"),
              (dict(dtype=_lib.MT_FP8, value_strides=(2048, 128, 8)), "16 bytes"),
              (dict(value_strides=(1 << 31, 128, 128)), "4 GiB"), (dict(key=None), "null"), (dict(value=264), "aligned"),
              (dict(key_scale=2.0), "scales of 1"),
              (dict(dtype=_lib.MT_FP8, key_scale=0.0), "positive"),
              (dict(dtype=_lib.MT_FP8, value_scale=float("inf")), "normal"),
              (dict(dtype=_lib.MT_FP8, value_scale=float("nan")), "positive")]


def message(status):
    assert status == _lib.MT_ERR_INVALID_ARGUMENT
    return _lib.lib().mt_last_error().decode()


def attend(desc, ws=None, nbytes=0, **changes):
    a = dict(query=256, qs=128, qh=128, tables=256, ts=4, lengths=256, out=256, lse=0, requests=1,
             heads=1, width=4, window=0, scale=1.0, dtype=0)
    a.update(changes)
    return _lib.lib().mt_paged_attention(desc, _lib.PAGED_ATTENTION_ARGS.pack(*a.values()), ws,
                                         nbytes, None)


def append(desc, *args):
    return _lib.lib().mt_paged_append(desc, _lib.PAGED_APPEND_ARGS.pack(*args), None)


@pytest.mark.parametrize("changes,text", BAD_CACHES)
def test_caches_are_checked(changes, text):
    assert text in message(attend(cache(**changes)))
    assert text in message(append(cache(**changes), 256, 256, 128, 128, 128, 128, 256, 1, 0))
    assert _lib.lib().mt_paged_attention_workspace_bytes(cache(**changes), 1, 1, 4, 0) == 0


@pytest.mark.parametrize("changes,text", [
    (dict(requests=0), "requests"), (dict(heads=0), "heads"), (dict(width=0), "width"),
    (dict(width=1 << 27), "2^31"), (dict(width=(1 << 27) - 3), "2^31"), (dict(window=-1), "window"), (dict(dtype=2), "dtype"),
    (dict(dtype=1), "query's dtype"), (dict(scale=float("nan")), "finite"), (dict(scale=3e38), "finite"),
    (dict(query=0), "null"), (dict(out=264), "16 bytes"),
    (dict(qh=100), "16 bytes"), (dict(qs=-128), "16 bytes"),
    (dict(requests=1 << 30, width=1 << 20), "units of work"),
    (dict(requests=1 << 20, width=1 << 20), "units of work")])
def test_attention_arguments_are_checked(changes, text):
    assert text in message(attend(cache(), **changes))


def test_attention_needs_its_workspace():
    lib = _lib.lib()
    need = lib.mt_paged_attention_workspace_bytes(cache(), 3, 8, 4, 0)
    assert need > 64 * 1024
    # what a call needs goes by shapes alone, and is bounded whatever they are
    most = lib.mt_paged_attention_workspace_bytes(cache(), 4000, 16, 4000, 0)
    assert need <= most == lib.mt_paged_attention_workspace_bytes(cache(), 8000, 16, 4000, 0)
    assert attend(cache(), requests=3, heads=8) == _lib.MT_ERR_WORKSPACE
    assert attend(cache(), requests=3, heads=8, ws=BUF, nbytes=need - 1) == _lib.MT_ERR_WORKSPACE


def test_append_and_tables_arguments_are_checked():
    lib = _lib.lib()
    for args, text in (((256, 256, 100, 128, 128, 128, 256, 1, 0), "16 bytes"),
                       ((256, 264, 128, 128, 128, 128, 256, 1, 0), "16 bytes"),
                       ((0, 256, 128, 128, 128, 128, 256, 1, 0), "null"),
                       ((256, 256, 128, 128, 128, 128, 256, -1, 0), "tokens"),
                       ((256, 256, 128, 128, 128, 128, 256, 1 << 30, 0), "below 2^31"),
                       ((256, 256, 128, 128, 128, 128, 256, 1, 1), "rows' dtype"),
                       ((256, 256, 128, 128, 128, 128, 256, 1, 2), "dtype")):
        assert text in message(append(cache(), *args))
    assert append(cache(), 0, 0, 0, 0, 0, 0, 0, 0, 0) == _lib.MT_OK
    good = dict(cached=256, new=256, table=256, stride=4, free=256, start=0, slots=256,
                positions=256, owners=256, starts=256, lengths=256, taken=256, requests=2, width=4,
                count=1, page=16, tokens=1)
    for changes, text in ((dict(requests=-1), "negative"), (dict(tokens=-1), "negative"),
                          (dict(count=-1), "negative"), (dict(page=0), "page_size"),
                          (dict(width=0), "width"), (dict(width=1 << 27), "2^31"),
                          (dict(stride=3), "overlap"), (dict(cached=0), "null"),
                          (dict(free=0), "null"), (dict(slots=0), "null"),
                          (dict(starts=0), "null"), (dict(taken=0), "null")):
        args = _lib.PAGED_TABLES_ARGS.pack(*{**good, **changes}.values())
        assert text in message(lib.mt_paged_tables(args, None))


def test_norm_arguments_are_checked():
    good = dict(residual=256, block=256, weight=256, bias=0, pw=0, pb=0, gate=0, out=256, normed=256,
                rs=64, bs=64, gs=0, rows=1, width=64, gr=1, scalar=0, scale=1.0, eps=1e-6, kind=0,
                dtype=0, rdtype=0)

    def fn(**changes):
        return _lib.lib().mt_residual_norm(
            _lib.RESIDUAL_NORM_ARGS.pack(*{**good, **changes}.values()), None)

    for changes, text in ((dict(dtype=2), "dtype"), (dict(rdtype=1), "residual_dtype"),
                          (dict(kind=2), "kind"), (dict(width=0), "width"),
                          (dict(width=65537), "width"), (dict(rows=-1), "rows"),
                          (dict(eps=-1.0), "eps"), (dict(eps=float("nan")), "eps"),
                          (dict(scale=float("inf")), "residual_scale"),
                          (dict(gate=256, gr=0), "gate_rows"), (dict(gate=256, gs=-1), "gate_"),
                          (dict(weight=0), "null"), (dict(residual=0), "null"),
                          (dict(normed=0), "null")):
        assert text in message(fn(**changes))
    assert fn(rows=0) == _lib.MT_OK


@pytest.mark.parametrize("shape", [(6, 4), (2, 3, 4), (2, 3, 5, 4), (1, 3, 4), (2, 1, 4), (5, 1),
                                   (4,), (2, 3, 1)])
def test_gates_of_every_broadcast(shape):
    width, rows = shape[-1], torch.Size(shape).numel() // shape[-1]
    sizes = [()]
    for n in range(1, len(shape) + 1):
        sizes += [tuple(v if bit >> i & 1 else 1 for i, v in enumerate(shape[-n:]))
                  for bit in range(1 << n)]
    for size in set(sizes):
        gate = torch.randn(size)
        flat, stride, per, scalar = norms._gate(gate, torch.Size(shape), width, rows)
        assert scalar or width == 1 or flat.stride(-1) == 1
        got = torch.stack([
            torch.as_strided(flat, (1 if scalar else width,), (1,), flat.storage_offset()
                             + (r // per) * stride).expand(width) for r in range(rows)])
        assert torch.equal(got, gate.expand(shape).reshape(rows, width)), size
    with pytest.raises(ValueError, match="broadcast"):
        norms._gate(torch.randn(*shape[:-1], width + 2), torch.Size(shape), width, rows)


def test_guards_before_the_device():
    x = torch.zeros(2, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        mt.residual_norm(x, weight=x[0])
    t = torch.zeros(4, 16, 1, 64, dtype=torch.bfloat16)
    with pytest.raises(ValueError, match="ROCm device"):
        mt.PagedCache(t, t)
    i = torch.zeros(2, dtype=torch.int32)
    with pytest.raises(ValueError, match="ROCm device"):
        mt.paged_tables(i, i, i[:, None], i, page_size=16, tokens=2)


def test_reference_tables_by_hand():
    table, slots, positions, owners, starts, lengths, taken = ref.tables(
        [3, 4, 0], [3, 1, 0], [[7, -1], [5, -1], [-1, -1]], [9, 8], 4, 6)
    assert table == [[7, 9], [5, 8], [-1, -1]]
    assert slots == [31, 36, 37, 32, -1, -1]
    assert positions == [3, 4, 5, 4, 0, 0] and owners == [0, 0, 0, 1, -1, -1]
    assert starts == [0, 3, 4, 4] and lengths == [6, 5, 0] and taken == [2]


def test_reference_fp8_against_torch():
    x = torch.cat([torch.linspace(-500, 500, 4001), torch.randn(4000) * 2.0 ** -7])
    want = x.clamp(-448, 448).to(torch.float8_e4m3fn).double()
    assert ref.fp8_values(x.clamp(-448, 448).double().numpy()).tolist() == want.tolist()


def test_reference_attention_against_torch():
    g = torch.Generator().manual_seed(0)
    key, value = torch.randn(2, 5, 4, 2, 8, generator=g, dtype=torch.float64)
    query = torch.randn(1, 4, 8, generator=g).half()
    tables = torch.tensor([[3, 1, 4]])
    out, lse, _, _ = ref.attention(query, key, value, tables, [10], 0.3, window=7)
    k = key[[3, 1, 4]].reshape(12, 2, 8)[3:10].repeat_interleave(2, 1)
    v = value[[3, 1, 4]].reshape(12, 2, 8)[3:10].repeat_interleave(2, 1)
    want = torch.nn.functional.scaled_dot_product_attention(
        query.double().transpose(0, 1), k.transpose(0, 1), v.transpose(0, 1), scale=0.3)
    assert torch.allclose(out, want.transpose(0, 1), atol=1e-12)
