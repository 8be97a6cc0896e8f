"""CPU tests of the 4-bit cache's definition and of the refusals that need no GPU."""
import ctypes
import math
import random
import shutil
import struct
import subprocess
from pathlib import Path

import pytest
import torch

from lmpool_b200 import _build, _capi
from lmpool_b200 import attention as at
from oracle import attention_ref as ref


def test_row_bytes():
    assert at.q4_row_bytes(128) == 72 and at.q4_row_bytes(64) == 36
    with pytest.raises(ValueError):
        at.q4_row_bytes(24)


def test_e4m3_table_is_torchs():
    want = torch.arange(127, dtype=torch.uint8).view(torch.float8_e4m3fn).double().tolist()
    assert ref.E4M3 == want


def test_definition_keeps_values_on_the_grid():
    """What the format can hold is kept as it is; everything else moves by at most half a step of the group."""
    row = torch.tensor(ref.LEVELS + [-v for v in ref.LEVELS]) * 0.375
    codes, scales = ref.q4_encode_row(row)
    assert ref.q4_decode(codes, scales) == row.tolist()
    x = torch.randn(4096, generator=torch.Generator().manual_seed(1))
    back = torch.tensor(ref.q4_decode(*ref.q4_encode_row(x)), dtype=torch.float64)
    top = x.double().view(-1, 16).abs().amax(1, keepdim=True)
    # widest step 2 of 6 levels: half of it is top / 6, and the scale is off by at most 2^-4 (e4m3)
    assert ((back - x.double()).view(-1, 16).abs() <= top / 6 * (1 + 2.0 ** -4) + 1e-9).all()


def test_definition_of_odd_groups():
    assert ref.q4_encode_row(torch.zeros(16)) == ([0] * 16, [0])
    assert ref.q4_encode_row(torch.full((16,), math.inf)) == ([0] * 16, [0x7F])
    assert ref.q4_encode_row(torch.full((16,), 1e9))[1] == [126]
    codes, scales = ref.q4_encode_row(torch.full((16,), 2.0 ** -10))
    assert scales == [0] and codes == [0] * 16


def _args(**kw):
    base = dict(ptr=[1 << 20] * 6, cu=0, strides=[1024, 256, 1024, 256, 4096, 256, 128, 8], num_blocks=4, T=2, S=2, heads=4,
                kv=2, dim=64, bs=16, width=8, dtype=0, bits=16, window=0, sinks=0, scale=0.1, ks=1.0, vs=1.0, r=0)
    base.update(kw)
    b = base
    return _capi.pack_attention(*b["ptr"], b["cu"], *b["strides"], b["num_blocks"], b["T"], b["S"], b["heads"], b["kv"],
                                b["dim"], b["bs"], b["width"], b["dtype"], b["bits"], b["window"], b["sinks"], b["scale"],
                                b["ks"], b["vs"], b["r"], 0)


BAD = [dict(r=1), dict(dtype=2), dict(bits=8), dict(dim=96), dict(T=-1), dict(S=-1), dict(heads=5), dict(kv=0),
       dict(heads=1024, kv=2), dict(bs=0), dict(bs=8, bits=4), dict(width=-1), dict(width=1 << 28), dict(num_blocks=0),
       dict(window=-1), dict(sinks=-1), dict(scale=0.0), dict(scale=math.nan), dict(scale=math.inf), dict(scale=-1.0),
       dict(bits=4, ks=3.0), dict(bits=4, vs=0.0), dict(ks=2.0), dict(T=3), dict(bits=4, ks=-2.0),
       dict(bits=4, scale=1e30, ks=2.0 ** 60), dict(bits=4, scale=1e-30, ks=2.0 ** -60)]
BAD_POINTERS = [dict(ptr=[0] + [1 << 20] * 5), dict(ptr=[1 << 20] * 5 + [0]), dict(ptr=[8] + [1 << 20] * 5),
                dict(strides=[1000, 256, 1024, 256, 4096, 256, 128, 8]), dict(strides=[1024, 256, 1024, 256, 4096, 250, 128, 8])]


@pytest.mark.parametrize("bad", BAD + BAD_POINTERS, ids=str)
def test_attention_refuses_before_touching_a_gpu(kvx_lib, bad):
    status = ctypes.c_int32(0)
    rc = kvx_lib.kvx_paged_attention(0, _args(**bad), None, 0, ctypes.addressof(status), None)
    assert rc == _capi.KVX_EINVAL and kvx_lib.kvx_last_error()


@pytest.mark.parametrize("dim,bs", [(128, 1 << 25), (64, 1 << 26), (128, (1 << 23) + 16)])
def test_4bit_pages_beyond_32_bit_offsets_are_refused(kvx_lib, dim, bs):
    """Offsets within a (page, head) are 32-bit numbers: the store refuses such pages, and so does what reads them."""
    status = ctypes.c_int32(0)
    strides = [dim * 8, dim * 2, dim * 8, dim * 2, bs * dim // 16 * 9 * 2, 0, 0, 8]
    args = _args(dim=dim, bs=bs, bits=4, width=1, strides=strides)
    need = ctypes.c_uint64(0)
    for rc in (kvx_lib.kvx_attention_workspace(0, args, ctypes.byref(need)),
               kvx_lib.kvx_paged_attention(0, args, None, 0, ctypes.addressof(status), None)):
        assert rc == _capi.KVX_EINVAL and b"too large" in kvx_lib.kvx_last_error()


def test_more_tokens_and_sequences_than_items_are_counted_for_are_refused(kvx_lib):
    need = ctypes.c_uint64(0)
    for sizes in (dict(T=2 ** 31 - 1, S=1), dict(T=2 ** 30, S=2 ** 30), dict(T=2, S=2 ** 31 - 1)):
        rc = kvx_lib.kvx_attention_workspace(0, _args(cu=1 << 20, **sizes), ctypes.byref(need))
        assert rc == _capi.KVX_EINVAL and b"beyond" in kvx_lib.kvx_last_error()


def test_the_packed_struct_is_the_headers(kvx_lib, tmp_path):
    """pack_attention writes kvx_attention field by field: same size, same places."""
    src = tmp_path / "layout.c"
    src.write_text("""
#include <stdio.h>
#include "kvx.h"
int main(void) {
    printf("%zu %zu %zu %zu %zu %zu\\n", sizeof(kvx_attention), offsetof(kvx_attention, cu_seqlens_q),
           offsetof(kvx_attention, num_blocks), offsetof(kvx_attention, num_tokens), offsetof(kvx_attention, sinks),
           offsetof(kvx_attention, v_scale));
    return 0;
}
""")
    if shutil.which("gcc") is None:
        pytest.skip("gcc not installed")
    root = Path(__file__).resolve().parent.parent
    subprocess.run(["gcc", "-std=c11", "-Wall", "-Werror", "-I", str(root / "include"), str(src), "-o", str(tmp_path / "l")],
                   check=True, capture_output=True)
    got = [int(x) for x in subprocess.run([str(tmp_path / "l")], capture_output=True, text=True, check=True).stdout.split()]
    at_of = lambda n: struct.calcsize("=" + n)  # noqa: E731
    assert got == [struct.calcsize("=7Q9q11i3f2i"), at_of("6Q"), at_of("7Q8q"), at_of("7Q9q"), at_of("7Q9q10i"),
                   at_of("7Q9q11i2f")]
    assert len(_args()) == got[0]


def test_attention_needs_a_status_word(kvx_lib):
    assert kvx_lib.kvx_paged_attention(0, _args(), None, 0, None, None) == _capi.KVX_EINVAL
    assert kvx_lib.kvx_paged_attention(0, None, None, 0, None, None) == _capi.KVX_EINVAL


def test_attention_with_no_tokens_is_no_work(kvx_lib):
    status = ctypes.c_int32(0)
    assert kvx_lib.kvx_paged_attention(0, _args(T=0, S=0), None, 0, ctypes.addressof(status), None) == _capi.KVX_OK


@pytest.mark.parametrize("bad", [dict(dtype=2), dict(T=-1), dict(N=0), dict(bs=8), dict(dim=24), dict(dim=272), dict(heads=0),
                                 dict(ks=1.5), dict(vs=math.inf), dict(stride=1000), dict(ptr=8), dict(ptr=0)], ids=str)
@pytest.mark.parametrize("name", ["kvx_store_kvcache_q4", "kvx_load_kvcache_q4"])
def test_q4_rows_refuse_before_touching_a_gpu(kvx_lib, name, bad):
    a = dict(dtype=0, T=2, N=4, bs=16, dim=64, heads=2, ks=1.0, vs=1.0, stride=256, ptr=1 << 20)
    a.update(bad)
    status = ctypes.c_int32(0)
    rc = getattr(kvx_lib, name)(0, a["dtype"], a["ptr"], 1 << 20, a["stride"], 256, 1 << 20, 1 << 20, 4608, 1 << 20, a["T"],
                                a["N"], a["bs"], a["heads"], a["dim"], a["ks"], a["vs"], ctypes.addressof(status), None)
    assert rc == _capi.KVX_EINVAL and kvx_lib.kvx_last_error()


def test_cpu_tensors_are_refused():
    x = torch.zeros(2, 1, 64, dtype=torch.float16)
    kc = torch.zeros(1, 16, 1, 36, dtype=torch.uint8)
    with pytest.raises(RuntimeError, match="CUDA"):
        at.store_kvcache_q4(x, x, kc, kc, torch.zeros(2, dtype=torch.int64), 16)
    with pytest.raises(RuntimeError, match="CUDA"):
        at.load_kvcache_q4(kc, kc, torch.zeros(2, dtype=torch.int64), 16)
    kv = torch.zeros(1, 16, 1, 64, dtype=torch.float16)
    with pytest.raises(RuntimeError, match="CUDA"):
        at.paged_attention(x, kv, kv, torch.zeros(2, 1, dtype=torch.int32), torch.zeros(2, dtype=torch.int32), 16)


@pytest.mark.parametrize("shape,strides,offset,copied", [
    ((1, 4, 64), (257, 64, 1), 0, False), ((1, 4, 64), (3, 64, 1), 0, False), ((3, 1, 64), (64, 5, 1), 0, False),
    ((1, 1, 64), (7, 9, 1), 0, False), ((1, 4, 64), (257, 64, 1), 1, True), ((1, 4, 64), (257, 72, 1), 0, True),
    ((3, 4, 64), (257, 64, 1), 0, True), ((3, 4, 64), (264, 64, 1), 0, False), ((1, 4, 64), (1, 1, 4), 0, True)])
def test_rows_to_store_have_strides_that_the_library_takes(shape, strides, offset, copied):
    x = torch.arange(2048).to(torch.bfloat16).as_strided(shape, strides, offset)
    rows = at._rows_of(x)
    assert torch.equal(rows, x) and (rows.data_ptr() != x.data_ptr()) == copied
    assert rows.data_ptr() % 16 == 0 and at._token_stride(rows) % 16 == 0
    assert rows.stride(2) == 1 and (shape[1] == 1 or rows.stride(1) == shape[2])
    assert shape[0] == 1 or at._token_stride(rows) == 2 * rows.stride(0)


def test_rows_that_share_elements_are_found():
    """Against all pairs, over layouts of every kind: nested, crossed, repeated."""
    rng = random.Random(1)
    seen = [0, 0]
    for _ in range(4000):
        size, tokens, heads = rng.choice((4, 8)), rng.randint(0, 5), rng.randint(0, 5)
        step, head = (rng.choice((0, size // 2, size, rng.randint(0, 6) * size, rng.randint(0, 50))) for _ in range(2))
        starts = sorted(t * step + h * head for t in range(tokens) for h in range(heads))
        want = any(b - a < size for a, b in zip(starts, starts[1:]))
        assert at._rows_overlap(tokens, step, heads, head, size) == want, (tokens, step, heads, head, size)
        seen[want] += 1
    assert min(seen) > 500


def _ptxas(*kernels):
    return "\n".join(f"ptxas info    : Compiling entry function '{name}' for 'sm_100a'\nptxas info    : Function properties for "
                     f"{name}\n    0 bytes stack frame\nptxas info    : Used {n} registers, used 1 barriers" for name, n in kernels)


def test_a_build_with_other_register_counts_is_refused():
    """The tile kernel's warps pass registers on: what the compiler gave is checked when it is built, not at a user's call."""
    good = [("_ZN3kvx16attn_tile_kernelIa", 96), ("_ZN3kvx17attn_split_kernelIa", 120), ("_ZN3kvx16attn_tile_kernelIb", 96)]
    _build.check_registers(_ptxas(*good))
    for bad in (good[1:2], [], good[:2] + [("_ZN3kvx16attn_tile_kernelIb", 88)], [("_ZN3kvx16attn_tile_kernelIb", 104)] + good):
        with pytest.raises(RuntimeError, match="96 registers"):
            _build.check_registers(_ptxas(*bad))
