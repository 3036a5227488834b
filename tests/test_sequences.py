"""What happens to sequences between two steps: beam selection, reordering of slots, key weights, eviction.

Every operator against a plain implementation in 64 bits; whole numbers and moved bytes have to be equal.
"""

import ctypes
import math
import re
import subprocess
import sys
from pathlib import Path
from types import SimpleNamespace

import pytest
import torch

from megakernels_b200.native import mk_sequences as ops

ROOT = Path(__file__).resolve().parent.parent
HALF = 2.0**-24  # an fp32 rounding, relative


# ---- interface (no GPU) ------------------------------------------------------------------------ #
def header():
    return re.sub(r"/\*.*?\*/", "", (ROOT / "include" / "mkb200_sequences.h").read_text(), flags=re.S)


def test_library_exports_every_declared_function():
    lib = ops.load_library()
    names = sorted(set(re.findall(r"\b(mkb_[a-z_0-9]+)\s*\(", header())))
    assert len(names) == 10
    for name in names:
        assert hasattr(lib, name), name


def test_makefile_lists_the_files_of_the_build():
    from megakernels_b200.build import CSRC, LIBRARIES

    lists = {k.strip(): set(v.split()) for k, v in (line.split(":=", 1) for line in (CSRC / "Makefile").read_text().splitlines() if ":=" in line)}
    assert lists["SEQUENCES_SRC"] == set(LIBRARIES["sequences"].sources) and lists["SEQUENCES_HDR"] == set(LIBRARIES["sequences"].headers)


def test_struct_fields_match_the_header():
    text = header()
    for struct in ops.STRUCTS:
        body = re.search(r"typedef struct %s \{(.*?)\} %s;" % (struct.__name__, struct.__name__), text, flags=re.S).group(1)
        names = []
        for line in body.split(";"):
            line = line.strip()
            if line:
                line = re.sub(r"^(const\s+)?\w+\s+", "", line)
                names += [re.sub(r"[\s*]|\[\w+\]", "", n) for n in line.split(",")]
        assert names == [f[0] for f in struct._fields_], struct.__name__
    for name in ("MAX_BEAMS", "MAX_BEST", "MAX_REGIONS", "MAX_SLOTS"):
        assert int(re.search(rf"#define MKBS_{name} (\d+)", text).group(1)) == getattr(ops, name)


FAKE = 0x10000


def fill(struct, **kw):
    s = ops._struct(struct)
    for name, kind in struct._fields_:
        if kind is ctypes.c_void_p and name not in ("done", "kept", "status", "lengths"):
            setattr(s, name, FAKE)
    for name, v in kw.items():
        setattr(s, name, v)
    return s


def beams_struct(**kw):
    return fill(ops.MkbsBeams, **{**dict(groups=2, beams=4, vocab=1000, k=8, row_stride=1000, eos=3, workspace_bytes=1 << 30), **kw})


def weights_struct(**kw):
    base = dict(layers=2, sequences=2, queries=3, heads=8, kv_heads=2, dim=64, positions=100, length=50, scale=0.1, q_layer=6144, q_sequence=1536,
                k_layer=25600, k_sequence=12800, w_layer=400, w_sequence=200, w_head=100, workspace_bytes=1 << 30)
    return fill(ops.MkbsKeyWeights, **{**base, **kw})


def select_struct(**kw):
    base = dict(layers=2, sequences=2, kv_heads=2, positions=100, length=50, keep=10, sinks=2, recent=3, w_layer=400, w_sequence=200, w_head=100)
    return fill(ops.MkbsSelect, **{**base, **kw})


def move_struct(**kw):
    s = fill(ops.MkbsMove, layers=2, sequences=2, kv_heads=2, positions=100, length=50, keep=10, head_bytes=128, c_layer=51200, c_sequence=25600)
    s.caches[0], s.caches[1] = FAKE, 2 * FAKE
    for name, v in kw.items():
        if name in ("cache", "second"):
            s.caches[name == "second"] = v
        else:
            setattr(s, name, v)
    return s


def reorder_struct(region=None, **kw):
    r = ops.MkbsRegion(FAKE, 2, 10, 8000, 1000, 100)
    for name, v in (region or {}).items():
        setattr(r, name, v)
    s = fill(ops.MkbsReorder, slots=8, num_regions=1)
    s.regions = ctypes.pointer(r)
    s._region = r  # (kept alive)
    for name, v in kw.items():
        setattr(s, name, v)
    return s


REFUSED = [
    ("beam_select", beams_struct, [
        (dict(struct_bytes=8), 1, "struct size"), (dict(dtype=2), 1, "dtype"), (dict(groups=0), 1, "positive"), (dict(vocab=0), 1, "positive"), (dict(k=0), 1, "positive"),
        (dict(beams=65), 5, "at most"), (dict(k=129), 5, "at most"), (dict(groups=20000), 5, "at most"), (dict(vocab=1 << 28, row_stride=1 << 28), 5, "vocab"),
        (dict(beams=2, vocab=3, k=7), 1, "continuations"), (dict(row_stride=999), 1, "row_stride"), (dict(logits=None), 1, "logits"), (dict(logits=FAKE + 1), 1, "logits"),
        (dict(dtype=1, logits=FAKE + 2), 1, "logits"), (dict(scores=FAKE + 2), 1, "unaligned"), (dict(out_tokens=None), 1, "outputs"),
        (dict(eos=1000), 1, "eos"), (dict(eos=-2), 1, "eos"), (dict(eos=-1, done=FAKE), 1, "eos"), (dict(workspace=None), 1, "workspace"), (dict(workspace=FAKE + 8), 1, "workspace"),
        (dict(workspace_bytes=16), 1, "workspace"),
    ]),
    ("reorder_slots", reorder_struct, [
        (dict(struct_bytes=8), 1, "struct size"), (dict(slots=0), 1, "positive"), (dict(num_regions=0), 1, "positive"), (dict(first=-1), 1, "negative"),
        (dict(slots=257), 5, "at most"), (dict(num_regions=49), 5, "at most"), (dict(parents=None), 1, "parents"), (dict(lengths=FAKE + 1), 1, "lengths"), (dict(status=FAKE + 2), 1, "status"),
        (dict(region=dict(base=None)), 1, "empty"), (dict(region=dict(rows=0)), 1, "empty"), (dict(region=dict(row_bytes=0)), 1, "empty"),
        (dict(region=dict(slot_stride=999)), 1, "overlap"), (dict(region=dict(outer_stride=999)), 1, "overlap"), (dict(region=dict(row_bytes=1 << 31)), 1, "overlap"),
    ]),
    ("key_weights", weights_struct, [
        (dict(struct_bytes=8), 1, "struct size"), (dict(layers=0), 1, "positive"), (dict(positions=0), 1, "positive"), (dict(queries=0), 1, "queries"), (dict(heads=7), 1, "multiple"),
        (dict(heads=0), 1, "multiple"), (dict(dim=96), 5, "dim"), (dict(heads=258), 5, "128 heads"), (dict(q_layer=1528), 1, "overlap"), (dict(k_layer=12792), 1, "overlap"), (dict(length=101), 1, "length"), (dict(length=-1), 1, "length"), (dict(lengths=FAKE + 2), 1, "length"),
        (dict(layers=60000), 5, "65535"), (dict(positions=1 << 29), 5, "positions"), (dict(queries=1 << 20), 5, "2^20"), (dict(layers=1, kv_heads=8, sequences=1024, positions=1 << 25), 5, "tiles"), (dict(q=FAKE + 8), 1, "unaligned"), (dict(k=None), 1, "missing"),
        (dict(weights=FAKE + 2), 1, "unaligned"), (dict(q_layer=4), 1, "multiples of 8"), (dict(k_sequence=12804), 1, "multiples of 8"), (dict(k_sequence=12792), 1, "overlap"),
        (dict(q_sequence=1528), 1, "overlap"), (dict(w_head=99), 1, "overlap"), (dict(w_sequence=99), 1, "overlap"), (dict(w_layer=99), 1, "overlap"), (dict(scale=math.nan), 1, "finite"),
        (dict(scale=math.inf), 1, "finite"), (dict(workspace=FAKE + 16), 1, "workspace"), (dict(workspace_bytes=16), 1, "workspace"), (dict(status=FAKE + 1), 1, "unaligned"),
    ]),
    ("select_rows", select_struct, [
        (dict(struct_bytes=8), 1, "struct size"), (dict(sequences=0), 1, "positive"), (dict(kv_heads=40000), 5, "65535"), (dict(length=101), 1, "length"), (dict(keep=0), 1, "keep"),
        (dict(sinks=-1), 1, "keep"), (dict(recent=-1), 1, "keep"), (dict(sinks=8, recent=3), 1, "keep"), (dict(weights=None), 1, "weights"), (dict(rows=FAKE + 2), 1, "rows"),
        (dict(kept=FAKE + 2), 1, "unaligned"), (dict(kept=FAKE, w_head=99), 1, "overlap"), (dict(kept=FAKE, w_sequence=99), 1, "overlap"), (dict(kept=FAKE, w_layer=0), 1, "overlap"),
    ]),
    ("move_rows", move_struct, [
        (dict(struct_bytes=8), 1, "struct size"), (dict(layers=0), 1, "positive"), (dict(length=-1), 1, "length"), (dict(keep=0), 1, "keep"), (dict(head_bytes=8), 5, "16 bytes"),
        (dict(head_bytes=1040), 5, "1024"), (dict(rows=None), 1, "rows"), (dict(cache=None), 1, "caches"), (dict(cache=FAKE + 8), 1, "caches"), (dict(c_sequence=25592), 1, "unaligned"),
        (dict(c_sequence=25584), 1, "overlap"), (dict(c_layer=25584), 1, "overlap"), (dict(second=FAKE), 1, "the same"),
    ]),
]


@pytest.mark.parametrize("name,make,kw,code,said", [(n, m, *case) for n, m, cases in REFUSED for case in cases], ids=lambda v: str(v)[:40] if isinstance(v, (str, dict)) else "")
def test_library_refuses(name, make, kw, code, said):
    """Each wrong argument by itself, in a call that is right without it; nothing is launched (there may be no device)."""
    lib = ops.load_library()
    s = make(**kw)
    assert getattr(lib, f"mkb_{name}")(ctypes.byref(s), None) == code
    assert said in lib.mkb_sequences_last_error().decode()


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls are right: with a device they would run")
@pytest.mark.parametrize("name,make", [(n, m) for n, m, _ in REFUSED])
def test_only_the_device_is_missing_in_the_calls_that_the_refusals_start_from(name, make):
    lib = ops.load_library()
    assert getattr(lib, f"mkb_{name}")(ctypes.byref(make()), None) == 2
    assert getattr(lib, f"mkb_{name}")(None, None) == 1


OVERLAPPING = [  # strides of more than one block's size, that several blocks share all the same
    ("key_weights", weights_struct, [dict(w_sequence=100), dict(w_sequence=150), dict(w_layer=100), dict(w_layer=200), dict(w_layer=399), dict(w_head=200), dict(w_head=250, w_layer=1000)]),
    ("select_rows", select_struct, [dict(kept=FAKE, w_sequence=100), dict(kept=FAKE, w_layer=300), dict(kept=FAKE, w_layer=200), dict(kept=FAKE, kv_heads=3, w_head=200, w_sequence=350, w_layer=2000)]),
    ("move_rows", move_struct, [dict(c_layer=25600), dict(c_layer=25616), dict(c_layer=38400), dict(c_sequence=51200), dict(sequences=3, c_layer=38400, c_sequence=51200)]),
    ("reorder_slots", reorder_struct, [dict(region=dict(outer_stride=1000)), dict(region=dict(outer_stride=7000)), dict(region=dict(outer_stride=1500)), dict(region=dict(slot_stride=8000))]),
]


@pytest.mark.parametrize("name,make,kw", [(n, m, kw) for n, m, cases in OVERLAPPING for kw in cases], ids=lambda v: str(v)[:60] if isinstance(v, (str, dict)) else "")
def test_strides_that_meet_are_refused(name, make, kw):
    lib, s = ops.load_library(), make(**kw)
    assert getattr(lib, f"mkb_{name}")(ctypes.byref(s), None) == 1
    assert "overlap" in lib.mkb_sequences_last_error().decode()


APART = [
    ("key_weights", weights_struct, [dict(w_layer=100, w_sequence=200, w_head=400), dict(w_layer=200, w_sequence=400, w_head=100), dict(w_layer=1, layers=1), dict(w_head=0, kv_heads=1)]),
    ("select_rows", select_struct, [dict(w_head=0, w_layer=0), dict(kept=FAKE, w_layer=100, w_sequence=200, w_head=400), dict(kept=FAKE, kv_heads=3, w_head=200, w_sequence=300, w_layer=800)]),
    ("move_rows", move_struct, [dict(c_layer=25600, c_sequence=51200), dict(sequences=3, c_layer=38400, c_sequence=76800), dict(sequences=1, c_sequence=0)]),
    ("reorder_slots", reorder_struct, [dict(region=dict(outer_stride=1000, slot_stride=2000)), dict(region=dict(outer_stride=1500, slot_stride=3000)), dict(region=dict(outer=1, outer_stride=0))]),
]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls are right: with a device they would run")
@pytest.mark.parametrize("name,make,kw", [(n, m, kw) for n, m, cases in APART for kw in cases], ids=lambda v: str(v)[:60] if isinstance(v, (str, dict)) else "")
def test_any_order_of_dimensions_is_taken_that_keeps_blocks_apart(name, make, kw):
    """(Also interleaved ones, where no dimension steps over all of another.)"""
    assert getattr(ops.load_library(), f"mkb_{name}")(ctypes.byref(make(**kw)), None) == 2


ONE = [("key_weights", weights_struct, dict(layers=1, q_layer=1, k_layer=7, w_layer=0)), ("key_weights", weights_struct, dict(sequences=1, q_sequence=3, k_sequence=1, w_sequence=0)),
       ("move_rows", move_struct, dict(layers=1, c_layer=2)), ("move_rows", move_struct, dict(sequences=1, c_sequence=2))]


@pytest.mark.skipif(torch.cuda.is_available(), reason="the calls are right: with a device they would run")
@pytest.mark.parametrize("name,make,kw", ONE, ids=lambda v: str(v)[:60] if isinstance(v, (str, dict)) else "")
def test_a_dimension_of_one_has_any_stride(name, make, kw):
    assert getattr(ops.load_library(), f"mkb_{name}")(ctypes.byref(make(**kw)), None) == 2


def test_the_same_region_twice_is_refused():
    """Two regions, then the same one twice."""
    lib, s = ops.load_library(), reorder_struct()
    regions = (ops.MkbsRegion * 2)(s._region, ops.MkbsRegion(2 * FAKE, 2, 10, 8000, 1000, 100))
    s.regions, s.num_regions = ctypes.cast(regions, ctypes.POINTER(ops.MkbsRegion)), 2
    if not torch.cuda.is_available():  # (with a device it would run)
        assert lib.mkb_reorder_slots(ctypes.byref(s), None) == 2
    regions[1].base = FAKE
    assert lib.mkb_reorder_slots(ctypes.byref(s), None) == 1
    assert "0 and 1 are the same" in lib.mkb_sequences_last_error().decode()


def test_a_wait_that_gave_up_is_raised_and_cleared():
    """(The record as a kernel leaves it; no call here waits in vain.)"""
    status = torch.zeros(16, dtype=torch.int32)
    ops.raise_status(status)
    status[0], status[1] = 3, 77
    with pytest.raises(ops.SequenceError, match="block 77") as e:
        ops.raise_status(status)
    assert e.value.code == 3 and not status.any()
    ops.raise_status(status)


def test_a_record_of_inference_mode_is_raised_and_cleared():
    with torch.inference_mode():
        status = torch.zeros(16, dtype=torch.int32)
        status[:2] = torch.tensor([3, 9], dtype=torch.int32)
    with pytest.raises(ops.SequenceError, match="block 9"):
        ops.raise_status(status)
    assert not status.any()


@pytest.mark.parametrize("length", [-1, 101, 2**32 + 5, -(2**32) + 5])
def test_a_length_outside_the_cache_is_refused(length):
    s = ops._struct(ops.MkbsSelect)
    with pytest.raises(ValueError, match="outside"):
        ops._set_lengths(s, length, 0, 1, 100)
    ops._set_lengths(s, 100, 0, 1, 100)
    assert s.length == 100


FAR = 2**32 + 5  # five, when it is cut to 32 bits


@pytest.mark.parametrize("call", [
    lambda z: ops.beam_select(z(2, 100), beams=2, k=FAR), lambda z: ops.beam_select(z(2, FAR), beams=2, k=3), lambda z: ops.beam_select(z(2, 100), beams=2, k=3, eos=FAR),
    lambda z: ops.beam_select(z(2, 100), beams=2, k=5 - 2**32), lambda z: ops.reorder_slots([z(4, 9)], z(4).int(), first=FAR, lengths=z(4).int()),
    lambda z: ops.key_weights(z(1, 1, 1, 8, 64), z(1, 1, FAR, 2, 64), z(1, 1, 2, FAR), 5, scale=1.0), lambda z: ops.key_weights(z(1, 1, FAR, 8, 64), z(1, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0),
    lambda z: ops.key_weights(z(1, 1, 1, 8, 64), z(1, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0, wait_timeout_ms=FAR),
    lambda z: ops.key_weights(z(1, 1, 1, 8, 64), z(1, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0, wait_timeout_ms=-1 - 2**31),
    lambda z: ops.select_rows(z(1, 1, 2, 100), 50, keep=FAR), lambda z: ops.select_rows(z(1, 1, 2, 100), 50, keep=9, sinks=FAR), lambda z: ops.select_rows(z(1, 1, 2, 100), 50, keep=9, recent=5 - 2**32),
    lambda z: ops.select_rows(z(FAR, 1, 2, 100), 50, keep=9), lambda z: ops.move_rows(z(1, FAR, 9, 2, 64), None, z(1, 1, 2, 9), 50), lambda z: ops.key_weights(z(FAR, 1, 1, 8, 64), z(FAR, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0),
    lambda z: ops.select_rows(z(1, 1, 2, FAR), 50, keep=9), lambda z: ops.move_rows(z(1, 1, FAR, 2, 64), None, z(1, 1, 2, 9), 50), lambda z: ops.move_rows(z(1, 1, 9, 2, 64), None, z(1, 1, 2, FAR), 5),
])
def test_numbers_that_do_not_fit_are_refused(call):
    with pytest.raises(ValueError, match="32 bits"):
        call(lambda *shape: torch.zeros(()).expand(shape))


def test_a_negative_limit_is_refused():
    z = lambda *shape: torch.zeros(()).expand(shape)  # noqa: E731
    with pytest.raises(ValueError, match="limit"):
        ops.key_weights(z(1, 1, 1, 8, 64), z(1, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0, wait_timeout_ms=-1)


def test_the_longest_limit_is_taken():
    """(What is refused then is where the tensors are.)"""
    z = lambda *shape: torch.zeros(()).expand(shape)  # noqa: E731
    with pytest.raises(ValueError, match="CUDA device"):
        ops.key_weights(z(1, 1, 1, 8, 64), z(1, 1, 9, 2, 64), z(1, 1, 2, 9), 5, scale=1.0, wait_timeout_ms=2**32 - 1)


@pytest.mark.gpu
def test_rows_of_a_region_that_do_not_fit_are_refused():
    """(8 GB of bytes, that nothing touches.)"""
    t = torch.empty(2, FAR, dtype=torch.uint8, device="cuda")
    with pytest.raises(ValueError, match="32 bits"):
        ops.reorder_slots([t], torch.tensor([1, 0], dtype=torch.int32).cuda(), lengths=torch.tensor([5, 5], dtype=torch.int32).cuda())


def test_a_stream_of_another_device_is_refused(monkeypatch):
    """(Of a device that need not be there.)"""
    monkeypatch.setattr(torch.cuda, "current_device", lambda: 0)
    with pytest.raises(ValueError, match="stream is cuda:1's"):
        ops._Where(SimpleNamespace(device_index=1, cuda_stream=5), torch.zeros(1))
    assert ops._Where(SimpleNamespace(device_index=0, cuda_stream=5), torch.zeros(1)).handle == 5


def test_torch_without_its_quick_entry_points():
    """All three are replaced, each by itself, and what is there is taken."""
    names = ("_cuda_getCurrentRawStream", "_cuda_cudaCachingAllocator_raw_alloc", "_cuda_cudaCachingAllocator_raw_delete")
    assert all(callable(f) for f in ops._entry_points(SimpleNamespace()))
    for i, name in enumerate(names):
        points = ops._entry_points(SimpleNamespace(**{name: "quick"}))
        assert points[i] == "quick" and all(callable(f) for j, f in enumerate(points) if j != i)


@pytest.mark.gpu
def test_calls_by_torch_s_public_entry_points(monkeypatch):
    for name, f in zip(("_raw_stream", "_raw_alloc", "_raw_free"), ops._entry_points(SimpleNamespace())):
        monkeypatch.setattr(ops, name, f)
    side, held = torch.cuda.Stream(), []
    for _ in range(2):  # (the first pass may leave what torch itself keeps)
        check_beams(draw(1, 4, 3001), beams=2, k=5)
        check_beams(draw(1, 4, 3001), beams=2, k=5, stream=side)
        with torch.cuda.stream(side):
            check_beams(draw(1, 4, 3001), beams=2, k=5)
        q, k, w, scale = weights_case(3, 1, 1, 30, 8, 2, 64, 200, [200])
        check_weights(q, k, w, [200], scale)
        del q, k, w
        held.append(torch.cuda.memory_allocated())
    assert held[0] == held[1]  # (workspaces go back)


def test_beam_selection_takes_all_it_says_it_takes():
    """Every shape at the limits has a plan that fits shared memory."""
    lib = ops.load_library()
    for k in range(1, 129):
        for beams in (1, 2, 3, 5, 8, 13, 16, 32, 63, 64):
            vocab = (1 << 30) // (beams * k)
            for v in {vocab, vocab // 2, vocab // 3, 128256}:
                if v * beams * k <= 1 << 30:
                    assert lib.mkb_beam_bytes(ctypes.byref(beams_struct(groups=1, beams=beams, vocab=v, k=k))) > 0, (k, beams, v)


def test_workspace_sizes_of_wrong_shapes_are_zero():
    lib = ops.load_library()
    assert lib.mkb_beam_bytes(ctypes.byref(beams_struct())) > 0 and lib.mkb_beam_bytes(ctypes.byref(beams_struct(k=0))) == 0
    assert lib.mkb_key_weights_bytes(ctypes.byref(weights_struct())) > 0 and lib.mkb_key_weights_bytes(ctypes.byref(weights_struct(dim=32))) == 0
    assert lib.mkb_beam_bytes(None) == lib.mkb_key_weights_bytes(None) == 0


def test_the_shim_refuses_what_is_not_on_the_device():
    x = torch.zeros(4, 100)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.beam_select(x, beams=2, k=3)
    with pytest.raises(ValueError, match="groups of 3"):
        ops.beam_select(x, beams=3, k=3)
    with pytest.raises(ValueError, match="bfloat16 or float32"):
        ops.beam_select(x.half(), beams=2, k=3)
    with pytest.raises(ValueError, match="no tensors"):
        ops.reorder_slots([], torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="needs lengths"):
        ops.reorder_slots([x], torch.zeros(4, dtype=torch.int32), first=1)
    with pytest.raises(ValueError, match="CUDA device"):
        ops.reorder_slots([x], torch.zeros(4, dtype=torch.int32))
    with pytest.raises(ValueError, match="CUDA device"):
        ops.select_rows(torch.zeros(1, 1, 2, 9), 5, keep=3)
    with pytest.raises(ValueError, match="kv_heads"):
        ops.move_rows(x, x, torch.zeros(1, 1, 1, 1, dtype=torch.int32), 1)
    with pytest.raises(ValueError, match="must be"):
        ops.key_weights(x, x, x, 1, scale=1.0)


# ---- beam selection ------------------------------------------------------------------------------ #
def beam_reference(logits, scores, beams, k, done, eos):
    rows, vocab = logits.shape
    x = logits.double()
    x[x.isnan()] = -math.inf
    top = x.max(dim=1, keepdim=True).values
    from_top = torch.where(x == top, torch.zeros_like(x), x - top)  # (infinite logits share everything)
    log_p = from_top - from_top.exp().sum(dim=1, keepdim=True).log()
    c = (scores.double() if scores is not None else x.new_zeros(rows // beams, beams)).reshape(-1, 1)
    total = torch.where(x == -math.inf, torch.full_like(x, -math.inf), c + log_p)
    if done is not None:
        over = done.reshape(-1) != 0
        total[over] = -math.inf
        total[over, eos] = c[over, 0]
    total[~c.isfinite().reshape(-1)] = -math.inf
    flat = total.view(rows // beams, beams * vocab)
    best, at = torch.sort(flat, dim=1, descending=True, stable=True)
    best, at = best[:, :k], at[:, :k]
    parents = at // vocab + torch.arange(rows // beams, device=x.device).unsqueeze(1) * beams
    tokens = at % vocab
    ended = tokens == (-1 if eos is None else eos)
    if done is not None:
        ended |= done.reshape(-1)[parents] != 0
    return best.cpu(), parents.cpu(), tokens.cpu(), ended.cpu()


def check_beams(logits, scores=None, *, beams, k, done=None, eos=None, stream=None):
    got = ops.beam_select(logits, scores, beams=beams, k=k, done=done, eos=eos, stream=stream)
    torch.cuda.synchronize()
    best, parents, tokens, ended = beam_reference(logits, scores, beams, k, done, eos)
    assert torch.equal(got[1].cpu().long(), parents) and torch.equal(got[2].cpu().long(), tokens)
    assert torch.equal(got[3].cpu() != 0, ended)
    have = got[0].cpu().double()
    fine = best.isfinite()
    assert torch.equal(have[~fine], best[~fine].float().double())
    # The sum of exponentials: an element's own error is a few roundings (its exponent is one product of size 40 at most, that
    # of a summand of size 2^-58), a lane adds up to vocab / 32 of them in turn, one after the other eight, and 5 lanes' sums
    bound = (logits.shape[1] / 32 + 48) * HALF + best[fine].abs() * HALF
    assert ((have[fine] - best[fine]).abs() <= bound).all()
    return got


def draw(seed, *shape, dtype=torch.float32, std=1.0):
    return (torch.randn(*shape, generator=torch.Generator().manual_seed(seed)) * std).to(dtype).cuda()


BF16, F32 = torch.bfloat16, torch.float32


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("groups,beams,vocab,k", [
    (1, 1, 1, 1), (2, 1, 7, 7), (3, 2, 5, 10), (1, 4, 255, 4), (2, 3, 256, 6), (1, 5, 257, 128), (5, 2, 4099, 16), (1, 64, 1000, 128), (1, 64, 128256, 64),
    (1, 4, 128256, 4), (8, 8, 128256, 16), (64, 1, 32003, 3), (1, 16, 32003, 33), (2, 1, 262144, 128), (1, 64, 131072, 128), (1, 64, 262144, 32), (1, 2, 500_000, 1),
])
def test_beam_select(groups, beams, vocab, k, dtype):
    rows = groups * beams
    logits = draw(vocab + k, rows, vocab, dtype=dtype, std=2.5)
    scores = draw(k, groups, beams) * 2 - 10
    check_beams(logits, scores, beams=beams, k=k)
    done = (torch.rand(groups, beams, generator=torch.Generator().manual_seed(3)) < 0.4).to(torch.uint8).cuda()
    check_beams(logits, scores, beams=beams, k=k, done=done, eos=vocab // 3)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_beam_select_of_rows_any_distance_apart(dtype):
    wide = draw(1, 6, 1003, dtype=dtype, std=3)
    for first in range(9):  # rows start at every alignment
        check_beams(wide[:, first : first + 777], draw(2, 2, 3), beams=3, k=9)
    check_beams(wide[::2], beams=3, k=5)
    assert wide[::2].stride(0) == 2006


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_beam_select_breaks_ties_by_place(dtype):
    logits = draw(5, 1, 2048, dtype=dtype, std=1).round().expand(8, -1).contiguous()  # equal rows: equal scores in all of them
    check_beams(logits, beams=4, k=128)
    check_beams(logits, torch.zeros(1, 8).cuda(), beams=8, k=100)
    check_beams(torch.zeros(4, 100_000, dtype=dtype).cuda(), beams=2, k=77)
    check_beams(torch.arange(5000.0).div(100).floor().expand(2, -1).to(dtype).cuda(), beams=2, k=128)  # all of a segment's elements are among the best
    check_beams(-torch.arange(5000.0).div(100).floor().expand(2, -1).to(dtype).cuda(), beams=1, k=128)
    check_beams(torch.tensor([[0.0, -0.0, 0.0, -0.0]]).to(dtype).cuda(), beams=1, k=4)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_beam_select_of_masked_logits(dtype):
    inf = math.inf
    logits = draw(7, 8, 3001, dtype=dtype, std=2)
    logits[0, 5:] = -inf  # five continuations
    logits[1] = -inf  # none
    logits[2, ::2] = torch.finfo(dtype).min
    logits[3, 1::3] = math.nan
    logits[4, 17] = inf
    logits[5, [3, 900, 2999]] = inf
    logits[6] = math.nan
    logits[7, 1:] = torch.finfo(dtype).min
    for beams, k in ((8, 128), (1, 7), (2, 128), (4, 16)):
        check_beams(logits, beams=beams, k=k)
        check_beams(logits, draw(8, 8 // beams, beams), beams=beams, k=k)
    scores = torch.tensor([[0.0, -inf, -inf, -inf], [-inf, math.nan, inf, -inf]]).cuda()  # a first step; no beam at all
    check_beams(logits, scores, beams=4, k=128)
    done = torch.tensor([[1, 0, 1, 0], [1, 1, 1, 1]], dtype=torch.uint8).cuda()
    check_beams(logits, scores, beams=4, k=9, done=done, eos=3000)
    check_beams(logits, draw(9, 2, 4), beams=4, k=9, done=done, eos=0)
    check_beams(logits, draw(9, 8, 1), beams=1, k=128, done=done.view(8, 1), eos=60)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("k", [1, 5, 16, 64])
def test_beam_select_of_logits_in_few_places(dtype, k):
    """A run of large logits holds more of the best than other runs have: many elements beat every other run's largest one."""
    x = draw(5, 4, 20_011, dtype=dtype)
    for row, (first, last) in enumerate([(700, 2300), (0, 300), (19_500, 20_011), (5000, 5003)]):
        x[row, first:last] += 30
    for beams in (1, 2, 4):
        scores = draw(6, 4 // beams, beams)
        done = torch.tensor([0, 0, 0, 1], dtype=torch.uint8).cuda().view(4 // beams, beams)
        check_beams(x, scores, beams=beams, k=k)
        check_beams(x, scores, beams=beams, k=k, done=done, eos=701)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
@pytest.mark.parametrize("beams,vocab,k", [(11, 5814, 11), (8, 1000, 8), (4, 32003, 16), (64, 3001, 64), (8, 128256, 16)])
def test_beam_select_where_one_beam_is_ahead(beams, vocab, k, dtype):
    """All of the best, or most of them, are one beam's continuations."""
    x = draw(vocab, 2 * beams, vocab, dtype=dtype, std=2)
    for gap in (3, 12, 200):
        scores = draw(k, 2, beams) - gap
        scores[0, beams - 1] = scores[1, 0] = 0
        done = torch.zeros(2, beams, dtype=torch.uint8)
        done[0, 0] = done[1, 0] = 1  # (in the second group the one that is ahead has ended)
        check_beams(x, scores, beams=beams, k=k)
        check_beams(x, scores, beams=beams, k=k, done=done.cuda(), eos=vocab - 1)


@pytest.mark.gpu
@pytest.mark.parametrize("dtype", [BF16, F32])
def test_the_first_selection_of_a_process_may_need_any_amount_of_shared_memory(dtype):
    """48 KB less a few bytes, 48 KB exactly and more; each shape in a process of its own, since one selection's permission serves the next."""
    for beams, vocab, k in ((1, 8200, 128), (3, 2600, 128), (2, 6200, 96), (33, 100, 128), (1, 7000, 128), (1, 9000, 128)):
        code = f"""
import sys; sys.path.insert(0, {str(ROOT)!r})
import torch
from tests.test_sequences import check_beams, draw
check_beams(draw(1, {2 * beams}, {vocab}, dtype={dtype}, std=2), beams={beams}, k={k})
"""
        subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


@pytest.mark.gpu
def test_beam_select_far_apart_and_large_logits():
    x = torch.full((2, 5000), -1e4).cuda()
    x[0, 4321], x[1, 7] = 3e38, -3e38
    check_beams(x, beams=2, k=5)
    check_beams(draw(3, 4, 3333) * 1e4, draw(4, 1, 4) * 100, beams=4, k=40)
    for low in (torch.finfo(F32).min, -2e6, -1.2e6, 0.9e6, 1.1e6, 3e37):  # rows whose logits are all of that size
        x = torch.full((3, 3000), low)
        x[0, 5::7] += abs(low) * 2**-20
        x[1, 1000:] = torch.finfo(F32).min
        x[2, 3::2] = -math.inf
        check_beams(x.cuda(), beams=3, k=20)
        x[:, 7] = math.nan
        check_beams(x.cuda(), torch.tensor([[0.0, 1.0, -2.0]]).cuda(), beams=3, k=20)
    near = torch.full((2, 9000), -1e6) + torch.arange(9000) % 100 / 4 - 10  # on both sides of where sums change their reference
    check_beams(near.cuda(), beams=1, k=7)
    check_beams(-near.cuda(), beams=2, k=7)


# ---- reordering ----------------------------------------------------------------------------------- #
def check_reorder(tensors, parents, dim=0, first=0, lengths=None, stream=None):
    want = []
    for t in tensors:
        old = t.cpu().clone()
        new = old.clone()
        for slot, parent in enumerate(parents):
            if not 0 <= parent < len(parents) or parent == slot:
                continue
            if lengths is None:
                rows = slice(None)
                new.select(dim, slot).copy_(old.select(dim, parent))
            else:
                rows = slice(first, max(first, min(max(lengths[parent], 0), t.shape[dim + 1])))
                new.select(dim, slot).narrow(dim, rows.start, rows.stop - rows.start).copy_(old.select(dim, parent).narrow(dim, rows.start, rows.stop - rows.start))
        want.append(new)
    i32 = lambda v: torch.tensor(v, dtype=torch.int32).cuda()  # noqa: E731
    ops.reorder_slots(tensors, i32(parents), dim=dim, first=first, lengths=None if lengths is None else i32(lengths), stream=stream)
    torch.cuda.synchronize()
    for t, w in zip(tensors, want):
        assert torch.equal(t.cpu().view(torch.uint8), w.view(torch.uint8))


@pytest.mark.gpu
@pytest.mark.parametrize("parents", [[0], [0, 0], [1, 0], [1, 2, 3, 0], [3, 3, 3, 3], [0, 1, 2, 3], [4, -1, 0, 7, 2], [6, 5, 4, 3, 2, 1, 0]])
@pytest.mark.parametrize("shape,dtype", [((3, 40, 2, 64), BF16), ((2, 17, 3), F32), ((2, 5, 7), torch.uint8), ((1, 3000, 1, 8), BF16)])
def test_reorder_of_cache_rows(parents, shape, dtype):
    slots = len(parents)
    make = lambda seed: draw(seed, shape[0], slots, *shape[1:], std=50).to(dtype)  # noqa: E731
    rows = shape[1]
    check_reorder([make(1), make(2)], parents, dim=1, lengths=[rows] * slots)
    check_reorder([make(1), make(2)], parents, dim=1, first=3, lengths=[(7 * s) % (rows + 2) for s in range(slots)])  # some of them behind the first row's
    check_reorder([make(3)], parents, dim=1, first=rows, lengths=[rows] * slots)
    check_reorder([make(3)], parents, dim=1, first=0, lengths=[-3, rows + 100, 0, 1, rows, 2, 3][:slots])
    check_reorder([make(4)[0]], parents, dim=0, lengths=[rows - 1] * slots)


@pytest.mark.gpu
def test_reorder_of_whole_states():
    gen = torch.Generator().manual_seed(1)
    for slots in (2, 6, 64, 256):
        parents = torch.randint(0, slots, (slots,), generator=gen).tolist()
        check_reorder([draw(slots, slots, 4, 64, 64), draw(slots + 1, slots, 3, 37), draw(slots, slots, 5, dtype=BF16), draw(2, slots)], parents)
    check_reorder([draw(i, 4, 3, 16) for i in range(101)], [2, 0, 0, 1])  # more regions than a call takes
    check_reorder([draw(1, 3, 4, 50, 8)[:, :, 5:20]], [1, 2, 3, 0], dim=1)  # rows of a part, the slots further apart
    check_reorder([draw(1, 9, 4, 5, 8)[::2]], [1, 1, 3, 0], dim=1, lengths=[5, 4, 3, 2])


@pytest.mark.gpu
def test_reorder_of_a_large_cache():
    """Every source more bytes than shared memory holds, offsets beyond 2^31."""
    k = torch.empty(2, 5, 60_000, 2048, dtype=BF16, device="cuda")
    k[:, :, ::1000] = draw(1, 2, 5, 60, 2048).to(BF16)
    k[1, 4, -1] = 7
    rows = k[:, :, ::1000].clone()
    parents = torch.tensor([4, 0, 0, 1, 2], dtype=torch.int32).cuda()
    ops.reorder_slots([k], parents, dim=1, first=0, lengths=torch.full((5,), 60_000, dtype=torch.int32).cuda())
    assert torch.equal(k[:, :, ::1000], rows[:, parents.long()]) and (k[1, 0, -1] == 7).all()


@pytest.mark.gpu
def test_reorder_of_many_tensors():
    """More than a call of the library takes; none of them twice."""
    tensors = [draw(i, 3, 16) for i in range(ops.MAX_REGIONS + 2)]
    old, parents = [t.clone() for t in tensors], torch.tensor([2, 0, 0], dtype=torch.int32).cuda()
    with pytest.raises(ValueError, match="twice"):
        ops.reorder_slots([*tensors, tensors[0]], parents)
    assert all(torch.equal(t, o) for t, o in zip(tensors, old))
    ops.reorder_slots(tensors, parents)
    assert all(torch.equal(t, o[parents.long()]) for t, o in zip(tensors, old))


# ---- key weights ------------------------------------------------------------------------------------ #
def weights_case(seed, layers, sequences, queries, heads, kv_heads, dim, positions, lengths, scale=None):
    q = draw(seed, layers, sequences, queries, heads, dim, dtype=BF16)
    k = draw(seed + 1, layers, sequences, positions, kv_heads, dim, dtype=BF16)
    w = draw(seed + 2, layers, sequences, kv_heads, positions).abs()
    for b, n in enumerate(lengths):  # what nobody may look at
        k[:, b, max(n, 0) :] = math.nan
    return q, k, w, dim**-0.5 if scale is None else scale


def weights_reference(q, k, w, lengths, scale):
    """The weights in 64 bits, and how far 32-bit arithmetic may be from them, relative to what is added."""
    layers, sequences, queries, heads, dim = q.shape
    positions, kv_heads = k.shape[2:4]
    per, out, worst = heads // kv_heads, w.double().clone(), 0.0
    for layer in range(layers):
        for b, n in enumerate(lengths):
            n = min(max(n, 0), positions)
            if n == 0:
                continue
            last = n - queries + torch.arange(queries, device=q.device)
            seen = torch.arange(n, device=q.device)[None] <= last[:, None]
            for h in range(heads):
                x, y = q[layer, b, :, h].double(), k[layer, b, :n, h // per].double()
                z = (x @ y.T * scale).masked_fill(~seen, -math.inf)
                p = torch.softmax(z, dim=-1).masked_fill(~seen.any(dim=1, keepdim=True), 0.0)
                out[layer, b, h // per, :n] += p.sum(dim=0)
                worst = max(worst, float((x.abs() @ y.abs().T).max()) * abs(scale))
    # A score is a sum of `dim` products that the tensor cores cut off at 2^-23 of the largest: both a key's score and its row's sum
    # move a weight by that; the exponent's own rounding is of the score's size; sums over keys (in parts) and rows
    tol = 2 * (dim + 4) * 2 * HALF * worst + (queries * per + 128) * 2 * HALF
    return out, tol


def check_weights(q, k, w, lengths, scale, as_number=False, stream=None):
    want, tol = weights_reference(q, k, w, lengths, scale)
    before = w.clone()
    given = lengths[0] if as_number else torch.tensor(lengths, dtype=torch.int32).cuda()
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    ops.key_weights(q, k, w, given, scale=scale, status=status, stream=stream)
    torch.cuda.synchronize()
    assert int(status.abs().sum()) == 0
    added = want - before.double()
    err = (w.double() - want).abs()
    assert (err <= tol * added + 2 * HALF * want + 1e-37).all(), float((err / (tol * added + 2 * HALF * want + 1e-37)).max())
    for b, n in enumerate(lengths):
        n = min(max(n, 0), k.shape[2])
        assert torch.equal(w[:, b, :, n:], before[:, b, :, n:])
    return tol


@pytest.mark.gpu
@pytest.mark.parametrize("queries,positions,lengths", [
    (1, 1, [1]), (1, 70, [70, 1, 0, 33]), (2, 300, [300, 1]), (3, 129, [129, 2, 128]), (16, 1000, [999, 16, 500]), (17, 200, [5, 200]), (33, 257, [256, 257, -4]), (64, 2000, [2000]),
    (130, 130, [130]), (301, 700, [650]), (1, 5001, [5001]),
])
@pytest.mark.parametrize("heads,kv_heads,dim", [(8, 2, 64), (8, 2, 128), (4, 4, 64), (16, 2, 128)])
def test_key_weights(queries, positions, lengths, heads, kv_heads, dim):
    check_weights(*weights_case(queries, 2, len(lengths), queries, heads, kv_heads, dim, positions, lengths)[:3], lengths, dim**-0.5)


@pytest.mark.gpu
@pytest.mark.parametrize("queries", [1, 40])
def test_key_weights_of_dimensions_of_one_with_odd_strides(queries):
    """Tensors whose layers' and sequences' dimensions of one came from elsewhere: a stride of 1."""
    q, k, w, scale = weights_case(5, 1, 1, queries, 8, 2, 64, 300, [300])
    q, k, w = (t[0, 0].unsqueeze(-1).unsqueeze(-1).permute(-1, -2, *range(t.ndim - 2)) for t in (q, k, w))
    assert q.stride()[:2] == (1, 1) and k.stride()[:2] == (1, 1)
    check_weights(q, k, w, [300], scale)
    old = k.clone()
    rows = ops.select_rows(w, 300, keep=50)
    ops.move_rows(k, None, rows, 300)
    for h in range(2):
        assert torch.equal(k[0, 0, :50, h], old[0, 0, rows[0, 0, h].long(), h])


@pytest.mark.gpu
@pytest.mark.parametrize("per", [3, 5, 7, 12, 24, 100])
def test_key_weights_of_odd_numbers_of_heads(per):
    q, k, w, scale = weights_case(per, 1, 2, 21, 2 * per, 2, 64, 333, [333, 200])
    check_weights(q, k, w, [333, 200], scale)


@pytest.mark.gpu
def test_key_weights_of_sharp_and_flat_rows():
    for scale in (0.0, -0.3, 4.0):  # equal weights; the other way round; one key takes nearly all
        q, k, w, _ = weights_case(11, 1, 1, 40, 8, 2, 64, 600, [600])
        check_weights(q, k, w, [600], scale, as_number=True)
    q, k, w, scale = weights_case(12, 1, 1, 5, 8, 2, 64, 400, [400])
    w.zero_()
    tol = check_weights(q, k, w, [400], scale)
    assert (w.double().sum(dim=-1) - 5 * 4).abs().max() <= 5 * 4 * (tol + 2 * HALF)  # every row's weights add up to one


@pytest.mark.gpu
def test_key_weights_of_parts_of_larger_tensors():
    big_q, big_k = draw(1, 3, 4, 9, 8, 64, dtype=BF16), draw(2, 3, 4, 250, 2, 64, dtype=BF16)
    big_w = torch.zeros(3, 4, 2, 300, device="cuda")
    q, k, w = big_q[::2, 1:3], big_k[::2, 1:3], big_w[::2, 1:3, :, 7:257]
    check_weights(q, k, w, [250, 31], 0.125)
    rest = big_w.clone()
    rest[::2, 1:3, :, 7:257] = 0
    assert not rest.any()


@pytest.mark.gpu
@pytest.mark.parametrize("queries,heads,kv_heads", [(1, 4, 1), (1, 16, 2), (3, 10, 2), (16, 1, 1)])
def test_weights_of_few_rows_of_large_scores(queries, heads, kv_heads):
    """Every score is some 32768 and differs from others by 0 to 6: products are exact whole numbers, and what is rounded is small."""
    n, per = 2000, heads // kv_heads
    q = torch.full((1, 1, queries, heads, 64), 16.0)
    k = torch.full((1, 1, n, kv_heads, 64), 16.0)
    q[..., 63] = 1
    k[..., 63] = torch.randint(0, 4, (1, 1, n, kv_heads), generator=torch.Generator().manual_seed(queries)).float()
    q, k, w = q.to(BF16).cuda(), k.to(BF16).cuda(), torch.zeros(1, 1, kv_heads, n, device="cuda")
    want, _ = weights_reference(q, k, w, [n], 2.0)
    ops.key_weights(q, k, w, n, scale=2.0)
    # The scale is rounded twice and multiplies differences of 6; an exponential is off by 2^-22, a row's sum by that, by what changing its reference
    # takes (the same, up to three times in each of 8 lanes' and warps' joins) and by its additions
    tol = 6 * 2.0**-22 + 2.0**-22 * (2 + 3 * 8) + (n / 32 + 64 + per * queries) * HALF
    assert ((w.double() - want).abs() <= tol * want).all(), float(((w.double() - want).abs() / want).max())


@pytest.mark.gpu
def test_waits_do_not_count_the_time_of_the_launch_before():
    """One sequence's rows pass takes some 3 ms, while the blocks of the keys pass already wait on all other SMs: 1 ms is a limit for each wait of
    a block for its own copies and products."""
    others, long = 74, 600_000
    lengths = [long] + [100] * others
    q = draw(1, 1, 1 + others, 17, 1, 64, dtype=BF16)
    k = torch.empty(1, 1 + others, long, 1, 64, dtype=BF16, device="cuda")
    k[:, 0] = torch.randn(long, 1, 64, generator=torch.Generator("cuda").manual_seed(1), device="cuda").to(BF16)
    k[:, 1:, :100] = draw(2, 1, others, 100, 1, 64, dtype=BF16)
    w = torch.zeros(1, 1 + others, 1, long, device="cuda")
    status = torch.zeros(16, dtype=torch.int32, device="cuda")
    ops.key_weights(q, k, w, torch.tensor(lengths, dtype=torch.int32).cuda(), scale=0.125, status=status, wait_timeout_ms=1)
    torch.cuda.synchronize()
    assert not status.any(), status.tolist()
    want, tol = weights_reference(q[:, 1:], k[:, 1:, :100], torch.zeros(1, others, 1, 100, device="cuda"), [100] * others, 0.125)
    assert ((w[:, 1:, :, :100].double() - want).abs() <= tol * want).all() and not w[:, 1:, :, 100:].any()
    assert abs(float(w[0, 0].double().sum()) - 17) <= 17 * (tol + 2 * HALF)


@pytest.mark.gpu
def test_a_wait_that_gives_up_is_recorded_without_a_status(monkeypatch):
    """Calls that are given no status name the device's own record, which is raised and cleared.  (No call here waits in vain.)"""
    q, k, w = draw(1, 1, 1, 20, 4, 64, dtype=BF16), draw(2, 1, 1, 50, 2, 64, dtype=BF16), torch.zeros(1, 1, 2, 50, device="cuda")
    named, launch = [], ops._Where.launch
    monkeypatch.setattr(ops._Where, "launch", lambda self, name, s, *used: (named.append(s.status), launch(self, name, s, *used)))
    ops.key_weights(q, k, w, 50, scale=0.1)
    ops.reorder_slots([draw(1, 4, 16)], torch.tensor([1, 0, 0, 2], dtype=torch.int32).cuda())
    record = ops._records[torch.cuda.current_device()]
    assert named == [record.data_ptr()] * 2
    ops.raise_status()
    record[:2] = torch.tensor([3, 41])
    with pytest.raises(ops.SequenceError, match="block 41") as e:
        ops.raise_status()
    assert e.value.code == 3
    ops.raise_status()
    given = torch.zeros(16, dtype=torch.int32, device="cuda")
    ops.key_weights(q, k, w, 50, scale=0.1, status=given)
    assert named[2] == given.data_ptr()


@pytest.mark.gpu
def test_a_status_is_read_when_other_streams_have_ended():
    """(A record that a stream writes a tenth of a second late.)"""
    status, gave_up, side = torch.zeros(16, dtype=torch.int32, device="cuda"), torch.full((16,), 3, dtype=torch.int32, device="cuda"), torch.cuda.Stream()
    for cycles in (10, 200_000_000):  # (first the loading of what runs, which waits for the device)
        status.zero_()
        ops.raise_status(status)
        with torch.cuda.stream(side):
            torch.cuda._sleep(cycles)
            status.copy_(gave_up)
        if cycles == 10:
            torch.cuda.synchronize()
        with pytest.raises(ops.SequenceError, match="block 3"):
            ops.raise_status(status)


@pytest.mark.gpu
def test_a_call_without_a_status_may_be_the_first_and_captured():
    code = f"""
import sys; sys.path.insert(0, {str(ROOT)!r})
import torch
from megakernels_b200.native import mk_sequences as ops
a, b = torch.arange(12.0, device="cuda").view(3, 4), torch.tensor([2, 0, 0], dtype=torch.int32, device="cuda")
torch.cuda.synchronize()
graph = torch.cuda.CUDAGraph()
with torch.cuda.graph(graph):
    ops.reorder_slots([a], b)
graph.replay()
ops.raise_status()
assert a[:, 0].tolist() == [8.0, 0.0, 0.0], a
next(iter(ops._records.values()))[0] = 3  # (as a kernel leaves it; a replay does not clear it)
graph.replay()
try:
    ops.raise_status()
except ops.SequenceError as e:
    assert e.code == 3
else:
    raise AssertionError
"""
    subprocess.run([sys.executable, "-c", code], check=True, timeout=300)


@pytest.mark.gpu
def test_key_weights_are_the_same_bits_every_time():
    q, k, w, scale = weights_case(5, 1, 1, 100, 8, 2, 128, 3000, [3000])
    lengths, first = torch.tensor([3000], dtype=torch.int32).cuda(), None
    for _ in range(20):
        out = torch.zeros_like(w)
        ops.key_weights(q, k, out, lengths, scale=scale)
        first = out if first is None else first
        assert torch.equal(out, first)


# ---- eviction ------------------------------------------------------------------------------------- #
def rows_reference(weights, lengths, keep, sinks, recent):
    layers, sequences, heads, positions = weights.shape
    w = weights.cpu().double()
    w[w.isnan()] = -math.inf
    out = torch.full((layers, sequences, heads, keep), -1, dtype=torch.int32)
    for layer in range(layers):
        for b, n in enumerate(lengths):
            n = min(max(n, 0), positions)
            for h in range(heads):
                if n <= keep:
                    out[layer, b, h, :n] = torch.arange(n, dtype=torch.int32)
                    continue
                v = w[layer, b, h].tolist()
                middle = sorted(range(sinks, n - recent), key=lambda j: (-v[j], j))[: keep - sinks - recent]
                out[layer, b, h] = torch.tensor([*range(sinks), *sorted(middle), *range(n - recent, n)], dtype=torch.int32)
    return out


def check_rows(weights, lengths, keep, sinks, recent, kept=None, stream=None):
    want = rows_reference(weights, lengths, keep, sinks, recent)
    old = weights.clone()
    before = None if kept is None else kept.clone()
    rows = ops.select_rows(weights, torch.tensor(lengths, dtype=torch.int32).cuda(), keep=keep, sinks=sinks, recent=recent, kept=kept, stream=stream)
    torch.cuda.synchronize()
    assert torch.equal(rows.cpu(), want)
    if kept is not None:
        for b, n in enumerate(lengths):
            n = min(max(n, 0), keep, weights.shape[3])
            have, source = kept[:, b, :, :n], rows[:, b, :, :n].long()
            assert torch.equal(have.contiguous().view(torch.int32), old[:, b].gather(2, source).view(torch.int32))
            assert torch.equal(kept[:, b, :, n:], before[:, b, :, n:])
    return rows


@pytest.mark.gpu
@pytest.mark.parametrize("positions,lengths,keep,sinks,recent", [
    (1, [1], 1, 0, 0), (1, [1, 0], 1, 0, 1), (10, [10, 3, 0, 9, 30, -1], 3, 1, 1), (100, [100, 99], 40, 0, 0), (1500, [1500, 1023, 1025], 512, 4, 64), (1500, [1500], 68, 4, 64),
    (1500, [1499, 1500], 1499, 0, 3), (40000, [40000], 9999, 4, 250), (130_001, [130_001], 70_000, 1, 0), (300, [300], 300, 4, 4),
])
def test_select_rows(positions, lengths, keep, sinks, recent):
    w = draw(positions + keep, 2, len(lengths), 3, positions, std=2).exp()
    w[w < 0.1] = 0  # ties
    check_rows(w, lengths, keep, sinks, recent)
    check_rows(w, lengths, keep, sinks, recent, kept=torch.zeros_like(w))
    check_rows(w.round(), lengths, keep, sinks, recent)
    check_rows(w, lengths, keep, sinks, recent, kept=w)


@pytest.mark.gpu
@pytest.mark.parametrize("n", [700, 8191, 8197, 16384, 16385, 54016 + 9, 60_001])
def test_select_rows_of_weights_that_begin_alike(n):
    """All of one leading digit, of two, and of few values: none, some or most of the rows share what the limit begins with."""
    x = draw(n, 1, 2, 3, n).abs() % 1
    for w in (1 + x / 8, 1 + x * 2**-14, 1 + (x * 50).round() / 512, x * 3):
        for keep in (n // 10, n - 70):
            check_rows(w, [n, n - 13], keep, 3, 20)


@pytest.mark.gpu
def test_select_rows_of_unusual_weights():
    n = 2500
    for fill in (0.0, -1.0, -math.inf, math.inf, math.nan):
        w = torch.full((1, 1, 2, n), fill).cuda()
        check_rows(w, [n], 700, 3, 5)
        w[..., 100::7] = 2.0
        w[..., 101::14] = -2.0
        w[0, 0, 0, 200::50] = math.nan
        w[0, 0, 1, 300::70] = -0.0
        w[0, 0, 1, 301::71] = 0.0
        check_rows(w, [n], 700, 3, 5)
    check_rows(draw(1, 1, 1, 2, n) * 1e-42, [n], 333, 0, 0)  # (numbers below the smallest normal one)
    w = draw(2, 3, 2, 4, 999)
    check_rows(w[1:, :1, ::2, 100:900], [800], 99, 1, 1)
    view = w[1:, :1, ::2, 100:900]
    check_rows(view, [800], 99, 1, 1, kept=view)


@pytest.mark.gpu
@pytest.mark.parametrize("dim,dtype", [(64, BF16), (128, BF16), (8, BF16), (24, BF16), (256, F32)])
@pytest.mark.parametrize("positions,lengths,keep", [(1, [1], 1), (50, [50, 20, 0, 33], 20), (3000, [3000, 2999], 1111), (3000, [2000], 1999)])
def test_move_rows(positions, lengths, keep, dim, dtype):
    heads, b = 3, len(lengths)
    k, v = (draw(s, 2, b, positions, heads, dim, std=9).to(dtype) for s in (1, 2))
    rows = rows_reference(draw(3, 2, b, heads, positions), lengths, keep, 0, min(keep, 1)).cuda()
    want = []
    for c in (k, v):
        new = c.clone()
        for s, n in enumerate(lengths):
            n = min(n, keep)
            at = rows[:, s, :, :n].long().transpose(1, 2).unsqueeze(-1).expand(-1, -1, -1, dim)
            new[:, s, :n] = c[:, s].gather(1, at)
        want.append(new)
    one = k.clone()
    given = torch.tensor(lengths, dtype=torch.int32).cuda()
    ops.move_rows(k, v, rows, given)
    ops.move_rows(one, None, rows, given)
    torch.cuda.synchronize()
    assert torch.equal(k, want[0]) and torch.equal(v, want[1]) and torch.equal(one, want[0])


@pytest.mark.gpu
def test_move_rows_leaves_alone_what_it_is_not_told():
    k = draw(1, 1, 1, 40, 2, 64, dtype=BF16)
    old = k.clone()
    rows = torch.tensor([[0, 5, -1, 40, 9], [1, 2, 39, 1000, -7]], dtype=torch.int32).cuda().view(1, 1, 2, 5)
    ops.move_rows(k, None, rows, 40)
    for h, pairs in enumerate(({1: 5, 4: 9}, {0: 1, 1: 2, 2: 39})):
        for r in range(40):
            assert torch.equal(k[0, 0, r, h], old[0, 0, pairs.get(r, r), h])


@pytest.mark.gpu
@pytest.mark.parametrize("keep", [5, 700, 2500])
def test_rows_in_any_order_move_at_once(keep):
    """Entries that are no selection: descending, the same one many times, from all over.  Those below their own row leave it as it is, the
    others take what the row held before the call."""
    positions, gen = 3000, torch.Generator().manual_seed(keep)
    rows = torch.stack([torch.arange(positions - 1, positions - 1 - keep, -1), torch.full((keep,), keep // 2), torch.randint(-5, positions + 5, (keep,), generator=gen),
                        torch.zeros(keep, dtype=torch.int64)]).view(1, 2, 2, keep)
    k, v = draw(1, 1, 2, positions, 2, 64, dtype=BF16), draw(2, 1, 2, positions, 2, 64, dtype=BF16)
    want = [k.clone(), v.clone()]
    for b in range(2):
        for h in range(2):
            r = torch.arange(keep)
            take = (rows[0, b, h] > r) & (rows[0, b, h] < positions)
            for new, old in zip(want, (k, v)):
                new[0, b, r[take], h] = old[0, b, rows[0, b, h][take], h]
    ops.move_rows(k, v, rows.int().cuda(), positions)
    assert torch.equal(k, want[0]) and torch.equal(v, want[1])


@pytest.mark.gpu
def test_long_caches():
    """Rows further than 2^31 elements from a cache's beginning (2^32 bytes and more): one key of each head draws all weight, and moves."""
    kv_heads, dim, n = 32, 128, 530_000
    k = torch.zeros(1, 1, n + 7, kv_heads, dim, dtype=BF16, device="cuda")
    at = [n - 1 - 5 * h for h in range(kv_heads)]
    assert min(at) * kv_heads * dim > 2**31
    for h, j in enumerate(at):
        k[0, 0, j, h, h] = 64
    for queries in (1, 5):  # few rows, and many
        q = torch.zeros(1, 1, queries, 4 * kv_heads, dim, dtype=BF16, device="cuda")
        for h in range(kv_heads):
            q[..., 4 * h : 4 * h + 4, h] = 4
        w = torch.zeros(1, 1, kv_heads, n + 7, device="cuda")
        ops.key_weights(q, k, w, n, scale=1.0)
        want = torch.zeros(kv_heads, n + 7)
        for h, j in enumerate(at):  # e^256 against n: the others get nothing; queries see the key from its own on
            want[h, j] = 4 * sum(n - queries + t >= j for t in range(queries))
        # (a query that does not see its head's key shares its weight out over the n keys that it sees)
        spread = 4 * queries / (n - queries)
        assert (w[0, 0].cpu() - want).abs().max() <= 1.01 * spread
        assert torch.allclose(w[0, 0].double().sum(dim=1).cpu(), torch.full((kv_heads,), 4.0 * queries, dtype=torch.float64), rtol=2.0**-12, atol=0)
    rows = ops.select_rows(w, n, keep=64, sinks=2, recent=4)
    old = torch.stack([k[0, 0, rows[0, 0, h].long(), h] for h in range(kv_heads)])
    assert all(j in rows[0, 0, h].tolist() for h, j in enumerate(at))
    ops.move_rows(k, None, rows, n)
    assert torch.equal(k[0, 0, :64].transpose(0, 1), old) and old.any()


# ---- together --------------------------------------------------------------------------------------- #
@pytest.mark.gpu
def test_weights_selection_and_move_in_a_graph_on_another_stream():
    """Observe, select and move as an engine does, captured once and replayed on other inputs and other lengths."""
    heads, kv_heads, dim, positions, keep = 8, 2, 64, 500, 100
    q, k, w, scale = weights_case(3, 2, 2, 9, heads, kv_heads, dim, positions, [positions] * 2)
    v = draw(9, *k.shape, dtype=BF16)
    lengths = torch.tensor([500, 77], dtype=torch.int32).cuda()
    state = [q, k, v, w, lengths]
    start = [t.clone() for t in state]

    def passes():
        ops.key_weights(q, k, w, lengths, scale=scale)
        rows = ops.select_rows(w, lengths, keep=keep, sinks=4, recent=16, kept=w)
        ops.move_rows(k, v, rows, lengths)
        return rows

    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        passes()
    torch.cuda.current_stream().wait_stream(side)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        rows = passes()
    for turn, given in enumerate(([500, 77], [333, 500], [0, 99])):
        for t, s in zip(state, start):
            t.copy_(s)
        q.copy_(draw(100 + turn, *q.shape))
        lengths.copy_(torch.tensor(given))
        want, tol = weights_reference(q, k, w, given, scale)
        alone = w.clone()
        ops.key_weights(q, k, alone, lengths, scale=scale)
        graph.replay()
        torch.cuda.synchronize()
        expected = rows_reference(alone, given, keep, 4, 16)
        assert torch.equal(rows.cpu(), expected)
        for b, n in enumerate(given):
            n = min(n, keep)
            at = expected[:, b, :, :n].long().cuda()
            assert torch.equal(w[:, b, :, :n], alone[:, b].gather(2, at))
            full = at.transpose(1, 2).unsqueeze(-1).expand(-1, -1, -1, dim)
            assert torch.equal(k[:, b, :n], start[1][:, b].gather(1, full)) and torch.equal(v[:, b, :n], start[2][:, b].gather(1, full))
        assert ((alone.double() - want).abs() <= (tol + 2 * HALF) * want).all()


@pytest.mark.gpu
def test_two_selections_at_once_on_two_streams():
    jobs = [(draw(i, 8, 32003, dtype=BF16, std=2), draw(i + 9, 2, 4)) for i in range(2)]
    alone = [[t.clone() for t in ops.beam_select(x, s, beams=4, k=8)] for x, s in jobs]
    streams = [torch.cuda.Stream() for _ in jobs]
    torch.cuda.synchronize()
    for _ in range(20):
        got = [ops.beam_select(x, s, beams=4, k=8, stream=stream) for (x, s), stream in zip(jobs, streams)]
        torch.cuda.synchronize()
        for a, b in zip(alone, got):
            assert all(torch.equal(x, y) for x, y in zip(a, b))
    handle = ops.beam_select(*jobs[0], beams=4, k=8, stream=streams[1].cuda_stream)
    torch.cuda.synchronize()
    assert all(torch.equal(x, y) for x, y in zip(alone[0], handle))
