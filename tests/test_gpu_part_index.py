"""GPU: the part index of parallel-codec slabs (xksv_plan_index on plans of few
slabs) and the ragged serial decode: decoded bytes against the source words,
bit for bit, over shapes whose substreams begin and end anywhere, codebooks of
every kind, odd payload offsets, and streams changed after the index."""
import numpy as np
import pytest

torch = pytest.importorskip("torch")
pytestmark = pytest.mark.gpu

import xksv_gpu as xg  # noqa: E402
from helpers import words_for  # noqa: E402

DEV = "cuda:0"


def slabs(shapes, codec, kind, seed, lead=5):
    rng = np.random.default_rng(seed)
    payload, entries, words, dst = bytearray(b"\0" * lead), [], [], 0
    for rows, cols in shapes:
        w = words_for(kind, rows * cols, rng).astype("<u2")
        blob = xg.host_pack(w.tobytes(), rows, cols, codec)
        entries.append(dict(src_offset=len(payload), src_size=len(blob), rows=rows, cols=cols, dst_offset=dst, codec=codec))
        payload += blob + b"\x5a"
        words.append(w)
        dst += rows * cols * 2
    return torch.frombuffer(payload, dtype=torch.uint8).to(DEV), entries, np.concatenate(words)


# whole rows, odd numbers of tiles, ragged last tiles, few rows, and substreams too short for a second part
SHAPES = [[(16, 8192)], [(16, 4112), (16, 2064)], [(16, 1848)] * 5, [(7, 3000), (16, 13000), (1, 9000)],
          [(16, 40), (3, 5), (16, 9000)], [(16, 28672)] * 3]


@pytest.mark.parametrize("shapes", SHAPES)
@pytest.mark.parametrize("kind", ["normal002", "student3", "uniform", "three_exp", "single"])
def test_parallel_parts_decode_the_same_bytes(shapes, kind):
    payload, entries, want = slabs(shapes, xg.CODEC_PARALLEL32, kind, len(shapes))
    plan = xg.Plan(entries)
    for shift in (0, 2):  # 32-byte aligned output, and not
        for indexed in (False, True):
            if indexed:
                assert plan.index(payload) == 0
            out = torch.full((want.size * 2 + 8,), 0xEE, dtype=torch.uint8, device=DEV)
            plan.decode(payload, out[shift:])
            assert plan.status() == 0
            got = out.cpu().numpy()
            assert (got[shift:shift + want.size * 2].view("<u2") == want).all()
            assert (got[shift + want.size * 2:] == 0xEE).all() and (got[:shift] == 0xEE).all()
    plan.close()


@pytest.mark.parametrize("shapes", [[(16, 1024)] * 2, [(16, 1008)], [(16, 1032), (1, 64), (2, 33)], [(13, 1300)] * 40])
@pytest.mark.parametrize("kind", ["normal002", "uniform", "three_exp"])
def test_parallel_parts_of_few_codes(shapes, kind):
    """Around the smallest slabs that are shared, and parts of two groups."""
    payload, entries, want = slabs(shapes, xg.CODEC_PARALLEL32, kind, 9)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    out = torch.full((want.size * 2 + 8,), 0xEE, dtype=torch.uint8, device=DEV)
    for _ in range(2):
        plan.decode(payload, out)
        assert plan.status() == 0
        got = out.cpu().numpy()
        assert (got[:want.size * 2].view("<u2") == want).all() and (got[want.size * 2:] == 0xEE).all()
        assert plan.index(payload) == 0  # built again
    plan.close()


def test_parallel_parts_report_a_changed_stream():
    payload, entries, want = slabs([(16, 8192)], xg.CODEC_PARALLEL32, "normal002", 3)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    out = torch.empty(want.size * 2, dtype=torch.uint8, device=DEV)
    good = payload.clone()
    # bits of the last substream's end, its bit count, a code length, the container's magic
    e = entries[0]
    seg = e["src_offset"] + 32 + 8 * 32
    for at in (e["src_offset"] + e["src_size"] - 40, seg + 8, seg + 16 + 120, e["src_offset"]):
        payload.copy_(good)
        payload[at:at + 4] ^= 0x55
        plan.decode(payload, out)
        bad = plan.status()
        same = bool((out.cpu().numpy().view("<u2") == want).all())
        assert bad == 1 or same, at
    payload.copy_(good)
    plan.decode(payload, out)
    assert plan.status() == 0 and (out.cpu().numpy().view("<u2") == want).all()
    plan.close()


def test_index_of_a_bad_parallel_slab_leaves_the_decode_to_report_it():
    payload, entries, want = slabs([(16, 8192)], xg.CODEC_PARALLEL32, "normal002", 4)
    payload[entries[0]["src_offset"] + 32 + 8 * 32 + 8] ^= 1
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0 and plan.status() == 0
    plan.decode(payload, torch.empty(want.size * 2, dtype=torch.uint8, device=DEV))
    assert plan.status() == 1
    plan.close()


def test_ragged_tiles_report_a_changed_stream():
    payload, entries, want = slabs([(14, 9000), (16, 520)], xg.CODEC_TILE16, "normal002", 6)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    out = torch.empty(want.size * 2, dtype=torch.uint8, device=DEV)
    bits = entries[0]["src_offset"] + 272 + 14 * 9000
    good = payload.clone()
    for at in (bits + 100, entries[0]["src_offset"] + entries[0]["src_size"] - 8):
        payload.copy_(good)
        payload[at:at + 6] ^= 0x3C
        plan.decode(payload, out)
        assert plan.status() in (0, 1)  # tiles before the change may still read as codes of the right length
        plan.decode(good, out)          # another payload pointer: without the index
        assert plan.status() == 0 and (out.cpu().numpy().view("<u2") == want).all()
    plan.close()


@pytest.mark.parametrize("shapes", [[(14, 11104)], [(16, 1848)] * 3, [(5, 17), (16, 33), (1, 1), (9, 4096)], [(40, 200)],
                                    [(16, 512), (3, 512), (16, 500), (20, 64)], [(1, 30000), (13, 7)]])
@pytest.mark.parametrize("kind", ["normal002", "uniform", "single"])
def test_ragged_serial_slabs_decode(shapes, kind):
    payload, entries, want = slabs(shapes, xg.CODEC_TILE16, kind, len(shapes))
    plan = xg.Plan(entries)
    for indexed in (False, True):
        if indexed:
            assert plan.index(payload) == 0
        out = torch.zeros(want.size * 2, dtype=torch.uint8, device=DEV)
        plan.decode(payload, out)
        assert plan.status() == 0
        assert (out.cpu().numpy().view("<u2") == want).all()
    plan.close()


def test_ragged_tiles_of_a_changed_stream_are_reported_or_read_alike():
    """Bits changed after the index: every element is the source's, or the call
    reports the slab; tiles whose bits are as they were read the same, and
    nothing is written outside the output."""
    rows, cols = 14, 9000
    payload, entries, want = slabs([(rows, cols), (16, 520)], xg.CODEC_TILE16, "normal002", 6)
    plan = xg.Plan(entries)
    assert plan.index(payload) == 0
    first, e = 64, entries[0]
    bits = e["src_offset"] + 272 + rows * cols
    good, last = payload.clone(), e["src_offset"] + e["src_size"]
    words = want[:rows * cols].reshape(rows, cols)
    reported = 0
    # inside the stream, in its first and its last bytes
    for at in (bits, bits + 100, (bits + last) // 2, last - 8):
        for mask in (0x01, 0x3C, 0xFF):
            payload.copy_(good)
            payload[at:at + 2] ^= mask
            out = torch.full((first + want.size * 2 + first,), 0xEE, dtype=torch.uint8, device=DEV)
            plan.decode(payload, out[first:])
            bad = plan.status()
            got = out.cpu().numpy()
            assert (got[:first] == 0xEE).all() and (got[-first:] == 0xEE).all()
            elems = got[first:-first].view("<u2")
            assert (elems[rows * cols:] == want[rows * cols:]).all()  # the other slab
            wrong = (elems[:rows * cols].reshape(rows, cols) != words).any(0).nonzero()[0] // 16
            assert len(set(wrong.tolist())) <= 2, (at, mask)  # two bytes lie in at most two tiles' bits
            reported += bad
    assert reported  # a tile whose codes no longer end where the next one begins
    payload.copy_(good)
    out = torch.empty(want.size * 2, dtype=torch.uint8, device=DEV)
    plan.decode(payload, out)
    assert plan.status() == 0 and (out.cpu().numpy().view("<u2") == want).all()
    plan.close()


def test_index_keeps_an_unread_error():
    """An error that no status call has read yet is still there after an index."""
    for codec, shape in ((xg.CODEC_PARALLEL32, (16, 8192)), (xg.CODEC_TILE16, (16, 1000)), (xg.CODEC_TILE16, (16, 1024))):
        payload, entries, want = slabs([shape], codec, "normal002", 5)
        good = payload.clone()
        plan = xg.Plan(entries)
        payload[entries[0]["src_offset"] + 8:entries[0]["src_offset"] + 10] ^= 1  # a size in the header
        plan.decode(payload, torch.empty(want.size * 2, dtype=torch.uint8, device=DEV))
        assert plan.index(good) == 0
        assert plan.status() == 1 and plan.status() == 0, (codec, shape)
        plan.close()


def test_calls_after_an_index_without_room_for_the_parts():
    """Too little memory for the part index leaves it off, and no more."""
    payload, entries, want = slabs([(16, 1024)] * 1000, xg.CODEC_PARALLEL32, "normal002", 8)
    plan = xg.Plan(entries)
    out = torch.empty(want.size * 2, dtype=torch.uint8, device=DEV)
    plan.decode(payload, out)
    assert plan.status() == 0
    torch.cuda.empty_cache()
    free, _ = torch.cuda.mem_get_info()
    full = None
    for spare in (6, 7, 8, 9):  # the parts' tables take 10 MB
        try:
            full = torch.empty(free - (spare << 20), dtype=torch.uint8, device=DEV)
            break
        except torch.OutOfMemoryError:
            continue
    if full is None:
        pytest.skip("the memory is not there to be taken")
    try:
        assert plan.index(payload) == 0
        plan.decode(payload, out)
        assert plan.status() == 0
    finally:
        del full
        torch.cuda.empty_cache()
    assert (out.cpu().numpy().view("<u2") == want).all()
    plan.close()


def test_index_without_parts():
    """The part index can be left off: its memory is not taken, and decodes are the same."""
    payload, entries, want = slabs([(16, 1024)] * 1000, xg.CODEC_PARALLEL32, "normal002", 9)
    torch.cuda.synchronize()
    taken = []
    for parts in (True, False, True):
        plan = xg.Plan(entries)
        before = torch.cuda.mem_get_info()[0]
        assert plan.index(payload, parts=parts) == 0
        taken.append(before - torch.cuda.mem_get_info()[0])
        out = torch.empty(want.size * 2, dtype=torch.uint8, device=DEV)
        plan.decode(payload, out)
        assert plan.status() == 0 and (out.cpu().numpy().view("<u2") == want).all()
        plan.close()
    assert taken[0] >= 8 << 20 and taken[1] <= 2 << 20 and taken[2] >= 8 << 20  # 10 KB a slab
