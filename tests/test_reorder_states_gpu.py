"""States in the beams' new order, in place, against index_select, bit for bit."""
import pytest
import torch

from quamba_amd import ops

pytestmark = pytest.mark.gpu


def reference(states, parents):
    batch, beams = parents.shape
    p = parents.long()
    own = torch.arange(beams, device=p.device).expand(batch, beams)
    p = torch.where((p >= 0) & (p < beams), p, own)
    rows = (p + beams * torch.arange(batch, device=p.device)[:, None]).reshape(-1)
    return [s.clone()[rows] for s in states]


def check(states, parents):
    want = reference(states, parents)
    assert ops.reorder_states(states, parents) is None
    for s, w in zip(states, want):
        assert torch.equal(s.contiguous().view(torch.uint8), w.contiguous().view(torch.uint8))


def some(rows, shape, dtype, dev, seed=0):
    g = torch.Generator().manual_seed(seed + rows)
    if dtype.is_floating_point:
        return torch.randn(rows, *shape, generator=g).to(dtype).to(dev)
    return torch.randint(-100, 100, (rows, *shape), generator=g).to(dtype).to(dev)


@pytest.mark.parametrize("index", [torch.int32, torch.int64])
@pytest.mark.parametrize("batch,beams", [(1, 1), (1, 2), (3, 3), (1, 4), (5, 4), (2, 5), (2, 8), (1, 9), (3, 16), (2, 17), (1, 32), (2, 33), (1, 64), (70, 2)])
def test_sizes(dev, index, batch, beams):
    """rows of 16 bytes' multiples, of 4 bytes', and of any number of them"""
    g = torch.Generator().manual_seed(batch + beams)
    rows = batch * beams
    for _ in range(3):
        parents = torch.randint(0, beams, (batch, beams), generator=g).to(index).to(dev)
        check([some(rows, (64, 16), torch.float32, dev), some(rows, (64, 4), torch.int8, dev), some(rows, (33, 3), torch.int8, dev), some(rows, (5,), torch.float32, dev),
               some(rows, (7,), torch.float16, dev), some(rows, (1000, 2), torch.int64, dev), some(rows, (), torch.bfloat16, dev), some(rows, (3000, 16), torch.int8, dev)], parents)


@pytest.mark.parametrize("beams", [4, 6, 40])
def test_orders(dev, beams):
    """as it is, all from one, exchanges and rings, and parents that are none of them"""
    ring = torch.arange(beams).roll(1)
    for row in (torch.arange(beams), torch.zeros(beams, dtype=torch.int64), torch.full((beams,), beams - 1), torch.arange(beams).flip(0), ring, ring.roll(1),
                torch.full((beams,), -1), torch.where(torch.arange(beams) % 2 == 0, ring, torch.tensor(-1)), torch.where(torch.arange(beams) % 3 == 0, torch.tensor(beams), ring),
                torch.where(torch.arange(beams) % 3 == 0, torch.tensor(1 << 40), ring), torch.where(torch.arange(beams) % 3 == 0, torch.tensor(-(1 << 40)), ring)):
        parents = torch.stack((row, torch.arange(beams))).to(dev)
        check([some(2 * beams, (50, 16), torch.float32, dev), some(2 * beams, (3,), torch.int8, dev)], parents)


def test_states_as_they_lie(dev):
    """dimensions of a row in any order, rows apart, parts of one buffer between each other's, on any address"""
    parents = torch.tensor([[3, 0, 0, 1], [1, 1, 2, 0]], device=dev)
    transposed = torch.randint(-9, 9, (8, 4, 640), dtype=torch.int8, device=dev).transpose(1, 2)
    check([transposed], parents)
    buffer = torch.randn(8, 100, 16, device=dev)
    check([buffer[:, :60], buffer[:, 60:]], parents)
    odd = torch.randint(-9, 9, (8, 1003), dtype=torch.int8, device=dev)
    kept = odd[:, 901:].clone()
    check([odd[:, 1:501], odd[:, 501:901]], parents)
    assert torch.equal(odd[:, 901:], kept)                         # (columns that are nobody's)
    stacked = torch.randn(3, 8, 33, 16, device=dev)
    check(list(stacked), parents)
    check([torch.randn(10, 40, device=dev)[2:]], parents)
    check([stacked[0]], parents.t().contiguous().t())
    single = torch.randn(8, 24, device=dev)
    want = reference([single], parents)[0]
    ops.reorder_states(single, parents)                            # (a tensor by itself)
    assert torch.equal(single, want)
    check((single,), parents)


def test_rows_behind_the_last_entry_stay(dev):
    buffer = torch.randn(12, 64, device=dev)
    kept = buffer[8:].clone()
    check([buffer[:8]], torch.tensor([[3, 0, 0, 1], [1, 1, 2, 0]], device=dev))
    assert torch.equal(buffer[8:], kept)


def test_many_tensors(dev):
    """more than one launch has room for, of three kinds"""
    parents = torch.tensor([[2, 0, 1], [0, 0, 2]], device=dev)
    states = [some(6, ((16, 40, 3)[i % 3],), (torch.float32, torch.int8, torch.int8)[i % 3], dev, seed=i) for i in range(331)]
    check(states, parents)


def test_nothing(dev):
    ops.reorder_states([], torch.zeros(2, 3, dtype=torch.int64, device=dev))
    ops.reorder_states([torch.zeros(0, 5, device=dev)], torch.zeros(0, 3, dtype=torch.int64, device=dev))
    ops.reorder_states([torch.zeros(6, 0, device=dev)], torch.zeros(2, 3, dtype=torch.int64, device=dev))


def test_versions(dev):
    """what autograd saved is seen to have changed; a state of inference mode has no version"""
    s, parents = torch.randn(4, 8, device=dev), torch.tensor([[1, 0, 0, 2]], device=dev)
    before = s._version
    ops.reorder_states([s], parents)
    assert s._version > before
    with torch.inference_mode():
        t = torch.randn(4, 8, device=dev)
        check([t], parents)


def test_refusals(dev):
    s, parents = torch.randn(8, 16, device=dev), torch.zeros(2, 4, dtype=torch.int64, device=dev)
    before = s.clone()
    for states, p in (([s[:7]], parents), ([s], parents[0]), ([s], parents.float()), ([s], parents.cpu()), ([s.cpu()], parents), ([s, s], parents), ([s, s[:, :4]], parents),
                      ([s[:, :9], s[:, 8:]], parents), ([s, s.t().contiguous().t()[:, ::2]], parents), ([s[:, ::2]], parents), ([s[:1].expand(8, 16)], parents),
                      ([torch.zeros(24, device=dev).as_strided((8, 16), (1, 1))], parents), ([parents.view(8, 1)], parents), ([s.view(8, 4, 4)[:, :, :2]], parents),
                      ([s], parents[:, :0]), ([torch.zeros((), device=dev)], parents)):
        with pytest.raises(RuntimeError):
            ops.reorder_states(states, p)
    # (more rows of another pitch over the same memory)
    buffer = torch.zeros(256, device=dev)
    with pytest.raises(RuntimeError):
        ops.reorder_states([buffer.as_strided((8, 8), (32, 1)), buffer.as_strided((8, 4), (24, 1), 8)], parents)
    for bad in ([s, None], [3], 3, None):
        with pytest.raises(TypeError):
            ops.reorder_states(bad, parents)
    with pytest.raises(NotImplementedError):
        ops.reorder_states([torch.zeros(65, 4, device=dev)], torch.zeros(1, 65, dtype=torch.int64, device=dev))
    with pytest.raises(NotImplementedError):
        ops.reorder_states([torch.zeros(65536, 4, device=dev)], torch.zeros(65536, 1, dtype=torch.int64, device=dev))
    torch.cuda.synchronize()
    assert torch.equal(s, before)


def test_offsets_past_32_bits(dev):
    """rows more than 2 GiB into a state"""
    s = torch.zeros(6, 1 << 30, dtype=torch.int8, device=dev)
    for r in range(6):
        s[r, ::1 << 20] = r + 1
        s[r, -1] = r + 11
    parents = torch.tensor([[1, 2, 0], [2, 2, 0]], device=dev)
    ops.reorder_states([s], parents)
    for r, want in enumerate((1, 2, 0, 5, 5, 3)):
        assert torch.equal(s[r, ::1 << 20], torch.full((1024,), want + 1, dtype=torch.int8, device=dev)) and s[r, -1] == want + 11 and s[r, 1] == 0
    del s


def test_captured_and_on_another_stream(dev):
    states, parents = [torch.randn(8, 40, 16, device=dev), torch.randint(-9, 9, (8, 33), dtype=torch.int8, device=dev)], torch.zeros(2, 4, dtype=torch.int64, device=dev)
    ops.reorder_states([t.clone() for t in states], parents)
    graph = torch.cuda.CUDAGraph()
    with torch.cuda.graph(graph):
        ops.reorder_states(states, parents)
    for step in range(4):
        for t in states:
            t.copy_(some(8, tuple(t.shape[1:]), t.dtype, dev, seed=step))
        parents.copy_(torch.randint(-1, 4, (2, 4), generator=torch.Generator().manual_seed(step)))
        want = reference(states, parents)
        graph.replay()
        torch.cuda.synchronize()
        assert all(torch.equal(a, b) for a, b in zip(states, want)), step
    side = torch.cuda.Stream()
    want = reference(states, parents)
    torch.cuda.synchronize()
    with torch.cuda.stream(side):
        ops.reorder_states(states, parents)
    side.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(states, want))


@pytest.mark.parametrize("beams", [3, 12, 24, 40])
def test_bytes_of_a_row(dev, beams):
    """rows of any number of bytes on any address, next to bytes that are nobody's"""
    g = torch.Generator().manual_seed(beams)
    for length in (1, 3, 4, 15, 16, 17, 31, 1023, 1024 + 3, 16 * 255 + 15, 16 * 256, 16 * 256 + 1, 16 * 257 + 7, 16 * 511 + 15, 16 * 512, 16 * 512 + 15, 16 * 513 + 1, 30011):
        for at in (0, 1, 6):
            buffer = torch.randint(-100, 100, (2 * beams, length + 9), dtype=torch.int8, generator=g).to(dev)
            parents = torch.randint(-1, beams, (2, beams), generator=g).to(dev)
            want = buffer.clone()
            want[:, at:at + length] = reference([buffer[:, at:at + length]], parents)[0]
            ops.reorder_states(buffer[:, at:at + length], parents)
            assert torch.equal(buffer, want), (length, at)
