"""The library's own fills: every byte asked for and no other, and captured work that contains one."""
import pytest
import torch

pytestmark = pytest.mark.gpu


def test_accumulator_reset_at_any_address_and_size(gpu_device):
    from evfly_amd import _lib
    L = _lib.lib()
    buf = torch.empty(3 << 20, dtype=torch.uint8, device="cuda")
    for off in (0, 1, 7, 15, 16, 33):
        for n in (1, 3, 15, 16, 17, 31, 64, 70, 89960, (2 << 20) + 5):
            buf.fill_(7)
            _lib.check(L.evfly_accumulate_reset(buf.data_ptr() + 64 + off, n, _lib.cur_stream()))
            lo, hi = 64 + off, 64 + off + n
            assert (buf[:lo] == 7).all() and (buf[lo:hi] == 128).all() and (buf[hi:] == 7).all(), (off, n)


def test_conditioning_in_a_graph(gpu_device):
    """condition_frames clears its working memory on every call: captured, replayed with new frames and eager calls between, it gives the eager bits."""
    from evfly_amd import synthetic as syn, voxelizer
    sets = [torch.from_numpy(syn.make_frames(s, 6)).cuda().clamp(-1, 1).reshape(6, 260, 346).contiguous() for s in (3, 4, 5, 6)]
    src = sets[0].clone()
    side = torch.cuda.Stream()
    side.wait_stream(torch.cuda.current_stream())
    with torch.cuda.stream(side):
        voxelizer.condition_frames(src, out_hw=(260, 346))
        side.synchronize()
        g = torch.cuda.CUDAGraph()
        with torch.cuda.graph(g, stream=side):
            got = voxelizer.condition_frames(src, out_hw=(260, 346))
    torch.cuda.synchronize()
    for s in sets:
        src.copy_(s)
        want = voxelizer.condition_frames(s, out_hw=(260, 346))
        g.replay()
        torch.cuda.synchronize()
        assert torch.equal(got, want)
