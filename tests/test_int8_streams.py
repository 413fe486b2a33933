"""The streams that the 8-bit operators take as `stream=`: torch's, foreign handles, and the default one, whose handle is 0."""
import pytest
import torch

from elips_b200._device import as_stream


def test_default_stream_is_no_new_one(monkeypatch):
    def refuse(*args, **kwargs):
        raise AssertionError("a new stream")
    monkeypatch.setattr(torch.cuda, "ExternalStream", refuse)
    monkeypatch.setattr(torch.cuda, "default_stream", lambda device: ("default", device))
    for stream in (0, 1):
        assert as_stream(stream, 3) == ("default", 3)
        assert as_stream(type("Foreign", (), {"cuda_stream": stream})(), 3) == ("default", 3)


@pytest.mark.parametrize("handle", [0, 1 << 40])
def test_torch_streams(monkeypatch, handle):
    """Used as they are on their own device, the default one too, and on no other."""
    class Stream:
        device_index, cuda_stream = 2, handle
    monkeypatch.setattr(torch.cuda, "Stream", Stream)
    stream = Stream()
    assert as_stream(stream, 2) is stream
    with pytest.raises(ValueError, match="cuda:2"):
        as_stream(stream, 0)


def test_foreign_handles(monkeypatch):
    monkeypatch.setattr(torch.cuda, "ExternalStream", lambda handle, device: (handle, device))
    assert as_stream(1 << 40, 2) == (1 << 40, 2)
    assert as_stream(type("Foreign", (), {"cuda_stream": 1 << 40})(), 2) == (1 << 40, 2)


@pytest.mark.gpu
@pytest.mark.parametrize("given", ["stream", "handle"])
def test_on_the_default_stream(given):
    """Each call waits for what the default stream was given before it, on whatever stream the caller is."""
    from elips_b200 import int8
    default = torch.cuda.default_stream()
    stream = default if given == "stream" else default.cuda_stream
    g = torch.Generator(device="cuda").manual_seed(1)
    x = torch.randn((300, 2, 64), generator=g, device="cuda")
    w, sw = int8.quantize_rows(torch.randn((200, 128), generator=g, device="cuda"))
    slots, table, offsets = torch.arange(300, device="cuda"), torch.arange(300, device="cuda")[None], torch.tensor([0, 300], device="cuda")

    def calls(y, **kw):
        codes = torch.zeros((1, 300, 1, 2, 64), dtype=torch.int8, device="cuda")
        scales = torch.zeros((1, 300, 1, 2), device="cuda")
        default.wait_stream(torch.cuda.current_stream())
        rows = int8.quantize_rows(y.view(300, 128), **kw)
        int8.cache_write(codes, scales, (y,), slots, **kw)
        return [*rows, int8.linear_int8(y.view(300, 128), w, sw, **kw), int8.gemm_int8(rows[0], w, rows[1], sw, **kw),
                *int8.cache_read(codes, scales, table, offsets, 300, **kw), codes, scales]

    want = calls(x)
    late = torch.zeros_like(x)
    side = torch.cuda.Stream()
    torch.cuda.synchronize()
    with torch.cuda.stream(default):
        torch.cuda._sleep(20_000_000)
        late.copy_(x)
    with torch.cuda.stream(side):
        got = calls(late, stream=stream)
    torch.cuda.synchronize()
    assert all(torch.equal(a, b) for a, b in zip(got, want))


@pytest.mark.gpu
@pytest.mark.skipif(torch.cuda.device_count() < 2, reason="needs two GPUs")
def test_stream_of_another_device_refused():
    from elips_b200 import int8
    with pytest.raises(ValueError):
        int8.quantize_rows(torch.zeros((4, 8), device="cuda:0"), stream=torch.cuda.Stream(device=1))
