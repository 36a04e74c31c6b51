"""Workspace sizes depend on a device's compute units: they are asked for with that device as the current one, whichever is current
in the caller's thread."""
import contextlib

import pytest
import torch

import self_forcing_amd as sfa

blk, l8 = sfa.block_ops, sfa.linear8


@pytest.mark.parametrize("ask", [lambda i: l8._bytes("sfm_linear8_bwd_workspace_bytes", 300, 64, 128, i),
                                 lambda i: l8._bytes("sfm_linear8_wgrad_workspace_bytes", 300, 64, 128, i), lambda i: blk._ln_bwd_bytes(300, 64, 300, i)])
def test_the_device_is_current(monkeypatch, ask):
    current = [0]

    @contextlib.contextmanager
    def device(index):
        was, current[0] = current[0], index
        yield
        current[0] = was

    class Library:
        def __getattr__(self, name):
            def query(*args):
                args[-1]._obj.value = 1000 + current[0]
                return 0
            return query
    monkeypatch.setattr(torch.cuda, "device", device)
    monkeypatch.setattr(l8._l, "load", Library)
    for f in (l8._bytes, blk._ln_bwd_bytes):
        f.cache_clear()
    try:
        assert [ask(i) for i in (0, 1, 0, 3)] == [1000, 1001, 1000, 1003] and current == [0]
    finally:
        for f in (l8._bytes, blk._ln_bwd_bytes):
            f.cache_clear()
