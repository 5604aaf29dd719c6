"""qw_buf_upload and qw_kv_store are blocking copies: what a command buffer does next, on a stream that does not order
with the default one, comes after the last uploaded byte."""
import numpy as np
import pytest

from gpu_util import Bufs, QwRef

pytestmark = pytest.mark.gpu


def test_upload_has_landed_when_it_returns(be):
    n, tail = 3 << 20, 64 << 10
    with Bufs(be) as B:
        zero, dst = B.device(np.zeros(tail, np.uint8)), B.device(np.zeros(n, np.uint8))
        got = np.empty(tail, np.uint8)
        for i in range(40):
            src = np.full(n, 1 + i, np.uint8)
            c = be.cmd_begin()
            be.buf_upload(dst, 0, src)
            be.op_copy(c, QwRef(dst, n - tail), QwRef(zero, 0), tail)      # must overwrite the upload's last bytes
            be.cmd_wait(c)
            be.cmd_free(c)
            be.buf_download(dst, n - tail, got)
            assert not got.any(), i


def test_store_has_landed_when_it_returns(be):
    n = 4096
    with Bufs(be) as B:
        arena, zeros = B.arena(1, 1, n), B.device(np.zeros((64, 256), np.float32))
        for i in range(20):
            c = be.cmd_begin()
            be.kv_store(arena, 0, 0, 0, np.full((n, 256), 0x3F80 + i, np.uint16), 1, n)
            be.op_kv_write(c, QwRef(arena, 0), QwRef(B.arena(1, 1, n), 0), QwRef(zeros, 0), QwRef(zeros, 0), 64, 1, 256, n, n - 64)
            be.cmd_wait(c)
            be.cmd_free(c)
            assert not be.kv_read(arena, 0, 0, n - 64, 64, 1, n).any(), i
