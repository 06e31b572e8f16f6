"""CPU tests of the decode calls' workspace: an address that its 32-bit counters and partials cannot
have is refused on the host before any HIP call."""
import pytest

from dadgpt_amd import attention as A

FAKE, STEP = 0x1000000, 0x10000000


@pytest.mark.parametrize("name", ["bf16", "f32"])
@pytest.mark.parametrize("window", [None, 1500])
def test_misaligned_workspace(name, window):
    p = [FAKE + i * STEP for i in range(5)]
    f = getattr(A.lib(), "dadgpt_decode_attention_" + ("" if window is None else "window_") + name)
    more = [] if window is None else [window, 4]
    need = A.decode_workspace_bytes(4, 2, 2000, 64)
    for off in (1, 2, 3, 6):
        assert f(*p, 4, 2, 2000, 64, 0.125, *more, FAKE + 8 * STEP + off, need, None) == 1
        assert "workspace is not 4-byte aligned" in A.last_error()
