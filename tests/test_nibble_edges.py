"""The 4-bit cache's entry points on the CPU: refusals that go with their edge cases (nothing is
launched)."""
from vllm_ttkv import _hip


def _refused(rc, code, text):
    msg = _hip.lib().ttkv_last_error().decode()
    assert rc == code and text in msg, (rc, msg)


def test_decode_starts_refusals():
    def call(starts, R):
        return _hip.lib().ttkv_nibble_decode_starts_paged(
            8, 24, 128, 0.088, 16, 1, 24 * 128, 4096, 64, 1152, 16, 16, 4, 4, 16, 16, starts, R, 64,
            16, 1, 24 * 128, 256, 1 << 30, 16, None)
    _refused(call(1, 2), 1, "query starts")
    _refused(call(0, 1), 1, "query starts")
    _refused(call(-1, 1), 1, "query starts")
    assert call(0, 0) == 0 and call(1, 0) == 0                      # nothing to do
