"""Host-side edges of the attention wrappers that need no GPU."""
import types


def test_a_stream_that_is_none_is_the_contexts_own():
    """Device.set_stream(None), as before the attention operators: the context's own stream, known to them as None."""
    from mrl_b200.api import Device

    seen = []
    dev = Device.__new__(Device)
    dev.ptr = None
    dev.lib = types.SimpleNamespace(mrl_ctx_set_stream=lambda ptr, s: seen.append(s.value) or 0)
    for stream, kept in ((None, None), (0, None), (77, 77), (1, 1)):
        dev.set_stream(stream)
        assert dev.torch_stream == kept and seen[-1] == kept
