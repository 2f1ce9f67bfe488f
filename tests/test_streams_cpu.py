"""Which stream a call runs on, from what it was given."""
import linalg_b200 as lb


class Stream:
    """As torch's streams are: the default one has handle 0."""

    def __init__(self, handle):
        self.cuda_stream = handle


def test_a_stream_object_names_its_own_stream():
    assert lb._stream(Stream(0x7f00)) == 0x7f00
    # 0 as an argument is the context's stream; the default stream of the device goes by its other name, 1
    assert lb._stream(Stream(0)) == 1


def test_none_and_handles_are_as_they_were():
    assert lb._stream(None) is None
    assert lb._stream(0) == 0 and lb._stream(1) == 1 and lb._stream(0x7f00) == 0x7f00


def test_an_object_without_a_handle_names_the_contexts_stream():
    assert lb._stream(Stream(None)) is None
