"""The word that reports a product's bounded wait, under first calls from several threads.  No GPU."""
import threading
import time

import numpy as np
import pytest
import torch


class SlowWord:
    """A pinned word whose allocation and view take long enough for other threads to come by."""
    made = []

    def __init__(self):
        time.sleep(0.05)
        self.array = np.zeros(1, dtype=np.int32)
        SlowWord.made.append(self)

    def numpy(self):
        time.sleep(0.05)
        return self.array

    def data_ptr(self):
        return self.array.ctypes.data


@pytest.mark.parametrize("late", [0.0, 0.02, 0.07])
def test_first_products_of_several_threads_share_one_word(monkeypatch, late):
    from advanced_optimizers_b200 import fp8
    SlowWord.made.clear()
    monkeypatch.setattr(torch, "zeros", lambda *a, **k: SlowWord())
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: False)
    word, got = fp8._ErrorWord(), []

    def first_product(i):
        time.sleep(i * late)
        try:
            got.append(word.pointer())
        except Exception as e:
            got.append(e)

    threads = [threading.Thread(target=first_product, args=(i,)) for i in range(4)]
    for t in threads:
        t.start()
    for t in threads:
        t.join()
    assert len(SlowWord.made) == 1 and got == [SlowWord.made[0].data_ptr()] * 4


def test_no_word_during_a_capture(monkeypatch):
    from advanced_optimizers_b200 import fp8
    monkeypatch.setattr(torch.cuda, "is_current_stream_capturing", lambda: True)
    word = fp8._ErrorWord()
    assert word.pointer() == 0 and word.word is None
