"""The caption losses around the word operators where a call goes wrong easily."""
import pytest
import torch

from tests import words_common  # noqa: F401  (first: the binding)
from tests.test_word_paths import DEVICES, _losses
from scan2cap_amd import loss_helper as lh


@pytest.mark.parametrize("device", DEVICES)
def test_a_teacher_in_the_students_dict_is_refused(device):
    dd, teacher = _losses(device)
    own = dict(dd)
    for wrong in (own, dict(lang_cap=own["lang_cap"])):
        with pytest.raises(ValueError, match="dict of its own"):
            lh.attach_teacher(own, wrong, top_k=4)
    assert "teacher_top_ids" not in own
    # a teacher that ran first, for a student that has not run yet
    early = {k: v for k, v in dd.items() if k != "lang_cap"}
    lh.attach_teacher(early, teacher, top_k=4)
    late = lh.attach_teacher(dict(dd), teacher, top_k=4)
    assert torch.equal(early["teacher_top_ids"], late["teacher_top_ids"])
