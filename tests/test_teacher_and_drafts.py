"""A teacher, its student and a draft model through the single-process model: top logits -> distillation -> drafts that the
target checks, on CPU."""
import pytest
import torch

from multimodal_training_b200.models.vlm import Qwen2_5_VLForConditionalGeneration
from test_vlm_wrapper import _batch


def test_teacher_targets_leave_out_what_is_not_predicted():
    m = Qwen2_5_VLForConditionalGeneration("tiny", seed=3)
    ids, pix, _ = _batch(m.config, [(1, 16, 16)], text_len=5)
    values, top = m.top_logits(7, ids, pix, [(1, 16, 16)])
    logits = m(ids, pix, [(1, 16, 16)])["logits"]
    assert values.shape == top.shape == (ids.numel(), 7)
    nxt = ids[0, 1:]
    off = torch.cat([nxt == m.config.image_token_id, torch.tensor([True])])
    assert (top[off] == -1).all() and torch.equal(logits.detach().gather(1, top.clamp(min=0))[~off], values[~off])
    assert torch.equal(top[~off, 0], logits[~off].argmax(1))


def test_student_step_against_a_plain_statement():
    teacher = Qwen2_5_VLForConditionalGeneration("tiny", seed=3)
    student = Qwen2_5_VLForConditionalGeneration("tiny", seed=4)
    ids, pix, labels = _batch(teacher.config, [(1, 16, 16)], text_len=5)
    values, top = teacher.top_logits(9, ids, pix, [(1, 16, 16)])
    out = student(ids, pix, [(1, 16, 16)], labels=labels, teacher_ids=top, teacher_logits=values, temperature=2.0,
                  label_weight=0.25)
    out["loss"].backward()
    grads = [p.grad.clone() for p in student.parameters() if p.grad is not None]
    student.zero_grad()
    z = student(ids, pix, [(1, 16, 16)])["logits"]
    rows = top[:, 0] >= 0
    p = (values[rows] / 2).softmax(1)
    kl = (p * (p.log() - (z[rows] / 2).log_softmax(1).gather(1, top[rows]))).sum(1).mean()
    ce = torch.nn.functional.cross_entropy(z[:-1], labels[0, 1:], ignore_index=-100)
    want = 0.75 * 4 * kl + 0.25 * ce
    assert abs(float(out["loss"].detach()) - float(want.detach())) < 1e-4
    want.backward()
    for a, b in zip(grads, [p.grad for p in student.parameters() if p.grad is not None]):
        assert torch.allclose(a, b, rtol=1e-3, atol=1e-6)


def test_greedy_answers_are_the_same_with_a_draft_model():
    target = Qwen2_5_VLForConditionalGeneration("tiny", seed=5)
    ids, pix, _ = _batch(target.config, [(1, 16, 16)], text_len=6)
    want = target.generate(ids[0], pix, [(1, 16, 16)], max_new_tokens=9)
    for draft, n in ((target, 3), (Qwen2_5_VLForConditionalGeneration("tiny", seed=6), 4), (target, 1)):
        assert torch.equal(target.generate(ids[0], pix, [(1, 16, 16)], 9, draft_model=draft, draft_tokens=n), want)
    eos = int(want[ids.numel() + 3])
    first = ids.numel() + int((want[ids.numel():] == eos).nonzero()[0])
    got = target.generate(ids[0], pix, [(1, 16, 16)], 9, eos_token_id=eos, draft_model=target, draft_tokens=4)
    assert torch.equal(got, want[:first + 1])
    assert torch.equal(target.generate(ids[0], pix, [(1, 16, 16)], 0, draft_model=target), ids[0])


def test_sampled_answers_and_refusals():
    target = Qwen2_5_VLForConditionalGeneration("tiny", seed=5)
    draft = Qwen2_5_VLForConditionalGeneration("tiny", seed=6)
    ids = torch.randint(0, 900, (11,), generator=torch.Generator().manual_seed(1))

    def draw(**kw):
        return target.generate(ids, max_new_tokens=6, temperature=0.9, generator=torch.Generator().manual_seed(2), **kw)

    a, b = draw(), draw(draft_model=draft, draft_tokens=2)
    assert a.shape == b.shape == (17,) and torch.equal(a, draw()) and torch.equal(b, draw(draft_model=draft, draft_tokens=2))
    assert torch.equal(a[:11], ids) and bool((a < target.config.text.vocab_size).all() and (a >= 0).all())
    with pytest.raises(ValueError):
        draw(draft_model=draft, draft_tokens=0)
    with pytest.raises(ValueError):
        draw(draft_model=Qwen2_5_VLForConditionalGeneration("smoke", seed=6))


def test_logits_that_are_no_distribution_are_refused():
    target = Qwen2_5_VLForConditionalGeneration("tiny", seed=5)
    draft = Qwen2_5_VLForConditionalGeneration("tiny", seed=6)
    ids = torch.randint(0, 900, (5,), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():
        draft.model.language_model.norm_w.fill_(float("nan"))
    for model, kw in ((target, dict(draft_model=draft)), (draft, {})):
        with pytest.raises(RuntimeError, match="no distribution"):
            model.generate(ids, max_new_tokens=3, temperature=1.0, **kw)


def test_placeholders_are_not_drawn():
    m = Qwen2_5_VLForConditionalGeneration("tiny", seed=5)
    ids = torch.randint(0, 900, (5,), generator=torch.Generator().manual_seed(1))
    with torch.no_grad():                           # nothing but the two placeholders would be drawn
        m.model.language_model.logits = lambda h, plain=m.model.language_model.logits: plain(h).index_add(
            1, torch.tensor([m.config.image_token_id, m.config.video_token_id]), torch.full((h.shape[0], 2), 1e4))
        got = m.generate(ids, max_new_tokens=6, temperature=1.0, generator=torch.Generator().manual_seed(0))
    assert got.numel() == 11
    assert not ((got == m.config.image_token_id) | (got == m.config.video_token_id)).any()
    with pytest.raises(ValueError, match="negative"):
        m.generate(ids, max_new_tokens=2, temperature=-1.0)
