"""A pass over drafted tokens is judged by its own states and tokens or not at
all: whatever replaces them in between is noticed."""
import pytest
import torch

from tests.test_gpu_tree import _model

pytestmark = pytest.mark.gpu


def _drafted(dev):
    m = _model(dev)
    m.set_drafts(8)
    m.forward([4, 5, 6], 0)
    return m


def _seed(x):
    return torch.tensor([x], dtype=torch.int32, device="cuda")


def test_seeding_lock_step_decoding_takes_the_drafts_away(dev):
    """start_slots replaces the tokens that a verification compares with."""
    m = _drafted(dev)
    for tokens in ([9], _seed(9)):
        m.forward_tree([[1, 2]], [[-1, 0]], [3])
        m.start_slots(tokens, [3])
        with pytest.raises(ValueError, match="another pass"):
            m.verify_tree()
        m.commit_tree()  # nothing verified: nothing to commit
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.verify_tree()
    m.free()


def test_a_replayed_step_takes_the_drafts_away(dev):
    """The captured decode step and the captured lock-step ones replace tokens
    and hidden states at every replay, the first one after a pass over drafted
    tokens included."""
    m = _drafted(dev)
    m.capture_decode()
    m.start_decode(_seed(3), 5)
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.graph.replay()
    with pytest.raises(ValueError, match="another pass"):
        m.verify_tree()
    m.set_slots(2)
    m.start_slots([3, 4], [0, 0])
    m.slots_step(2, graph=True)
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.slot_graphs[2].replay()
    with pytest.raises(ValueError, match="another pass"):
        m.verify_tree()
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.verify_tree()
    m.free()


def test_a_pass_that_fails_leaves_none_to_judge(dev):
    """Where one of a pass's calls is refused, neither its half-made states nor
    an earlier pass's, whose draft entries it has begun to replace, are there."""
    m = _drafted(dev)
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    m.verify_tree()
    call = m._call

    def refuse(name, *args):
        if name == "gx_qwen_attention_tree":
            raise MemoryError(name)
        call(name, *args)

    m._call = refuse
    with pytest.raises(MemoryError):
        m.forward_tree([[7, 8]], [[-1, 0]], [3])
    m._call = call
    for step in (m.verify_tree, m.commit_tree):
        with pytest.raises(ValueError, match="no pass over drafted"):
            step()
    # a pass refused for its arguments has replaced nothing
    m.forward_tree([[1, 2]], [[-1, 0]], [3])
    want = [x.clone() for x in m.verify_tree()]
    with pytest.raises(ValueError, match="no earlier node"):
        m.forward_tree([[7, 8]], [[-1, 4]], [3])
    for x, y in zip(want, m.verify_tree()):
        assert torch.equal(x, y)
    m.commit_tree()
    m.free()


def test_tensors_of_another_gpu_are_refused(dev):
    """Random numbers and draft logits that are not on the model's device."""
    m = _drafted(dev)
    m.forward_tree([[1, 2]], [[-1, 0]], [3])

    class Elsewhere:
        dtype, is_cuda, device = torch.float32, True, torch.device("cuda", 1)

        def __init__(self, *shape):
            self.shape = shape

        def is_contiguous(self):
            return True

        def data_ptr(self):
            raise AssertionError("its address was asked for")

    with pytest.raises(ValueError, match="random numbers.*cuda:1"):
        m.verify_tree(0.5, uniforms=Elsewhere(2))
    with pytest.raises(ValueError, match="draft logits.*cuda:1"):
        m.verify_tree(0.5, draft_logits=Elsewhere(2, m.cfg.vocab), uniforms=torch.rand(2, device="cuda"))
    m.free()
