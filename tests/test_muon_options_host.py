"""Options of the optimiser of matrices are checked for every group of parameters (no GPU needed)."""
import pytest

torch = pytest.importorskip("torch")

from f2cgt_amd import pipeline  # noqa: E402

BAD = [{"scale": "Spectral"}, {"lr": -0.1}, {"lr": float("nan")}, {"momentum": 1.0}, {"momentum": -0.1}, {"weight_decay": -1.0}, {"lr": 1.0, "weight_decay": 1.0},
       {"steps": 0}, {"steps": 101}, {"coefficients": (30.0, 0.0, 0.0)}, {"coefficients": (float("nan"), 0.0, 0.0)}, {"coefficients": (1.5, -0.5)}]


def _matrix(dtype=torch.float32):
    return torch.nn.Parameter(torch.zeros(3, 4, dtype=dtype))


@pytest.mark.parametrize("bad", BAD, ids=str)
def test_every_group(bad):
    with pytest.raises(ValueError):
        pipeline.Muon([_matrix()], **bad)
    with pytest.raises(ValueError):
        pipeline.Muon([{"params": [_matrix()]}, {"params": [_matrix()], **bad}])
    opt = pipeline.Muon([_matrix()])
    with pytest.raises(ValueError):
        opt.add_param_group({"params": [_matrix()], **bad})
    assert len(opt.param_groups) == 1
    opt.add_param_group({"params": [_matrix()], "scale": "rms", "lr": 0.5, "steps": 7, "coefficients": (1.5, -0.5, 0.0)})
    assert opt.param_groups[1]["scale"] == "rms" and opt.param_groups[1]["momentum"] == 0.95


def test_steps_are_a_whole_number():
    with pytest.raises(TypeError):
        pipeline.Muon([{"params": [_matrix()], "steps": 2.5}])
    pipeline.Muon([{"params": [_matrix()], "steps": torch.tensor(3)}])


def test_parameters():
    for bad in (torch.nn.Parameter(torch.zeros(3)), _matrix(torch.float64), _matrix(torch.complex64)):
        with pytest.raises(ValueError):
            pipeline.Muon([_matrix(), bad])
    for dtype in (torch.float16, torch.bfloat16):
        pipeline.Muon([_matrix(dtype)])
    opt = pipeline.Muon([_matrix()])
    opt.param_groups[0]["params"][0].grad = torch.zeros(3, 4)
    with pytest.raises(ValueError):                          # on the host
        opt.step()


@pytest.mark.gpu
@pytest.mark.parametrize("bad", BAD, ids=str)
def test_no_group_steps_with_another_ones_options_bad(bad):
    params = [torch.nn.Parameter(torch.randn((5, 6), device="cuda")) for _ in range(2)]
    opt = pipeline.Muon([{"params": [p]} for p in params])
    for p in params:
        p.grad = torch.randn_like(p)
    before = [p.detach().clone() for p in params]
    opt.param_groups[1].update(bad)                          # as a scheduler or a loaded state may
    with pytest.raises(ValueError):
        opt.step()
    assert all(torch.equal(p.detach(), b) for p, b in zip(params, before)) and not opt.state
    opt.param_groups[1].update({k: opt.defaults[k] for k in bad})
    params[1].grad = torch.randn((5, 6), device="cuda").to_sparse()
    with pytest.raises(ValueError):
        opt.step()
    assert torch.equal(params[0].detach(), before[0])
    params[1].grad = torch.randn_like(params[1])
    opt.step()
    assert not torch.equal(params[1].detach(), before[1])
