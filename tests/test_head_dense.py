"""The multiclass linear model on dense rows (``dense_head``): the rows, labels and weights that reach the class head are the
files' own, and building the rows repeats bit by bit."""
import pytest
import torch

from test_head import Ref, U, label_targets, near


@pytest.mark.gpu
def test_repeated_features_add_up_the_same_every_time(cuda):
    """A feature named many times in a row: the order of its sum does not change from call to call."""
    from ytk_learn_amd.models.continuous.multiclass import dense_rows
    from ytk_learn_amd.ops.sparse import SparseMatrix

    g = torch.Generator().manual_seed(5)
    n, F, each = 64, 7, 700
    cols = torch.randint(0, F, (n * each,), generator=g, dtype=torch.int32)
    vals = torch.randn(n * each, generator=g) * 10.0 ** torch.randint(-6, 7, (n * each,), generator=g)
    X = SparseMatrix((torch.arange(n + 1) * each).to(cuda), cols.to(cuda), vals.to(cuda), F)
    first = dense_rows(X)
    exact = torch.zeros(n, F, dtype=torch.float64)
    at = (torch.repeat_interleave(torch.arange(n), each), cols.long())
    exact.index_put_(at, vals.double(), accumulate=True)
    size = torch.zeros(n, F, dtype=torch.float64).index_put_(at, vals.double().abs(), accumulate=True)
    near(first, exact, each * U * size, "rows")
    for _ in range(8):
        assert torch.equal(dense_rows(X), first)


def _files(tmp, K):
    """Rows, labels and weights of two files, with absent features; the text holds them exactly."""
    out = {}
    g = torch.Generator().manual_seed(K)
    for name, n in (("tr", 230), ("te", 70)):
        x = torch.randint(-64, 65, (n, 9), generator=g).double() / 32
        x[torch.rand(n, 9, generator=g) < 0.3] = 0.0
        y = torch.randint(0, K, (n,), generator=g)
        y[:min(n, K)] = torch.arange(min(n, K))  # the last class, which has no weights, among them
        wt = torch.randint(1, 9, (n,), generator=g).double() / 4
        with open(f"{tmp}/{name}.txt", "w") as f:
            for i in range(n):
                f.write(f"{float(wt[i])}###{int(y[i])}###" + ",".join(f"f{j}:{float(x[i, j])}" for j in range(9) if x[i, j] != 0 or j == i % 9) + "\n")
        out[name] = (x, y, wt)
    return out


def _model(tmp, dev, K, dense):
    import os

    from ytk_learn_amd.config.hocon import parse_file
    from ytk_learn_amd.config.params import CommonParams
    from ytk_learn_amd.parallel.comm import Comm
    from ytk_learn_amd.train import build_continuous_model
    from ytk_learn_amd.utils.logging import get_logger

    root = os.path.dirname(os.path.dirname(os.path.abspath(__file__)))
    c = parse_file(os.path.join(root, "config", "model", "multiclass_linear.conf")).with_overrides({
        "data.train.data_path": f"{tmp}/tr.txt", "data.test.data_path": f"{tmp}/te.txt", "model.data_path": f"{tmp}/m", "k": K,
        "loss.evaluate_metric": [], "dense_head": dense})
    comm = Comm.local(dev)
    return build_continuous_model("multiclass_linear", CommonParams.from_config(c, "multiclass_linear"), comm, comm.device, get_logger(comm))


def _dense_model(tmp, dev, K):
    files = _files(tmp, K)
    model, sparse = _model(tmp, dev, K, True), _model(tmp, dev, K, False)
    assert model.data.names == sparse.data.names and model.F == 10
    g = torch.Generator().manual_seed(1)
    W = torch.randn(10, K - 1, generator=g).to(model.device)
    col = [9 if name == "_bias_" else int(name[1:]) for name in model.data.names]
    for part, call, call_sparse in (("tr", model.pure_loss_grad, sparse.pure_loss_grad), ("te", model.test_pure_loss_grad, sparse.test_pure_loss_grad)):
        x, y, wt = files[part]
        x = torch.cat([x, torch.ones(len(x), 1, dtype=torch.float64)], 1)[:, col].float()
        ref = Ref(x, W.t(), *label_targets(y), weight=wt, base=True)
        grad = torch.empty(10 * (K - 1), device=model.device)
        loss = call(W.reshape(-1), grad)
        assert abs(loss - float(ref.loss.sum())) <= float(ref.eloss.sum())
        near(grad.view(10, K - 1).t(), ref.dw, ref.edw, "gradient")
        assert abs(call_sparse(W.reshape(-1), None) - loss) <= 2 * float(ref.eloss.sum())


@pytest.mark.parametrize("K", [3, 90])
def test_dense_model_takes_the_files_rows_cpu(tmp_path, K):
    _dense_model(str(tmp_path), "cpu", K)


@pytest.mark.gpu
@pytest.mark.parametrize("K", [3, 90, 300])
def test_dense_model_takes_the_files_rows_gpu(cuda, tmp_path, K):
    _dense_model(str(tmp_path), cuda, K)
