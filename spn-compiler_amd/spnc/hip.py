"""``HIPCompiler``: compile SPNs for AMD MI355X (gfx950) and run batched log-likelihood inference.

Same surface as the reference's ``CUDACompiler`` (python-interface/spnc/gpu.py:24-219): constructor
flags ``preloadToSharedMem`` / ``computeInLogSpace`` / ``verbose`` plus free-form compiler options,
``compile_ll`` -> kernel, ``execute(kernel, inputs)``, ``log_likelihood(spn, inputs)`` and the static
``isAvailable()``. Error messages for bad inputs are the reference's.
"""
import os
import tempfile

import numpy as np

from xspn.serialization.binary.BinarySerialization import BinarySerializer
from xspn.structure.Model import SPNModel
from xspn.structure.Query import ErrorModel, JointProbability

from . import spncpy


def convertToFlag(value):
    return "true" if value else "false"


class HIPCompiler:
    """Convenience interface to the SPN compiler, targeting AMD GPUs through HIP.

    preloadToSharedMem : stage the input tile through LDS before computation ("gpu-shared-mem");
                         True / False force it on / off, None (the default here; the reference's
                         CUDACompiler defaults to False) lets the compiler decide from the SPN.
    computeInLogSpace  : compute in log-space (float32 unless ``hip-compute-type`` says float64);
                         False selects linear-space float64 with a final log, as in the reference.
    verbose            : print the options and the generated device code ("dump-ir").
    kwargs             : further compiler options, passed as strings (unknown names are errors).
    """

    def __init__(self, preloadToSharedMem=None, computeInLogSpace=True, verbose=False, **kwargs):
        self.verbose = verbose
        self.preloadToSharedMem = preloadToSharedMem
        self.computeInLogSpace = computeInLogSpace
        self.otherOptions = kwargs

    def compile_ll(self, spn, inputDataType="float64", errorModel=ErrorModel(), batchSize=64, supportMarginal=True,
                   name="spn_hip"):
        """Compile the SPN for the HIP target and return the compiled kernel."""
        model = SPNModel(spn, inputDataType, name)
        query = JointProbability(model, batchSize=batchSize, supportMarginal=supportMarginal, rootError=errorModel)

        tmpfile = tempfile.NamedTemporaryFile()
        if self.verbose:
            print(f"Serializing SPN to {tmpfile}")
        BinarySerializer(tmpfile.name).serialize_to_file(query)
        if not os.path.isfile(tmpfile.name):
            raise RuntimeError("Serialization of the SPN failed")

        options = {"target": "HIP",
                   "use-log-space": convertToFlag(self.computeInLogSpace),
                   "dump-ir": convertToFlag(self.verbose)}
        if self.preloadToSharedMem is not None:
            options["gpu-shared-mem"] = convertToFlag(self.preloadToSharedMem)
        if self.otherOptions is not None:
            for k, v in ((str(k), str(v)) for k, v in self.otherOptions.items()):
                if k in options and options[k] != v:
                    print(f"WARNING: Option {k} specified twice, ignoring option value {v}")
                else:
                    options[k] = v
        if self.verbose:
            print(f"Invoking compiler with options: {options}")

        kernel = spncpy.SPNCompiler().compileQuery(tmpfile.name, options)
        if not os.path.isfile(kernel.fileName()):
            raise RuntimeError("Compilation failed, not Kernel produced")
        return kernel

    def compile_mixture(self, spns, inputDataType="float64", errorModel=ErrorModel(), batchSize=64, supportMarginal=True, name="spn_hip"):
        """Compile SPNs over the same features into the experts of a gated mixture (``spnc.mixture.Mixture``). The kernel files
        of its ``kernels`` are the caller's, as those of ``compile_ll`` are."""
        from .mixture import Mixture
        return Mixture([self.compile_ll(spn, inputDataType, errorModel=errorModel, batchSize=batchSize, supportMarginal=supportMarginal,
                                        name=f"{name}_{i}") for i, spn in enumerate(spns)])

    def execute(self, kernel, inputs):
        """Execute a compiled kernel on the given inputs."""
        if type(inputs) is not np.ndarray:
            raise RuntimeError("Input is not an numpy array")
        if inputs.ndim != 2:
            raise RuntimeError("Input must be a two-dimensional array")
        return kernel.execute(inputs.shape[0], inputs)

    def log_likelihood(self, spn, inputs, errorModel=ErrorModel(), batchSize=64, supportMarginal=True):
        """Compile the SPN and immediately execute the compiled kernel on the given inputs."""
        if type(inputs) is not np.ndarray:
            raise RuntimeError("Input is not an numpy array")
        if inputs.ndim != 2:
            raise RuntimeError("Input must be a two-dimensional array")
        kernel = self.compile_ll(spn, str(inputs.dtype), errorModel=errorModel, batchSize=batchSize,
                                 supportMarginal=supportMarginal, name="spn_hip")
        results = self.execute(kernel, inputs)
        os.remove(kernel.fileName())
        return results

    @staticmethod
    def isAvailable():
        """Query the compiler if compilation for and execution on HIP GPUs is available."""
        return spncpy.SPNCompiler.isTargetSupported("HIP")
